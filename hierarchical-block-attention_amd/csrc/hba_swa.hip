// Sliding-window attention with sinks: row i of a head sees the keys j <= i with
// j > i - W or j < S, on queries and keys as they are given (any positions or
// norms already applied), forward and backward, any length.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i)
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - do_i . o_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// Forward and dq: a workgroup has 128 rows of one KV head's query heads
// (hba_rows.h) and walks the tiles of keys that they see.  dk and dv: a workgroup
// has 128 keys as the columns of S = Q . K^T and walks its KV head's query heads
// and their tokens, 32 a step, so the sum over the heads of a group stays in
// registers and nothing is added by atomics: the gradients are the same bits
// from run to run.  A tile whose keys many rows see (sinks: every later row) is
// cut into parts that sum into a workspace and are joined in order by a second
// kernel.
#include "hba_abi.h"
#include "hba_common.h"
#include "hba_rows.h"
#include "hba_xcd.h"

namespace hba {
namespace swa {

using namespace rows;

struct Args {
    const char *q, *k, *v, *dout;       // strided rows; byte strides of batch, token, head
    int64_t qs[3], ks[3], vs[3], dos[3];
    const int32_t *lens;                // rows of each sequence (nullptr: n)
    int n, Hq, Hkv, G, W, S;
    float scale, c;                     // c: logits to log2 units
    int Cn, ntiles, xmap;               // B * Hkv, row tiles of one of them, workgroup map
    char *out;                          // [B, n, Hq, D]
    float *lse, *delta;                 // [B, Hq, n]: log2-sum-exp2 (+inf: no row), do . o
    char *dq, *dk, *dv;
    float *part;                        // dk / dv sums of tiles in several parts
    int32_t *marks;                     // waves of swa_dkv whose sums are not finite
    int nst, Ps, Pn, schunk, chunk;     // tiles of sinks, parts of those and of the others, steps of a part of either
    int pslot, pslots;                  // first slot that has sums in `part`, and how many there are of one (batch, KV head)
    int first;                          // swa_join: place of the launch's first workgroup
};

__device__ __forceinline__ int seq_len(const Args &a, int b) {
    return a.lens ? max(0, min(a.n, a.lens[b])) : a.n;
}

// The rows of this wave: its lane's column and what they see.
struct Rows {
    int b, g, tok, head, len, lo, hi;   // lo .. hi: tiles' bounds over the workgroup
    bool in, valid;                     // a row of the batch; one of its sequence
    Sees w;
};

// Of 32 R rows a workgroup, wave i those of i % R.
template <int D, int R = NW> __device__ __forceinline__ bool find_rows(const Args &a, Rows &x) {
    constexpr int RT = 32 * R;
    int combo, tile;
    xcd_map(blockIdx.x, a.Cn, a.ntiles, a.xmap, combo, tile);
    if (tile >= a.ntiles || combo >= a.Cn) return false;
    x.b = combo / a.Hkv;
    x.g = combo % a.Hkv;
    x.len = seq_len(a, x.b);
    const int nr = a.n * a.G, vr = x.len * a.G;          // rows there are, rows of the sequence
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % R);
    const int r0 = tile * RT, rw = r0 + wave * RW, r = rw + (threadIdx.x & 31);
    x.in = r < nr;
    x.valid = r < vr;
    x.tok = min(r, nr - 1) / a.G;
    x.head = x.g * a.G + min(r, nr - 1) % a.G;
    // the workgroup's and the wave's tokens
    const int t0 = r0 / a.G, t1 = (min(r0 + RT, vr) - 1) / a.G;
    x.lo = max(0, t0 - a.W + 1);
    x.hi = r0 < vr ? t1 + 1 : 0;
    const int u0 = rw / a.G, u1 = (min(rw + RW, vr) - 1) / a.G;
    x.w.S = a.S;
    x.w.lo = max(0, x.tok - a.W + 1);
    x.w.hi = x.valid ? x.tok + 1 : 0;
    x.w.lo_min = max(0, u0 - a.W + 1);
    x.w.lo_max = max(0, u1 - a.W + 1);
    x.w.hi_min = u0 + 1;
    x.w.hi_max = rw < vr ? u1 + 1 : 0;
    return true;
}

template <int DT, int D>
__device__ __forceinline__ void load_rows(const char *p, bool ok, typename Op<DT>::F (&f)[D / 16]) {
    const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        f[ks] = ok ? Op<DT>::load(p + (16 * ks + 8 * hf) * Tile<DT, D>::ESZ) : Op<DT>::pack(z);
    }
}

template <int DT, int D, int KT = KEYS<DT, D>>
__device__ __forceinline__ DenseKV<DT, D, KT> keys(const Args &a, const Rows &x) {
    DenseKV<DT, D, KT> s;
    s.k = a.k + x.b * a.ks[0] + x.g * a.ks[2];
    s.v = a.v + x.b * a.vs[0] + x.g * a.vs[2];
    s.kb = a.ks[1];
    s.vb = a.vs[1];
    s.last = max(x.len, 1) - 1;
    s.ko = Tile<DT, D>::offset(s.kb);
    s.vo = Tile<DT, D>::offset(s.vb);
    return s;
}

// l: the sum that O is divided by, le: the one of the log-sum-exp.
template <int DT, int D>
__device__ __forceinline__ void store_fwd(const Args &a, const Rows &x, RowAcc<DT, D> &acc, float l, float le) {
    if (!x.in) return;
    if (!x.valid) {   // a row behind its sequence: 0
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) acc.O[dt] = f32x16{0.0f};
    }
    const int64_t row = ((int64_t)x.b * a.n + x.tok) * a.Hq + x.head;
    store_rows<DT, D>(a.out + row * D * Tile<DT, D>::ESZ, acc.O, x.valid ? 1.0f / l : 0.0f);
    if (a.lse && (threadIdx.x & 32) == 0)
        a.lse[((int64_t)x.b * a.Hq + x.head) * a.n + x.tok] = x.valid ? acc.m + __log2f(le) : INFINITY;
}

template <int DT, int D>
__device__ __forceinline__ const char *q_row(const Args &a, const Rows &x) {
    return a.q + x.b * a.qs[0] + x.tok * a.qs[1] + x.head * a.qs[2];
}
template <int DT, int D>
__device__ __forceinline__ const char *dout_row(const Args &a, const Rows &x) {
    return a.dout + x.b * a.dos[0] + x.tok * a.dos[1] + x.head * a.dos[2];
}

// 32768 tokens, 14 heads, d = 64, W = 1024, bf16: 165 us, 0.72 PFLOP/s (98 us at the
// 1.21 of a large product).  Bound by issue: per 32 rows and 32 keys 16 exponentials
// and as many multiply-adds and conversions a lane stand beside 8 matrix
// instructions (without the exponentials 144 us, without reading operands from LDS
// 150).  fp32, 2 x 2047 tokens, W = 512: 80 to 89 us, 37 at the fp32 matrix rate: 392
// workgroups with rows for 256 CUs, so some CUs have two and some one, and masked halves
// of tiles at the windows' ends.
// SEP: the log-sum-exp has a sum of its own (see attend): 155 us at 8192 tokens, 28
// heads, d = 128 with three waves per SIMD, 179 with two, 152 without it.
template <int DT, int D, bool SEP>
__global__ __launch_bounds__(64 * NW, (DT == 1 ? 3 : WAVES<DT, D>)) void swa_fwd(const Args a) {
    extern __shared__ __align__(16) char smem[];
    Rows x;
    if (!find_rows<D>(a, x)) return;
    DenseKV<DT, D> src = keys<DT, D>(a, x);
    int ns, wt0;
    const int nt = tile_list<KEYS<DT, D>>(x.lo, x.hi, a.S, ns, wt0);
    attend_begin(src, smem, 0, nt, ns, wt0);
    typename Op<DT>::F q[D / 16];
    load_rows<DT, D>(q_row<DT, D>(a, x), x.valid, q);
    RowAcc<DT, D> acc;
    attend<DT, D, false, false, SEP>(src, smem, q, nullptr, a.c, 0, nt, ns, wt0, x.w, acc);
    float l = acc.l + other_half(acc.l), le = SEP ? acc.le + other_half(acc.le) : l;
    if (__ballot(x.valid && (any_bad<D>(acc.O) || !finite(l)))) {
        attend_each<DT, D, false>(src, q, nullptr, a.c, 0, nt, ns, wt0, x.w, acc);
        le = l = acc.l + other_half(acc.l);
    }
    store_fwd<DT, D>(a, x, acc, l, le);
}

// swa_fwd where its workgroups leave CUs free: 8 waves of which `sets` have the same
// rows and share their keys, and meet in LDS.  Two sets of 4 waves (128 rows) have
// half of the tiles each; of four sets of 2 waves (64 rows, and so twice as many
// workgroups) a pair has half of the tiles of 64 keys and one of the pair 32 keys
// of each.  1001 tokens, 14 heads, W = 1024, d = 64: 20 us as one set (110 workgroups),
// 17 as two, 13 as four (220); fp32 75, 72 and 42; d = 128 25 as two and 19 as four.
template <int DT, int D, int SETS> using SetsKV = DenseKV<DT, D, (SETS == 4 ? 64 : KEYS<DT, D>)>;
template <int DT, int D, int SETS, bool SEP> constexpr size_t sets_lds() {
    constexpr size_t tiles = 4 * SetsKV<DT, D, SETS>::BYTES,
                     sums = (size_t)(SETS - 1) * 512 / SETS * (D / 2 + 2 + SEP) * 4;
    return tiles > sums ? tiles : sums;
}
template <int DT, int D, int SETS, bool SEP> __global__ __launch_bounds__(512) void swa_fwd_sets(const Args a) {
    extern __shared__ __align__(16) char smem[];
    constexpr int R = 8 / SETS, T = 64 * R;   // waves, lanes of a set
    Rows x;
    if (!find_rows<D, R>(a, x)) return;
    const int half = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    const int set = __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    constexpr int KT = SetsKV<DT, D, SETS>::KT;
    auto src = keys<DT, D, KT>(a, x);
    int ns, wt0;
    const int nt = tile_list<KT>(x.lo, x.hi, a.S, ns, wt0), mid = (nt + 1) / 2;
    const int it0 = half ? mid : 0, it1 = half ? nt : mid;
    char *mine = smem + half * 2 * src.BYTES;
    attend_begin(src, mine, it0, it1, ns, wt0);
    typename Op<DT>::F q[D / 16];
    load_rows<DT, D>(q_row<DT, D>(a, x), x.valid, q);
    RowAcc<DT, D> acc;
    attend<DT, D, false, SETS == 4, SEP>(src, mine, q, nullptr, a.c, it0, it1, ns, wt0, x.w, acc, set % 2);
    if (it1 - it0 < mid) __syncthreads();   // the other half's last tile: as many barriers for both
    // element i of set s: sums[(i (SETS - 1) + s - 1) T]
    float *sums = reinterpret_cast<float *>(smem) + threadIdx.x % T;
    constexpr int E = (SETS - 1) * T;
    if (set) {
        sums += (set - 1) * T;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[(16 * dt + r) * E] = acc.O[dt][r];
        sums[D / 2 * E] = acc.m;
        sums[(D / 2 + 1) * E] = acc.l;
        if constexpr (SEP) sums[(D / 2 + 2) * E] = acc.le;
    }
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int s = 0; s < SETS - 1; ++s, sums += T) {
        const float om = sums[D / 2 * E], m = fmaxf(acc.m, om);
        const float fa = acc.m == -INFINITY ? 0.0f : ex2(acc.m - m), fb = om == -INFINITY ? 0.0f : ex2(om - m);
        acc.m = m;
        acc.l = fmaf(sums[(D / 2 + 1) * E], fb, acc.l * fa);
        if constexpr (SEP) acc.le = fmaf(sums[(D / 2 + 2) * E], fb, acc.le * fa);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc.O[dt][r] = fmaf(sums[(16 * dt + r) * E], fb, acc.O[dt][r] * fa);
    }
    float l = acc.l + other_half(acc.l), le = SEP ? acc.le + other_half(acc.le) : l;
    if (__ballot(x.valid && (any_bad<D>(acc.O) || !finite(l)))) {
        attend_each<DT, D, false>(src, q, nullptr, a.c, 0, nt, ns, wt0, x.w, acc);
        le = l = acc.l + other_half(acc.l);
    }
    store_fwd<DT, D>(a, x, acc, l, le);
}

// The probabilities' gradient from the forward's log-sum-exps, and dq; delta =
// do . o on the way, for dk and dv.  o is the output as stored, so in bf16 delta has
// its rounding (2^-8 of sum |do||o| at most): o is what there is of the forward, and
// delta weighs on a ds only with the probability of its key.
template <int DT, int D>
__device__ __forceinline__ float row_delta(const Args &a, const Rows &x, const typename Op<DT>::F (&dO)[D / 16]) {
    typename Op<DT>::F o[D / 16];
    load_rows<DT, D>(a.out + (((int64_t)x.b * a.n + x.tok) * a.Hq + x.head) * D * Tile<DT, D>::ESZ, x.valid, o);
    float delta = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        float u[8], w[8];
        Op<DT>::unpack(o[ks], u);
        Op<DT>::unpack(dO[ks], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(u[e], w[e], delta);
    }
    return delta + other_half(delta);
}

template <int DT, int D>
__device__ __forceinline__ void store_dq(const Args &a, const Rows &x, f32x16 (&acc)[D / 32]) {
    if (!x.in) return;
    if (!x.valid) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) acc[dt] = f32x16{0.0f};
    }
    store_rows<DT, D>(a.dq + (((int64_t)x.b * a.n + x.tok) * a.Hq + x.head) * D * Tile<DT, D>::ESZ, acc, a.scale);
}

// The wave's rows of swa_dq key by key, the masked ones left out.  It finds its rows
// again: what swa_dq would hold for it through its loop costs a wave per SIMD.
template <int DT, int D> __device__ __forceinline__ void dq_each(const Args a) {
    typedef typename Op<DT>::F F;
    constexpr int KT = KEYS<DT, D>;
    const int hf = (threadIdx.x & 63) >> 5;
    Rows x;
    find_rows<D>(a, x);
    F q[D / 16], dO[D / 16];
    load_rows<DT, D>(q_row<DT, D>(a, x), x.valid, q);
    load_rows<DT, D>(dout_row<DT, D>(a, x), x.valid, dO);
    const float delta = row_delta<DT, D>(a, x, dO);
    const float lse = x.valid ? a.lse[((int64_t)x.b * a.Hq + x.head) * a.n + x.tok] : INFINITY;
    const DenseKV<DT, D> src = keys<DT, D>(a, x);
    int ns, wt0;
    const int nt = tile_list<KT>(x.lo, x.hi, a.S, ns, wt0);
    f32x16 acc[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) acc[dt] = f32x16{0.0f};
#pragma unroll 1
    for (int it = 0; it < nt; ++it) {
        const int j0 = (it < ns ? it : wt0 + it - ns) * KT;
#pragma unroll 1
        for (int j = j0; j < min(j0 + KT, x.w.hi_max); ++j) {
            const char *kj = src.k + (int64_t)min(j, src.last) * src.kb;
            const float s = dot_rows<DT, D>(q, kj, hf);
            const float dp = dot_rows<DT, D>(dO, src.v + (int64_t)min(j, src.last) * src.vb, hf);
            if (j < x.w.hi && (j >= x.w.lo || j < a.S))
                add_row<DT, D>(acc, kj, ex2(fmaf(s, a.c, -lse)) * (dp - delta), hf);
        }
    }
    store_dq<DT, D>(a, x, acc);
}

// What half16's rounding left of p.
template <int DT>
__device__ __forceinline__ typename Op<DT>::F rest16(const f32x16 &p, int u, typename Op<DT>::F f) {
    float y[8];
    Op<DT>::unpack(f, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = p[8 * u + e] - y[e];
    return Op<DT>::pack(y);
}
constexpr int FEW = 256;   // first rows of a sequence whose ds enters its products in two parts, see swa_dq

// Rows as swa_fwd, three products a tile (q . k again, do . v, ds . k).  8192 tokens,
// 28 heads, d = 128, W = 1024, bf16: 200 us, 140 at the rate of a large product; the
// matrix cores are busy 44 % of the time (the forward: 42 %).  fp32: 1.64 ms, 1.12 at
// the fp32 matrix rate.
template <int DT, int D> __global__ __launch_bounds__(64 * NW, DT == 1 ? 2 : 1) void swa_dq(const Args a) {
    extern __shared__ __align__(16) char smem[];
    typedef Tile<DT, D> TL;
    typedef typename Op<DT>::F F;
    constexpr int NKS = D / 16, NDT = D / 32, KT = KEYS<DT, D>;
    const int lane = threadIdx.x & 63, hf = lane >> 5;
    Rows x;
    if (!find_rows<D>(a, x)) return;
    const DenseKV<DT, D> src = keys<DT, D>(a, x);
    int ns, wt0;
    const int nt = tile_list<KT>(x.lo, x.hi, a.S, ns, wt0);
    const uint32_t lds = lds_offset(smem);
    if (nt > 0) src.stage(0 < ns ? 0 : wt0, lds);
    F q[NKS], dO[NKS];
    load_rows<DT, D>(q_row<DT, D>(a, x), x.valid, q);
    load_rows<DT, D>(dout_row<DT, D>(a, x), x.valid, dO);
    const int64_t hrow = ((int64_t)x.b * a.Hq + x.head) * a.n + x.tok;
    const float delta = row_delta<DT, D>(a, x, dO);
    if (x.valid && hf == 0) a.delta[hrow] = delta;
    const float lse = x.valid ? a.lse[hrow] : INFINITY;
    // ds enters the product rounded to bf16 (2^-8 at most).  A sequence's first rows see
    // few keys, so they have its largest gradients (as 1 / sqrt(keys)) and most of the
    // whole tensor's rounding error: their ds enters with its rest.  The rule goes by a
    // row's place, so it does little where a window leaves every row few keys, and a
    // later row's own relative error is what it was.  Its border was chosen at 1999
    // tokens, W = 512, N(0, 1), d = 64: dq is off by 2.2e-3 of its norm, 2.46e-3
    // without (2.26e-3 for 128 rows; its own rounding alone 1.66e-3), for 1 us of 31.
    const bool few = x.w.hi_max <= FEW;
    const f32x16 zero = {0.0f};
    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc[dt] = zero;
#pragma unroll 1
    for (int it = 0; it < nt; ++it) {
        wait_vm<0>();
        __syncthreads();
        const int cur = it & 1, nx = it + 1;
        if (nx < nt) src.stage(nx < ns ? nx : wt0 + nx - ns, lds + (cur ^ 1) * src.BYTES);
        const int j0 = (it < ns ? it : wt0 + it - ns) * KT;
        if (j0 >= x.w.hi_max || (j0 + KT <= x.w.lo_min && j0 >= a.S)) continue;
        const char *t = smem + cur * src.BYTES;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            const int jh = j0 + 32 * kt;
            if (jh >= x.w.hi_max || (jh + 32 <= x.w.lo_min && jh >= a.S)) continue;
            f32x16 s = zero, dp = zero;
            dp = dp - delta;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                s = Op<DT>::mma(src.kf(t, kt, ks, lane), q[ks], s);
                dp = Op<DT>::mma(TL::row(t + KT * TL::ROWB, 32 * kt + (lane & 31), ks, hf), dO[ks], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = ex2(fmaf(s[r], a.c, -lse)) * dp[r];
            if (!(jh + 32 <= x.w.hi_min && (jh >= x.w.lo_max || jh + 32 <= a.S))) {
                const uint64_t see = seen_bits(x.w.lo, x.w.hi, a.S, jh) >> src.key(0, hf);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = keep(s[r], see, src.key(r, 0), 0.0f);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const F df = half16<DT>(s, u);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
                    acc[dt] = Op<DT>::mma(TL::col(t, 32 * kt + 16 * u, dt, lane), df, acc[dt]);
                if (DT == 1 && few) {
                    const F rest = rest16<DT>(s, u, df);
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
                        acc[dt] = Op<DT>::mma(TL::col(t, 32 * kt + 16 * u, dt, lane), rest, acc[dt]);
                }
            }
        }
    }
    if (__ballot(x.valid && any_bad<D>(acc))) {
        dq_each<DT, D>(a);
        return;
    }
    store_dq<DT, D>(a, x, acc);
}

constexpr int KB = 32 * NW;   // keys of a dk / dv workgroup
constexpr int TT = 32;        // tokens of its steps

// Whether the keys' operands come from LDS each time: where keys, values and both
// sums would leave registers for one wave per SIMD only.
template <int DT, int D> constexpr bool keys_in_lds() { return DT == 1 && D == 128; }

// One past the last token that sees keys k0 .. k0 + KB - 1, and the steps over them.
__device__ __forceinline__ int last_token(int k0, int len, int W, int S) {
    return k0 < S ? len : min(len, k0 + KB - 1 + W);
}
__device__ __forceinline__ int steps(int k0, int len, int W, int S) {
    return max(0, (last_token(k0, len, W, S) + TT - 1) / TT - k0 / TT);
}

// The workgroup's key tile and part of it: tiles of sinks first.
__device__ __forceinline__ void find_part(const Args &a, int slot, int &tile, int &part) {
    const int sinks = a.nst * a.Ps;
    if (slot < sinks) {
        tile = slot / a.Ps;
        part = slot % a.Ps;
    } else {
        tile = a.nst + (slot - sinks) / a.Pn;
        part = (slot - sinks) % a.Pn;
    }
}

// A dk / dv workgroup's keys, and this lane's.
struct Keys {
    int b, g, len, k0, kw, j;     // k0: the workgroup's first key, kw: the wave's, j: the lane's
    int nst, i0, i1, parts;       // token tiles, this part's steps (head, token tile), the tile's parts
    int64_t at;                   // the lane's place among the parts
};

__device__ __forceinline__ void find_keys(const Args &a, Keys &x) {
    const int combo = blockIdx.x % a.Cn, slot = blockIdx.x / a.Cn;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tile, part;
    find_part(a, slot, tile, part);
    x.b = combo / a.Hkv;
    x.g = combo % a.Hkv;
    x.len = seq_len(a, x.b);
    x.k0 = tile * KB;
    x.kw = x.k0 + 32 * wave;
    x.j = x.kw + (lane & 31);
    x.nst = steps(x.k0, x.len, a.W, a.S);
    x.parts = tile < a.nst ? a.Ps : a.Pn;
    const int chunk = tile < a.nst ? a.schunk : a.chunk;
    x.i0 = part * chunk;
    x.i1 = min(x.nst * a.G, x.i0 + chunk);
    x.at = ((int64_t)combo * a.pslots + slot - a.pslot) * KB + 32 * wave + (lane & 31);
}

template <int DT, int D>
__device__ __forceinline__ void load_keys(const Args &a, const Keys &x, typename Op<DT>::F (&kf)[D / 16],
                                          typename Op<DT>::F (&vf)[D / 16]) {
    const int64_t j = min(x.j, a.n - 1);
    load_rows<DT, D>(a.k + x.b * a.ks[0] + j * a.ks[1] + x.g * a.ks[2], x.j < x.len, kf);
    load_rows<DT, D>(a.v + x.b * a.vs[0] + j * a.vs[1] + x.g * a.vs[2], x.j < x.len, vf);
}

template <int DT, int D>
__device__ __forceinline__ void store_keys(const Args &a, const Keys &x, f32x16 (&dk)[D / 32], f32x16 (&dv)[D / 32]) {
    if (x.parts > 1) {   // the sums as they are, for swa_join
        store_rows<0, D>(reinterpret_cast<char *>(a.part + x.at * 2 * D), dk, 1.0f);
        store_rows<0, D>(reinterpret_cast<char *>(a.part + x.at * 2 * D + D), dv, 1.0f);
        return;
    }
    if (x.j >= a.n) return;
    if (x.j >= x.len) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dk[dt] = dv[dt] = f32x16{0.0f};
    }
    const int64_t row = (((int64_t)x.b * a.n + x.j) * a.Hkv + x.g) * D * Tile<DT, D>::ESZ;
    store_rows<DT, D>(a.dk + row, dk, a.scale);
    store_rows<DT, D>(a.dv + row, dv, 1.0f);
}

// Four products a step of 32 tokens.  Same case as swa_dq: 310 to 350 us, 186 at the
// rate of a large product (fp32: 2.5 ms, 1.49).  Each operand that a wave reads from LDS serves one matrix
// instruction (its 32 keys are the other one): LDS is busy some 45 % of the time, the
// matrix cores 36 %, and two waves a SIMD do not hide one behind the other wholly.
template <int DT, int D>
__global__ __launch_bounds__(64 * NW, (DT == 1 ? (D == 64 ? 3 : 2) : 1)) void swa_dkv(const Args a) {
    extern __shared__ __align__(16) char smem[];
    typedef Tile<DT, D> TL;
    typedef typename Op<DT>::F F;
    constexpr int NKS = D / 16, NDT = D / 32, BYTES = 2 * TT * TL::ROWB + 2 * TT * 4;
    constexpr bool KL = keys_in_lds<DT, D>();
    const int lane = threadIdx.x & 63, hf = lane >> 5;
    Keys x;
    find_keys(a, x);
    if (x.i0 >= x.i1 && x.parts > 1) {   // a part with nothing to sum is not read either
        if (lane == 0) a.marks[blockIdx.x * NW + (threadIdx.x >> 6)] = 0;
        return;
    }
    const uint32_t lds = lds_offset(smem);
    const int last = max(x.len, 1) - 1;
    const uint32_t qo = TL::offset(a.qs[1]), doo = TL::offset(a.dos[1]);
    // the step that is staged next: head h, token tile tt of it
    int h = x.g * a.G + (x.nst ? x.i0 / x.nst : 0), tt = x.nst ? x.i0 % x.nst : 0;
    const auto stage = [&](int buf) {
        const int t0 = (x.k0 / TT + tt) * TT;
        const uint32_t to = lds + buf * BYTES;
        TL::template stage<TT>(a.q + x.b * a.qs[0] + h * a.qs[2], a.qs[1], qo, t0, last, to);
        TL::template stage<TT>(a.dout + x.b * a.dos[0] + h * a.dos[2], a.dos[1], doo, t0, last, to + TT * TL::ROWB);
        float *ld = reinterpret_cast<float *>(smem + buf * BYTES + 2 * TT * TL::ROWB);
        if (threadIdx.x < 2 * TT) {   // -lse, -delta
            const int t = min(t0 + ((int)threadIdx.x & (TT - 1)), last);
            ld[threadIdx.x] = -(threadIdx.x < TT ? a.lse : a.delta)[((int64_t)x.b * a.Hq + h) * a.n + t];
        }
        if (++tt == x.nst) {
            tt = 0;
            ++h;
        }
    };
    int ct = tt;   // token tile of the step that is computed
    char *tk = smem + 2 * BYTES;
    if (x.i0 < x.i1) {
        stage(0);
        if constexpr (KL)
            TL::template stage<KB>(a.k + x.b * a.ks[0] + x.g * a.ks[2], a.ks[1], TL::offset(a.ks[1]), x.k0, last,
                                   lds + 2 * BYTES);
    }
    F kf[NKS], vf[NKS];
    load_keys<DT, D>(a, x, kf, vf);
    const f32x16 zero = {0.0f};
    f32x16 dk[NDT], dv[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) dk[dt] = dv[dt] = zero;
    const int tend = x.kw < a.S ? x.len : min(x.len, x.kw + 31 + a.W);   // tokens that see one of the wave's keys
#pragma unroll 1
    for (int it = x.i0; it < x.i1; ++it) {
        wait_vm<0>();
        __syncthreads();
        const int cur = (it - x.i0) & 1, t0 = (x.k0 / TT + ct) * TT;
        ct = ct + 1 == x.nst ? 0 : ct + 1;
        if (it + 1 < x.i1) stage(cur ^ 1);
        const char *tq = smem + cur * BYTES, *td = tq + TT * TL::ROWB;
        const float *ld = reinterpret_cast<const float *>(td + TT * TL::ROWB);
        if (t0 + TT <= x.kw || t0 >= tend) continue;
        {
            const int th = t0;
            f32x16 s = zero, dp;
#pragma unroll
            for (int g = 0; g < 4; ++g) {   // do . v starts from -delta
                const f32x4 dl = *reinterpret_cast<const f32x4 *>(ld + TT + 8 * g + 4 * hf);
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[4 * g + e] = dl[e];
            }
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                s = Op<DT>::mma(TL::row(tq, lane & 31, ks, hf), KL ? TL::row(tk, x.kw - x.k0 + (lane & 31), ks, hf) : kf[ks], s);
                dp = Op<DT>::mma(TL::row(td, lane & 31, ks, hf), vf[ks], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 ls = *reinterpret_cast<const f32x4 *>(ld + 8 * g + 4 * hf);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * g + e] = ex2(fmaf(s[4 * g + e], a.c, ls[e]));
                    dp[4 * g + e] *= s[4 * g + e];
                }
            }
            if (!(th >= x.kw + 31 && th + 32 <= x.len && (th + 32 <= x.kw + a.W || x.kw + 32 <= a.S))) {
                // tokens j .. that see key j
                const uint64_t see =
                    seen_bits(x.j, x.j < a.S ? x.len : min(x.len, x.j + a.W), 0, th) >> (4 * hf);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = keep(s[r], see, 8 * (r >> 2) + (r & 3), 0.0f);
                    dp[r] = keep(dp[r], see, 8 * (r >> 2) + (r & 3), 0.0f);
                }
            }
            // p and ds rounded to bf16 (2^-8 each at most), as the matrix cores take them; sums in fp32
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const F pf = half16<DT>(s, u), df = half16<DT>(dp, u);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    dv[dt] = Op<DT>::mma(TL::col(td, 16 * u, dt, lane), pf, dv[dt]);
                    dk[dt] = Op<DT>::mma(TL::col(tq, 16 * u, dt, lane), df, dk[dt]);
                }
                if (DT == 1 && th < FEW) {   // as in swa_dq; dk: 1.46 times its own rounding without, 1.31 with, 3 us of 44
                    const F rest = rest16<DT>(dp, u, df);
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
                        dk[dt] = Op<DT>::mma(TL::col(tq, 16 * u, dt, lane), rest, dk[dt]);
                }
            }
        }
    }
    const uint64_t bad = __ballot(x.j < x.len && (any_bad<D>(dk) || any_bad<D>(dv)));
    if (lane == 0) a.marks[blockIdx.x * NW + (threadIdx.x >> 6)] = bad != 0;
    store_keys<DT, D>(a, x, dk, dv);
}

// dk and dv of the tiles in several parts: the parts' sums, in order.  A workgroup
// takes 1024 elements of one key tile and KV head, 4 a thread, so that there
// are enough of them to keep HBM busy (8192 tokens, 4 KV heads, d = 128, 3 parts: 20 us).
//
// Keys of a wave that swa_dkv marked are computed here instead, token by token,
// the masked ones left out: 2D / 4 threads a key, those of its dk with q . k, those
// of its dv with do . v.  (Inlined in swa_dkv that path's registers cost it a wave
// per SIMD: 8192 tokens, d = 128, 390 us and 735; 2000 tokens, d = 64, 39 and 52.)
constexpr int JE = 1024;
template <int DT, int D> __global__ __launch_bounds__(JE / 4) void swa_join(const Args a) {
    typedef typename St<DT>::T T;
    constexpr int PER = KB * 2 * D / JE, ESZ = Tile<DT, D>::ESZ;
    const int place = a.first + blockIdx.x;
    const int e = place % PER * JE + threadIdx.x * 4, r = e / (2 * D), x = e % (2 * D), xd = x % D;
    const int combo = place / PER % a.Cn, tile = place / PER / a.Cn;
    const int P = tile < a.nst ? a.Ps : a.Pn;
    const int slot = tile < a.nst ? tile * a.Ps : a.nst * a.Ps + (tile - a.nst) * a.Pn;
    const int b = combo / a.Hkv, g = combo % a.Hkv, len = seq_len(a, b), k0 = tile * KB, j = k0 + r;
    const int chunk = tile < a.nst ? a.schunk : a.chunk;
    const int used = min(P, (steps(k0, len, a.W, a.S) * a.G + chunk - 1) / chunk);
    bool marked = false;   // the same for the threads of a key
    for (int i = 0; i < used; ++i) marked |= a.marks[((slot + i) * a.Cn + combo) * NW + r / 32] != 0;
    if (j >= a.n || (P == 1 && !marked)) return;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (marked && j < len) {
        // this thread's 4 elements of the key (x < D) or the value
        const char *kv = x < D ? a.k + b * a.ks[0] + j * a.ks[1] + g * a.ks[2]
                               : a.v + b * a.vs[0] + j * a.vs[1] + g * a.vs[2];
        f32x4 own;
#pragma unroll
        for (int i = 0; i < 4; ++i) own[i] = St<DT>::ld(reinterpret_cast<const T *>(kv), xd + i);
        const int t1 = j < a.S ? len : min(len, j + a.W);
        for (int h = g * a.G; h < (g + 1) * a.G; ++h)
            for (int t = j; t < t1; ++t) {
                const char *qt = a.q + b * a.qs[0] + t * a.qs[1] + h * a.qs[2];
                const char *ot = a.dout + b * a.dos[0] + t * a.dos[1] + h * a.dos[2];
                f32x4 qo;   // the query's elements for the key's threads, do's for the value's, and the other way round
                float dot = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    qo[i] = St<DT>::ld(reinterpret_cast<const T *>(x < D ? qt : ot), xd + i);
                    dot = fmaf(own[i], qo[i], dot);
                }
#pragma unroll
                for (int o = 1; o < D / 4; o <<= 1) dot += __shfl_xor(dot, o, 64);
                const float other = __shfl_xor(dot, D / 4, 64);
                const int64_t at = ((int64_t)b * a.Hq + h) * a.n + t;
                const float p = ex2(fmaf(x < D ? dot : other, a.c, -a.lse[at]));
                const float w = x < D ? p * (other - a.delta[at]) : p;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(w, qo[i], sum[i]);
            }
    } else if (j < len) {
        const float *p = a.part + ((int64_t)combo * a.pslots + slot - a.pslot) * KB * 2 * D + e;
#pragma unroll 4
        for (int i = 0; i < used; ++i) sum = sum + *reinterpret_cast<const f32x4 *>(p + (int64_t)i * KB * 2 * D);
    }
    const float f = x < D ? a.scale : 1.0f;
    char *to = (x < D ? a.dk : a.dv) + ((((int64_t)b * a.n + j) * a.Hkv + g) * D + xd) * ESZ;
    if constexpr (DT == 1)
        *reinterpret_cast<uint2 *>(to) = make_uint2(pk_bf16(sum[0] * f, sum[1] * f), pk_bf16(sum[2] * f, sum[3] * f));
    else
        *reinterpret_cast<f32x4 *>(to) = sum * f;
}

// How dk and dv are cut.  The workgroups run in rounds of as many as the card holds;
// a tile without sinks is cut into the number of parts for which rounds times
// steps of a part (and a part's start and end, worth some 4 steps), and the
// traffic of the parts' sums, take least.  A step takes about 0.9 us at d = 64,
// 1.8 at d = 128 (bf16; fp32 eight times that).  Measured at 8192 tokens, 28 / 4
// heads, d = 128, kernel and join: 2 parts 481 us, 3 (taken) 360, 4 410, 8 412.
struct Cut {
    int ntiles, nst, Ps, Pn, schunk, chunk;
    int64_t slots;
    // tiles in one part store dk and dv at once: only the others' slots have sums to join
    int64_t part_slots() const { return (Ps > 1 ? (int64_t)nst * Ps : 0) + (Pn > 1 ? (int64_t)(ntiles - nst) * Pn : 0); }
};
static Cut cut(int dtype, int64_t d, int64_t Cn, int64_t n, int64_t G, int64_t W, int64_t S) {
    Cut c = {}, best = {};
    c.ntiles = (int)((n + KB - 1) / KB);
    c.nst = (int)(((S < n ? S : n) + KB - 1) / KB);
    const int64_t most = G * ((n + TT - 1) / TT);                     // steps of a tile of sinks
    int64_t usual = G * ((KB + W - 1 + TT - 1) / TT + 1);             // of another
    if (usual > most) usual = most;
    const int64_t room = dtype == HBA_DTYPE_BF16 && d == 64 ? 768 : d == 64 || dtype == HBA_DTYPE_BF16 ? 512 : 256;
    const double step = (double)d / 64 * 0.9 * (dtype == HBA_DTYPE_BF16 ? 1 : 8);
    double least = 0;
    for (int64_t P = 1; P <= 32 && P <= usual; ++P) {
        const int64_t ch = (usual + P - 1) / P;
        // Tiles of sinks, which every later row sees, get parts of as many steps; where
        // that were more than four rounds of parts, longer ones (a workspace of four
        // rounds at most, where thousands of sinks would ask for many GB).
        const int64_t even = (c.nst * Cn * most + 4 * room - 1) / (4 * room), sch = even > ch ? even : ch;
        c.chunk = (int)ch;
        c.schunk = (int)sch;
        c.Pn = (int)((usual + ch - 1) / ch);
        c.Ps = (int)((most + sch - 1) / sch);
        c.slots = (int64_t)c.nst * c.Ps + (int64_t)(c.ntiles - c.nst) * c.Pn;
        const auto rounds = [&](int64_t slots) { return (double)((slots * Cn + room - 1) / room); };
        const int64_t sinks = (int64_t)c.nst * c.Ps;
        const double us = (sch == ch ? rounds(c.slots) * (ch + 4)
                                     : rounds(sinks) * (sch + 4) + rounds(c.slots - sinks) * (ch + 4)) * step +
                          (double)(c.part_slots() * Cn) * KB * 2 * d * 8 / 4e6;
        if (P == 1 || us < least) {
            least = us;
            best = c;
        }
    }
    return best;
}

// The workspace: delta, marks, parts.
static size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }
static size_t delta_bytes(int64_t B, int64_t n, int64_t Hq) { return round256((size_t)(B * Hq * n) * 4); }
static size_t mark_bytes(int64_t Cn, const Cut &c) { return round256((size_t)(Cn * c.slots) * NW * 4); }

template <int DT, int D, class K> static int lds_room(K kern, size_t bytes) {
    if (bytes <= 65536) return HBA_OK;
    return hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)bytes) == hipSuccess
               ? HBA_OK
               : HBA_ERR_LAUNCH;
}

template <int DT, int D, int SETS, bool SEP> static int launch_sets(const Args &a, int64_t grid, hipStream_t s) {
    constexpr size_t lds = sets_lds<DT, D, SETS, SEP>();
    if (int st = lds_room<DT, D>(swa_fwd_sets<DT, D, SETS, SEP>, lds)) return st;
    hipLaunchKernelGGL((swa_fwd_sets<DT, D, SETS, SEP>), dim3((unsigned)grid), dim3(512), lds, s, a);
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}
template <int DT, int D, bool SEP> static int launch_fwd(const Args &a, int64_t grid, hipStream_t s) {
    constexpr size_t lds = 2 * DenseKV<DT, D>::BYTES;
    if constexpr (WAVES<DT, D> >= 2) {   // 8 waves on a CU
        // What the meeting costs, in keys: 300 tokens, d = 64, W = 64, 128 and 256 take 7.8, 8.6 and 9.7 us as one
        // set, the last 9.4 as two, and all 7.7, 7.9 and 8.2 as four; d = 128, W = 128 and 256: 12.2 and 14.0 as one,
        // 12.4 and 13.6 as two.  100 tokens: 6.3 as one, 6.6 as four.
        // And in workgroups, one, two and four sets at d = 64, W = 1024: 110 (of 128 rows) 20, 17 and 13; 166 23, 19
        // and 15; 220 23, 20 and 19 (with W = 128 9.4, 9.3 and 11.3); 308 24, 21 and 25; 660, W = 512 26, 31 and 26.
        // d = 128: 220 31, 26 and 26; 332 37, 31 and 44; 440 40, 48 and 39.  So the borders are safe rather than best
        // between 128 and 320 workgroups.  Sinks are not counted in `seen`.
        const int seen = a.W < a.n ? a.W : a.n;
        Args b = a;
        int64_t more;
        b.ntiles = (int)(((int64_t)a.n * a.G + 63) / 64);
        b.xmap = xcd_pick(b.Cn, b.ntiles, more);
        if (more <= 256 && seen >= 128) return launch_sets<DT, D, 4, SEP>(b, more, s);
        if (grid <= 256 && seen >= 256) return launch_sets<DT, D, 2, SEP>(a, grid, s);
    }
    if (int st = lds_room<DT, D>(swa_fwd<DT, D, SEP>, lds)) return st;
    hipLaunchKernelGGL((swa_fwd<DT, D, SEP>), dim3((unsigned)grid), dim3(64 * NW), lds, s, a);
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

template <int DT, int D> static int launch_bwd(Args a, int64_t grid, const Cut &c, hipStream_t s) {
    constexpr size_t lds = 2 * DenseKV<DT, D>::BYTES, ldk = 2 * (2 * TT * Tile<DT, D>::ROWB + 2 * TT * 4) +
                         (keys_in_lds<DT, D>() ? KB * Tile<DT, D>::ROWB : 0);
    if (int st = lds_room<DT, D>(swa_dq<DT, D>, lds)) return st;
    if (int st = lds_room<DT, D>(swa_dkv<DT, D>, ldk)) return st;
    hipLaunchKernelGGL((swa_dq<DT, D>), dim3((unsigned)grid), dim3(64 * NW), lds, s, a);
    HBA_LAUNCH_CHECK();
    a.ntiles = c.ntiles;
    hipLaunchKernelGGL((swa_dkv<DT, D>), dim3((unsigned)(c.slots * a.Cn)), dim3(64 * NW), ldk, s, a);
    HBA_LAUNCH_CHECK();
    // 16 or 32 workgroups a key tile: more than a launch takes from 2^20 or 2^19 tiles on
    const int64_t places = (int64_t)c.ntiles * a.Cn * (KB * 2 * D / JE), most = 1 << 23;
    for (int64_t at = 0; at < places; at += most) {
        a.first = (int)at;
        hipLaunchKernelGGL((swa_join<DT, D>), dim3((unsigned)(places - at < most ? places - at : most)), dim3(JE / 4), 0,
                           s, a);
        HBA_LAUNCH_CHECK();
    }
    return HBA_OK;
}

// Rows whose strides the kernels' 32-bit offsets within a tile can span.
static bool rows_near(const int64_t *st, int64_t esz) { return st[1] >= 0 && st[1] * esz < (1 << 24); }

static void set_strides(int64_t (&to)[3], const int64_t *from, int64_t esz) {
    for (int i = 0; i < 3; ++i) to[i] = from[i] * esz;
}

static int check(int dtype, int64_t B, int64_t n, int64_t Hq, int64_t Hkv, int64_t d, int64_t W, int64_t S,
                 float scale) {
    if (int st = abi::check_dtype_dim(dtype, d)) return st;
    if (B <= 0 || n <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || W < 1 || S < 0) return HBA_ERR_INVALID_ARG;
    if (!(scale > 0.0f) || !(scale < INFINITY)) return HBA_ERR_INVALID_ARG;
    // rows, steps and workgroups are counted in 32 bits
    if (n > (1 << 28) || n * (Hq / Hkv) > 0x7fffff00 || B * Hq * ((n + 31) / 32 + 8) > 0x7fffffff)
        return HBA_ERR_UNSUPPORTED;
    if (!abi::launchable(B * Hkv * ((n * (Hq / Hkv) + RT - 1) / RT) + 8, 64 * NW)) return HBA_ERR_UNSUPPORTED;
    return HBA_OK;
}

}  // namespace swa
}  // namespace hba

using namespace hba;

extern "C" int hba_swa_fwd(int dtype, const void *q, const int64_t q_strides[3], const void *k,
                           const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
                           const int32_t *lens, int64_t B, int64_t n, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                           int64_t S, float scale, void *out, float *lse, void *stream) {
    if (int st = swa::check(dtype, B, n, Hq, Hkv, d, W, S, scale)) return st;
    if (!q || !k || !v || !q_strides || !k_strides || !v_strides || !out) return HBA_ERR_INVALID_ARG;
    if (!abi::rows_aligned(dtype, q, q_strides) || !abi::rows_aligned(dtype, k, k_strides) ||
        !abi::rows_aligned(dtype, v, v_strides) || !abi::aligned16(out))
        return HBA_ERR_UNSUPPORTED;
    const int64_t e = abi::elem_size(dtype);
    if (!swa::rows_near(k_strides, e) || !swa::rows_near(v_strides, e)) return HBA_ERR_UNSUPPORTED;
    swa::Args a = {};
    a.q = (const char *)q;
    a.k = (const char *)k;
    a.v = (const char *)v;
    swa::set_strides(a.qs, q_strides, e);
    swa::set_strides(a.ks, k_strides, e);
    swa::set_strides(a.vs, v_strides, e);
    a.lens = lens;
    a.n = (int)n;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.G = (int)(Hq / Hkv);
    a.W = (int)(W < n ? W : n);
    a.S = (int)(S < n ? S : n);
    a.scale = scale;
    a.c = scale * rows::LOG2E;
    a.Cn = (int)(B * Hkv);
    a.ntiles = (int)((n * a.G + rows::RT - 1) / rows::RT);
    int64_t grid;
    a.xmap = xcd_pick(a.Cn, a.ntiles, grid);
    a.out = (char *)out;
    a.lse = lse;
    int st = HBA_OK;
#define HBA_SWA(DT, D)                                                                       \
    st = lse && DT == 1 ? swa::launch_fwd<DT, D, DT == 1>(a, grid, (hipStream_t)stream)      \
                        : swa::launch_fwd<DT, D, false>(a, grid, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_SWA);
#undef HBA_SWA
    return st;
}

extern "C" int hba_swa_bwd_workspace_bytes(int dtype, int64_t B, int64_t n, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                                           int64_t S, size_t *bytes) {
    if (!bytes) return HBA_ERR_INVALID_ARG;
    if (int st = swa::check(dtype, B, n, Hq, Hkv, d, W, S, 1.0f)) return st;
    if (W > n) W = n;
    if (S > n) S = n;
    const swa::Cut c = swa::cut(dtype, d, B * Hkv, n, Hq / Hkv, W, S);
    *bytes = swa::delta_bytes(B, n, Hq) + swa::mark_bytes(B * Hkv, c) +
             (size_t)(B * Hkv) * c.part_slots() * swa::KB * 2 * d * 4;
    return HBA_OK;
}

extern "C" int hba_swa_bwd(int dtype, const void *q, const int64_t q_strides[3], const void *k,
                           const int64_t k_strides[3], const void *v, const int64_t v_strides[3], const void *out,
                           const float *lse, const void *dout, const int64_t dout_strides[3], const int32_t *lens,
                           int64_t B, int64_t n, int64_t Hq, int64_t Hkv, int64_t d, int64_t W, int64_t S,
                           float scale, void *workspace, size_t ws_bytes, void *dq, void *dk, void *dv,
                           void *stream) {
    if (int st = swa::check(dtype, B, n, Hq, Hkv, d, W, S, scale)) return st;
    if (!q || !k || !v || !q_strides || !k_strides || !v_strides || !out || !lse || !dout || !dout_strides ||
        !workspace || !dq || !dk || !dv)
        return HBA_ERR_INVALID_ARG;
    size_t need = 0;
    if (int st = hba_swa_bwd_workspace_bytes(dtype, B, n, Hq, Hkv, d, W, S, &need)) return st;
    if (ws_bytes < need) return HBA_ERR_INVALID_ARG;
    if (!abi::rows_aligned(dtype, q, q_strides) || !abi::rows_aligned(dtype, k, k_strides) ||
        !abi::rows_aligned(dtype, v, v_strides) || !abi::rows_aligned(dtype, dout, dout_strides) ||
        !abi::aligned16(out) || !abi::aligned16(dq) || !abi::aligned16(dk) || !abi::aligned16(dv) ||
        !abi::aligned16(workspace))
        return HBA_ERR_UNSUPPORTED;
    const int64_t e = abi::elem_size(dtype);
    if (!swa::rows_near(q_strides, e) || !swa::rows_near(k_strides, e) || !swa::rows_near(v_strides, e) ||
        !swa::rows_near(dout_strides, e))
        return HBA_ERR_UNSUPPORTED;
    swa::Args a = {};
    a.q = (const char *)q;
    a.k = (const char *)k;
    a.v = (const char *)v;
    a.dout = (const char *)dout;
    swa::set_strides(a.qs, q_strides, e);
    swa::set_strides(a.ks, k_strides, e);
    swa::set_strides(a.vs, v_strides, e);
    swa::set_strides(a.dos, dout_strides, e);
    a.lens = lens;
    a.n = (int)n;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.G = (int)(Hq / Hkv);
    a.W = (int)(W < n ? W : n);
    a.S = (int)(S < n ? S : n);
    a.scale = scale;
    a.c = scale * rows::LOG2E;
    a.Cn = (int)(B * Hkv);
    a.ntiles = (int)((n * a.G + rows::RT - 1) / rows::RT);
    int64_t grid;
    a.xmap = xcd_pick(a.Cn, a.ntiles, grid);
    a.out = (char *)const_cast<void *>(out);
    a.lse = const_cast<float *>(lse);
    a.delta = (float *)workspace;
    a.marks = (int32_t *)((char *)workspace + swa::delta_bytes(B, n, Hq));
    a.dq = (char *)dq;
    a.dk = (char *)dk;
    a.dv = (char *)dv;
    const swa::Cut c = swa::cut(dtype, d, a.Cn, n, a.G, a.W, a.S);
    a.part = (float *)((char *)a.marks + swa::mark_bytes(a.Cn, c));
    a.nst = c.nst;
    a.Ps = c.Ps;
    a.Pn = c.Pn;
    a.pslot = c.Ps > 1 ? 0 : c.nst;
    a.pslots = (int)c.part_slots();
    a.schunk = c.schunk;
    a.chunk = c.chunk;
    if (!abi::launchable(c.slots * a.Cn, 64 * rows::NW) || c.slots * a.Cn * rows::NW > 0x7fffffff ||
        (int64_t)c.ntiles * a.Cn * (swa::KB * 2 * d / swa::JE) > 0x7fffffff)
        return HBA_ERR_UNSUPPORTED;
    int st = HBA_OK;
#define HBA_SWA(DT, D) st = swa::launch_bwd<DT, D>(a, grid, c, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_SWA);
#undef HBA_SWA
    return st;
}
