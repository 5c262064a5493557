// Attention of new tokens over the paged cache (kr_pages, v_pages): the newest token
// of each sequence (decode), several (a part of a prompt), whole or through a
// causal window with sinks; and of a batch whose sequences share their first
// pages, whose keys are then read once for all.
//
// The queries come raw: QKNorm, the rotation at each token's own position and its
// sequence's scale are applied here in fp32.  For the bf16 matrix cores the
// result is split into two bf16 parts (high + low, 16 bits of mantissa), so the
// logits keep fp32-like queries: one bf16 rounding would move a logit by 2^-9 of
// |q||k| and cost as much accuracy as all that follows.
//
//   decode_kernel  one token per sequence: memory-bound.  A wave takes a page of
//                  one KV head in operand order straight into registers (its
//                  heads are the 16 columns), workgroups share a sequence's pages
//                  when there are few sequences.
//   rows_kernel    128 rows (token, head) a workgroup over staged pages
//                  (hba_rows.h): parts of prompts, and the shared pages for the
//                  rows of the whole batch.
//   join_kernel    the parts of a row, by their maxima and sums.
#include "hba_abi.h"
#include "hba_common.h"
#include "hba_ragged.h"
#include "hba_rows.h"

namespace hba {
namespace paged {

using rows::ex2;
using rows::LOG2E;
using rows::Op;

struct Args {
    const char *q;                      // [T, Hq, D] raw; byte strides of token and head
    int64_t qst, qsh;
    const float *gain;                  // QKNorm gains (nullptr: no norm)
    float eps;
    const float *cos, *sin;             // [n_tab, D] (nullptr: no rotation)
    int64_t n_tab;
    const char *kr, *v;
    int64_t pages;
    const int32_t *table, *lens, *cu;   // cu: nullptr for one token per sequence
    const float *scales;
    int T, Bd, Hq, Hkv, G, maxp, max_len, W, S;   // W: 0 for every key
    int shared;                         // pages that all sequences begin with
    int slots, slot0, part;             // parts of a row: how many, this launch's first, pages of one of them
    char *out;                          // [T, Hq, D]
    float *po, *pml;                    // parts: [T, Hq, slots, D] sums, [T, Hq, slots, 2] maximum (log2 units) and sum
};

// A row's position and what it sees of its sequence.
__device__ __forceinline__ int length(const Args &a, int s) {
    return max(0, min(min(a.lens[s], a.max_len), a.maxp * rows::PAGE));
}

// QKNorm, rotation at pos and scale of a row's elements x[ks][e] = element
// STEP ks + off + e (STEP 16 or 32 wide steps, off: the lane's), in fp32; the
// rotation's partner, half a head away, is in the same lane.
template <int D, int STEP>
__device__ __forceinline__ void finish_q(float (&x)[D / STEP][8], int off, const float *gain, float eps,
                                         const float *cs, const float *sn, float scale) {
    constexpr int N = D / STEP;
    if (gain) {
        float ss = 0.0f;
#pragma unroll
        for (int ks = 0; ks < N; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[ks][e], x[ks][e], ss);
        if constexpr (STEP == 32) ss += __shfl_xor(ss, 16, 64);
        ss += __shfl_xor(ss, 32, 64);
        scale *= *gain / sqrtf(fmaxf(ss / (float)D, eps));
    }
#pragma unroll
    for (int ks = 0; ks < N; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[ks][e] *= scale;
    if (cs) {
#pragma unroll
        for (int ks = 0; ks < N / 2; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = STEP * ks + off + e;
                const float lo = x[ks][e], hi = x[ks + N / 2][e];
                x[ks][e] = lo * cs[t] - hi * sn[t];
                x[ks + N / 2][e] = hi * cs[t + D / 2] + lo * sn[t + D / 2];
            }
    }
}

// x as an operand, and what its rounding left (bf16).
template <int DT>
__device__ __forceinline__ void split(const float (&x)[8], typename Op<DT>::F &hi, typename Op<DT>::F &lo) {
    hi = Op<DT>::pack(x);
    float h[8], r[8];
    Op<DT>::unpack(hi, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e] - h[e];
    lo = Op<DT>::pack(r);
}

// ------------------------------------------------------------------ decode ----
template <int DT> struct Mma16;
template <> struct Mma16<1> {
    static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mma16<0> {   // eight 4-deep steps: in step e lane group lg supplies element 8 lg + e
    static __device__ __forceinline__ f32x4 mma(rows::f32x8 a, rows::f32x8 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

constexpr int DW = 4;   // waves of a decode workgroup

// Which pages of its sequence the newest token sees: page i of the list is
// i < ns ? i : w0 + i - ns (sinks, then the window or everything from `shared`).
struct Pages {
    int n, ns, w0, lo, L;
};
__device__ __forceinline__ Pages page_list(const Args &a, int L) {
    Pages p;
    p.L = L;
    p.lo = a.W > 0 ? max(0, L - a.W) : a.shared * rows::PAGE;
    p.n = rows::tile_list<rows::PAGE>(p.lo, L, a.W > 0 ? a.S : 0, p.ns, p.w0);
    return p;
}

// blockIdx.x: (sequence, KV head, 16 of its heads); blockIdx.y: part.  Units of
// UK keys: a page, or half of one where a page's operands would fill the
// registers.
template <int DT, int D, int UK> __global__ __launch_bounds__(64 * DW) void decode_kernel(const Args a) {
    typedef typename Op<DT>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, NKS = D / 32, NDT = D / 16, NH = UK / 32, UP = rows::PAGE / UK;
    __shared__ float so[DW][16][D + 4];
    __shared__ float sm[DW][16], sl[DW][16];
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ct = (a.G + 15) / 16;
    const int s = blockIdx.x / (a.Hkv * ct), g = blockIdx.x / ct % a.Hkv, c0 = blockIdx.x % ct * 16;
    const int L = length(a, s);
    const Pages pg = page_list(a, L);
    const int u0 = blockIdx.y * a.part * UP, u1 = min(pg.n, (int)(blockIdx.y + 1) * a.part) * UP;
    const int hl = c0 + l16, head = g * a.G + min(hl, a.G - 1);

    F qh[NKS], ql[NKS];
    {
        float x[NKS][8];
        const char *row = a.q + (int64_t)s * a.qst + head * a.qsh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) Op<DT>::unpack(Op<DT>::load(row + (32 * ks + 8 * lg) * ESZ), x[ks]);
        const int64_t pos = max((int64_t)0, min((int64_t)L - 1, a.n_tab - 1)) * D;
        finish_q<D, 32>(x, 8 * lg, a.gain ? a.gain + head : nullptr, a.eps, a.cos ? a.cos + pos : nullptr,
                        a.sin ? a.sin + pos : nullptr, a.scales[s] * LOG2E);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) split<DT>(x[ks], qh[ks], ql[ks]);
    }
    const char *kb = a.kr + (int64_t)g * rows::PAGE * D * ESZ, *vb = a.v + (int64_t)g * rows::PAGE * D * ESZ;
    const int64_t pstep = (int64_t)a.Hkv * rows::PAGE * D * ESZ;
    const int32_t *table = a.table + (int64_t)s * a.maxp;
    f32x4 O[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int u = u0 + wave; u < u1; u += DW) {
        const int i = u / UP, h0 = UP == 1 ? 0 : u % UP, pl = i < pg.ns ? i : pg.w0 + i - pg.ns;
        const int64_t id = max((int64_t)0, min((int64_t)table[pl], a.pages - 1));
        const char *kp = kb + id * pstep, *vp = vb + id * pstep;
        const int j0 = pl * rows::PAGE + 32 * h0;
        F kf[2 * NH][NKS], vf[NDT][NH];
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
                kf[mt][ks] = Op<DT>::load(kp + (((2 * h0 + mt) * NKS + ks) * 64 + lane) * 8 * ESZ);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int h = 0; h < NH; ++h) vf[dt][h] = Op<DT>::load(vp + ((dt * 2 + h0 + h) * 64 + lane) * 8 * ESZ);
        f32x4 S[2 * NH];
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt) {
            S[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                S[mt] = Mma16<DT>::mma(kf[mt][ks], qh[ks], S[mt]);
                if constexpr (DT == 1) S[mt] = Mma16<DT>::mma(kf[mt][ks], ql[ks], S[mt]);
            }
        }
        // S[mt][e]: key j0 + 32 (mt / 2) + 8 lg + 4 (mt % 2) + e
        const bool whole = j0 + UK <= L && (j0 >= pg.lo || j0 + UK <= a.S);
        if (!whole) {   // the keys that are not seen: no weight, and no value (it may be anything)
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                bool see[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = j0 + 32 * h + 8 * lg + e;
                    see[e] = j < L && (j >= pg.lo || j < a.S);
                    if (!see[e]) S[2 * h + (e >> 2)][e & 3] = -INFINITY;
                }
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    float x[8];
                    Op<DT>::unpack(vf[dt][h], x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = see[e] ? x[e] : 0.0f;
                    vf[dt][h] = Op<DT>::pack(x);
                }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, S[mt][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__ballot(mx > m)) {
            const float mn = fmaxf(m, mx), al = m == -INFINITY ? 0.0f : ex2(m - mn);
            l *= al;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt] = O[dt] * al;
            m = mn;
        }
        const float mc = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = ex2(S[2 * h + (e >> 2)][e & 3] - mc);
                l += p[e];
            }
            const F pf = Op<DT>::pack(p);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt] = Mma16<DT>::mma(vf[dt][h], pf, O[dt]);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lg == 0) {
        sm[wave][l16] = m;
        sl[wave][l16] = l;
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4 *>(&so[wave][l16][16 * dt + 4 * lg]) = O[dt];
    __syncthreads();
    // the waves' parts: thread (head, 4 elements)
    for (int x = threadIdx.x; x < 16 * D / 4; x += 64 * DW) {
        const int hc = x / (D / 4), e = x % (D / 4) * 4;
        if (c0 + hc >= a.G) break;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < DW; ++w) mm = fmaxf(mm, sm[w][hc]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float ll = 0.0f;
#pragma unroll
        for (int w = 0; w < DW; ++w) {
            const float f = sm[w][hc] == -INFINITY ? 0.0f : ex2(sm[w][hc] - mm);
            // a wave without keys has zeros; one whose scores are all -inf as well
            ll = fmaf(sl[w][hc], f, ll);
            o = o + *reinterpret_cast<const f32x4 *>(&so[w][hc][e]) * f;
        }
        const int64_t row = (int64_t)s * a.Hq + g * a.G + c0 + hc;
        if (a.slots == 1) {
            // nothing seen: 0; keys whose scores are all -inf: NaN, as a softmax of them
            const f32x4 r = L > 0 ? o / ll : f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (DT == 1)
                *reinterpret_cast<uint2 *>(a.out + (row * D + e) * 2) =
                    make_uint2(pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3]));
            else
                *reinterpret_cast<f32x4 *>(a.out + (row * D + e) * 4) = r;
        } else {
            const int64_t at = row * a.slots + a.slot0 + blockIdx.y;
            *reinterpret_cast<f32x4 *>(a.po + at * D + e) = o;
            if (e == 0) {
                a.pml[2 * at] = mm;
                a.pml[2 * at + 1] = ll;
            }
        }
    }
}

// -------------------------------------------------------------------- rows ----
// SHARED: the rows of all tokens over the shared pages (blockIdx.x: 128-row
// tile); else the rows of one sequence's tokens over its own pages (blockIdx.x:
// tile of the ragged batch).  blockIdx.y: KV head, blockIdx.z: part of the tiles.
template <int DT, int D, bool SHARED> __global__ __launch_bounds__(64 * rows::NW, (DT == 1 && D == 64 ? 3 : rows::WAVES<DT, D>)) void rows_kernel(const Args a) {
    extern __shared__ __align__(16) char smem[];
    typedef typename Op<DT>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, NKS = D / 16;
    constexpr bool LO = DT == 1;
    const int lane = threadIdx.x & 63, hf = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = blockIdx.y;
    int s = 0, tile = blockIdx.x, first = 0, cnt = a.T;
    if constexpr (!SHARED) {
        s = ragged::find(blockIdx.x, a.Bd, [&](int i) {
            int f;
            return (ragged::tokens(a.cu, i, a.T, f) * a.G + rows::RT - 1) / rows::RT;
        }, tile);
        if (s < 0) return;
        cnt = ragged::tokens(a.cu, s, a.T, first);
    }
    const int nr = cnt * a.G, r0 = tile * rows::RT, rw = r0 + wave * rows::RW, r = rw + (lane & 31);
    const bool in = r < nr;
    const int t = first + min(r, nr - 1) / a.G, head = g * a.G + min(r, nr - 1) % a.G;
    const int sq = SHARED ? (a.cu ? ragged::sequence(a.cu, a.Bd, t) : t) : s;
    const int L = length(a, sq);
    int sfirst = t, scnt = 1;
    if (a.cu) scnt = ragged::tokens(a.cu, sq, a.T, sfirst);
    const int pos = L - scnt + t - sfirst;       // < 0: the token is behind what the cache holds
    rows::Sees w;
    w.S = a.W > 0 ? a.S : 0;
    w.hi = in && pos >= 0 ? pos + 1 : 0;
    w.lo = a.W > 0 ? max(0, pos + 1 - a.W) : 0;
    if constexpr (SHARED) w.hi = min(w.hi, a.shared * rows::PAGE);
    else if (a.shared) w.lo = a.shared * rows::PAGE;
    // the wave's and the workgroup's bounds, over the rows that see anything
    int v[4] = {w.hi ? w.lo : 0x7fffffff, w.hi ? w.lo : 0, in ? w.hi : 0x7fffffff, w.hi};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        v[0] = min(v[0], __shfl_xor(v[0], o, 64));
        v[1] = max(v[1], __shfl_xor(v[1], o, 64));
        v[2] = min(v[2], __shfl_xor(v[2], o, 64));
        v[3] = max(v[3], __shfl_xor(v[3], o, 64));
    }
    w.lo_min = __builtin_amdgcn_readfirstlane(v[0]);
    w.lo_max = __builtin_amdgcn_readfirstlane(v[1]);
    w.hi_min = __builtin_amdgcn_readfirstlane(v[2]);
    w.hi_max = __builtin_amdgcn_readfirstlane(v[3]);
    __shared__ int bounds[rows::NW][2];
    if (lane == 0) {
        bounds[wave][0] = w.lo_min;
        bounds[wave][1] = w.hi_max;
    }
    __syncthreads();
    int lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int i = 0; i < rows::NW; ++i) {
        lo = min(lo, bounds[i][0]);
        hi = max(hi, bounds[i][1]);
    }
    int ns = 0, wt0 = 0;
    const int nt = hi > 0 ? rows::tile_list<rows::KEYS<DT, D>>(lo, hi, w.S, ns, wt0) : 0;
    constexpr int TP = rows::PAGE / rows::KEYS<DT, D>;   // tiles of a page
    const int z = blockIdx.z, it0 = z * a.part * TP, it1 = min(nt, it0 + a.part * TP);
    const int64_t row = (int64_t)t * a.Hq + head, at = row * a.slots + a.slot0 + z;
    if (it0 >= it1 && a.slots > 1) {   // nothing of the row's keys in this part
        if (in && hf == 0) {
            a.pml[2 * at] = -INFINITY;
            a.pml[2 * at + 1] = 0.0f;
        }
        return;
    }

    F qh[NKS], ql[NKS];
    {
        float x[NKS][8];
        const char *row = a.q + (int64_t)t * a.qst + head * a.qsh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) Op<DT>::unpack(Op<DT>::load(row + (16 * ks + 8 * hf) * ESZ), x[ks]);
        const int64_t turn = max((int64_t)0, min((int64_t)pos, a.n_tab - 1)) * D;
        finish_q<D, 16>(x, 8 * hf, a.gain ? a.gain + head : nullptr, a.eps, a.cos ? a.cos + turn : nullptr,
                        a.sin ? a.sin + turn : nullptr, a.scales[sq] * LOG2E);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) split<DT>(x[ks], qh[ks], ql[ks]);
    }
    rows::PageKV<DT, D> src;
    src.page = (int64_t)a.Hkv * rows::PAGE * D * ESZ;
    src.k = a.kr + (int64_t)g * rows::PAGE * D * ESZ;
    src.v = a.v + (int64_t)g * rows::PAGE * D * ESZ;
    src.table = a.table + (SHARED ? 0 : (int64_t)s * a.maxp);
    src.pages = a.pages;
    rows::RowAcc<DT, D> acc;
    rows::attend<DT, D, LO>(src, smem, qh, ql, 1.0f, it0, it1, ns, wt0, w, acc);
    float l = acc.l + rows::other_half(acc.l);
    const bool valid = w.hi > 0;
    if (__ballot(valid && (rows::any_bad<D>(acc.O) || !rows::finite(l)))) {
        rows::attend_each<DT, D, LO>(src, qh, ql, 1.0f, it0, it1, ns, wt0, w, acc);
        l = acc.l + rows::other_half(acc.l);
    }
    if (!in) return;
    if (!valid) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc.O[dt][e] = 0.0f;
        acc.m = -INFINITY;
        l = 0.0f;
    }
    if (a.slots == 1) {
        rows::store_rows<DT, D>(a.out + row * D * ESZ, acc.O, valid ? 1.0f / l : 0.0f);
    } else {
        rows::store_rows<0, D>(reinterpret_cast<char *>(a.po + at * D), acc.O, 1.0f);
        if (hf == 0) {
            a.pml[2 * at] = acc.m;
            a.pml[2 * at + 1] = l;
        }
    }
}

// out = sum of the parts' O 2^(m - max) over sum of their l 2^(m - max); a row
// without keys 0.  D / 4 threads a part, SG parts of a row at a time (all of a
// workgroup where a row has many parts, one where rows are many), each with sums
// of its own that LDS joins.
template <int DT, int D, int SG> __global__ __launch_bounds__(256) void join_kernel(const Args a, int64_t nrows) {
    constexpr int TP = D / 4, RB = 256 / (TP * SG);   // threads of a part, rows of a workgroup
    __shared__ float so[SG > 1 ? SG : 1][SG > 1 ? D : 1];
    __shared__ float sm[SG], sl[SG];
    const int x = threadIdx.x % TP * 4, sg = threadIdx.x / TP % SG;
    const int64_t row = (int64_t)blockIdx.x * RB + threadIdx.x / (TP * SG);
    if (row >= nrows) return;                         // SG > 1: the workgroup's one row
    const float *ml = a.pml + row * a.slots * 2, *po = a.po + row * a.slots * D + x;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    for (int i = sg; i < a.slots; i += 4 * SG) {      // four parts at a time
        float pm[4], pl[4];
        f32x4 px[4];
        float mn = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = min(i + e * SG, a.slots - 1);
            const bool in = i + e * SG < a.slots;
            pm[e] = in ? ml[2 * p] : -INFINITY;
            pl[e] = in ? ml[2 * p + 1] : 0.0f;
            px[e] = *reinterpret_cast<const f32x4 *>(po + (int64_t)p * D);
            mn = fmaxf(mn, pm[e]);
        }
        const float al = m == -INFINITY ? 0.0f : ex2(m - mn);
        l *= al;
        o = o * al;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (pm[e] == -INFINITY && pl[e] == 0.0f) continue;   // no keys here, or none that counts
            const float f = ex2(pm[e] - mn);
            l = fmaf(pl[e], f, l);
            o = o + px[e] * f;
        }
        m = mn;
    }
    if constexpr (SG > 1) {
        *reinterpret_cast<f32x4 *>(&so[sg][x]) = o;
        if (x == 0) {
            sm[sg] = m;
            sl[sg] = l;
        }
        __syncthreads();
        if (sg) return;
        float mm = -INFINITY;
#pragma unroll
        for (int i = 0; i < SG; ++i) mm = fmaxf(mm, sm[i]);
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < SG; ++i) {
            if (sm[i] == -INFINITY && sl[i] == 0.0f) continue;
            const float f = ex2(sm[i] - mm);
            l = fmaf(sl[i], f, l);
            o = o + *reinterpret_cast<const f32x4 *>(&so[i][x]) * f;
        }
    }
    // what the row sees: nothing gives 0, scores that are all -inf NaN
    const int t = (int)(row / a.Hq), s = a.cu ? ragged::sequence(a.cu, a.Bd, t) : t;
    int first = t, cnt = 1;
    if (a.cu) cnt = ragged::tokens(a.cu, s, a.T, first);
    const f32x4 r = length(a, s) - cnt + t - first >= 0 ? o / l : f32x4{0.f, 0.f, 0.f, 0.f};
    char *to = a.out + (row * D + x) * (DT == 1 ? 2 : 4);
    if constexpr (DT == 1)
        *reinterpret_cast<uint2 *>(to) = make_uint2(pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3]));
    else
        *reinterpret_cast<f32x4 *>(to) = r;
}

// ------------------------------------------------------------------- plan ----
// How the rows' keys are cut into parts: runs of pages, so that long sequences have
// more of them than short ones.
struct Plan {
    int prefix, own;              // parts over the shared pages, and over each sequence's own, at most
    int prefix_pages, own_pages;  // pages of one
    int64_t tiles, ptiles;        // 128-row tiles: of the ragged batch (at most), of all tokens
    int slots() const { return prefix + own; }
};
#ifndef AIMR
#define AIMR 1024
#endif
#ifndef AIMP
#define AIMP 512
#endif
#ifndef MINP
#define MINP 4
#endif
static int parts_of(int64_t pages, int64_t parts, int64_t least, int &per) {
    if (parts > pages / least) parts = pages / least;
    if (parts < 1) parts = 1;
    per = (int)((pages + parts - 1) / parts);
    return (int)((pages + per - 1) / per);
}
static Plan plan(int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t W, int64_t S, int64_t shared, bool one,
                 int64_t max_len) {
    Plan p = {};
    const int64_t G = Hq / Hkv, KT = rows::PAGE;
    int64_t keys = max_len - shared * KT;
    if (W > 0 && W < keys) keys = W;
    if (W > 0 && !one) keys = max_len;   // a part of a prompt may span any number of windows
    if (keys < 1) keys = 1;
    int64_t pages = (keys + KT - 1) / KT + 1 + (W > 0 ? (S + KT - 1) / KT : 0);
    const int64_t all = (max_len + KT - 1) / KT;
    if (pages > all) pages = all > 0 ? all : 1;
    p.ptiles = (T * G + rows::RT - 1) / rows::RT;
    if (one) {
        const int64_t groups = Bd * Hkv * ((G + 15) / 16);
        p.own = parts_of(pages, (2048 + groups - 1) / groups, 4, p.own_pages);
    } else {
        p.tiles = p.ptiles + Bd;
        p.own = parts_of(pages, AIMR / (p.ptiles * Hkv), 8, p.own_pages);
    }
    if (shared) p.prefix = parts_of(shared, AIMP / (p.ptiles * Hkv), MINP, p.prefix_pages);
    return p;
}

template <class K> static int lds_room(K kern, size_t bytes) {
    if (bytes <= 65536) return HBA_OK;
    return hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)bytes) == hipSuccess
               ? HBA_OK
               : HBA_ERR_LAUNCH;
}

template <int DT, int D> static int launch(Args a, const Plan &p, hipStream_t s) {
    constexpr size_t lds = 2 * rows::PageKV<DT, D>::BYTES;
    constexpr int UK = DT == 1 && D == 64 ? 64 : 32;
    a.slots = p.slots();
    if (p.prefix) {
        a.slot0 = 0;
        a.part = p.prefix_pages;
        if (int st = lds_room(rows_kernel<DT, D, true>, lds)) return st;
        hipLaunchKernelGGL((rows_kernel<DT, D, true>), dim3((unsigned)p.ptiles, (unsigned)a.Hkv, (unsigned)p.prefix),
                           dim3(64 * rows::NW), lds, s, a);
        HBA_LAUNCH_CHECK();
    }
    a.slot0 = p.prefix;
    if (a.cu) {
        a.part = p.own_pages;
        if (int st = lds_room(rows_kernel<DT, D, false>, lds)) return st;
        hipLaunchKernelGGL((rows_kernel<DT, D, false>), dim3((unsigned)p.tiles, (unsigned)a.Hkv, (unsigned)p.own),
                           dim3(64 * rows::NW), lds, s, a);
    } else {
        a.part = p.own_pages;
        const int64_t groups = (int64_t)a.Bd * a.Hkv * ((a.G + 15) / 16);
        hipLaunchKernelGGL((decode_kernel<DT, D, UK>), dim3((unsigned)groups, (unsigned)p.own), dim3(64 * DW), 0, s, a);
    }
    HBA_LAUNCH_CHECK();
    if (a.slots > 1) {
        const int64_t nrows = (int64_t)a.T * a.Hq;
        constexpr int SG = 1024 / D, RB = 1024 / D;   // parts at a time, or rows
        if (a.slots > 8)
            hipLaunchKernelGGL((join_kernel<DT, D, SG>), dim3((unsigned)nrows), dim3(256), 0, s, a, nrows);
        else
            hipLaunchKernelGGL((join_kernel<DT, D, 1>), dim3((unsigned)((nrows + RB - 1) / RB)), dim3(256), 0, s, a,
                               nrows);
        HBA_LAUNCH_CHECK();
    }
    return HBA_OK;
}

static int check(int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, int64_t W, int64_t S, int64_t shared,
                 int one, int64_t max_len, int64_t max_pages) {
    if (d != 64 && d != 128) return HBA_ERR_UNSUPPORTED;
    if (T <= 0 || Bd <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || W < 0 || S < 0 || shared < 0 || max_len <= 0 ||
        max_pages <= 0)
        return HBA_ERR_INVALID_ARG;
    if (W > 0 && shared > 0) return HBA_ERR_INVALID_ARG;   // a window past the prefix would not see it
    if (one && T != Bd) return HBA_ERR_INVALID_ARG;
    if (max_len > (1 << 30) || max_pages > (1 << 24) || shared > max_pages || T * Hq > (1 << 30) || Hkv > 65535 ||
        Bd * Hkv * (Hq / Hkv + 16) > 0x7fffffff)
        return HBA_ERR_UNSUPPORTED;
    return HBA_OK;
}

}  // namespace paged
}  // namespace hba

using namespace hba;

extern "C" int hba_paged_attn_workspace_bytes(int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                                              int64_t S, int64_t shared_pages, int one_each, int64_t max_len,
                                              size_t *bytes) {
    if (!bytes) return HBA_ERR_INVALID_ARG;
    if (int st = paged::check(T, Bd, Hq, Hkv, d, W, S, shared_pages, one_each, max_len, 1 << 24)) return st;
    const paged::Plan p = paged::plan(T, Bd, Hq, Hkv, W, S, shared_pages, one_each != 0, max_len);
    *bytes = p.slots() > 1 ? (size_t)(T * Hq) * p.slots() * (d + 2) * 4 : 0;
    return HBA_OK;
}

extern "C" int hba_paged_attn(int dtype, const void *q, const int64_t q_strides[2], const float *q_gain, float eps,
                              const float *cos_tab, const float *sin_tab, int64_t n_tab, const void *kr_pages,
                              const void *v_pages, int64_t num_pages, const int32_t *page_table, int64_t max_pages,
                              const int32_t *seq_lens, const float *scales, const int32_t *cu, int64_t T, int64_t Bd,
                              int64_t Hq, int64_t Hkv, int64_t d, int64_t Bk, int64_t W, int64_t S,
                              int64_t shared_pages, int64_t max_len, void *workspace, size_t ws_bytes, void *out,
                              void *stream) {
    if (int st = abi::check_dtype_dim(dtype, d)) return st;
    if (Bk != rows::PAGE) return HBA_ERR_UNSUPPORTED;
    if (int st = paged::check(T, Bd, Hq, Hkv, d, W, S, shared_pages, cu == nullptr, max_len, max_pages)) return st;
    if (!q || !q_strides || !kr_pages || !v_pages || !page_table || !seq_lens || !scales || !out || num_pages <= 0 ||
        !cos_tab != !sin_tab || (cos_tab && n_tab <= 0))
        return HBA_ERR_INVALID_ARG;
    const int64_t e = abi::elem_size(dtype), al = 16 / e;
    if (!abi::aligned16(q) || q_strides[0] % al || q_strides[1] % al || !abi::aligned16(kr_pages) ||
        !abi::aligned16(v_pages) || !abi::aligned16(out))
        return HBA_ERR_UNSUPPORTED;
    const paged::Plan p = paged::plan(T, Bd, Hq, Hkv, W, S, shared_pages, cu == nullptr, max_len);
    const size_t need = p.slots() > 1 ? (size_t)(T * Hq) * p.slots() * (d + 2) * 4 : 0;
    if (need && (!workspace || ws_bytes < need)) return HBA_ERR_INVALID_ARG;
    if (need && !abi::aligned16(workspace)) return HBA_ERR_UNSUPPORTED;
    paged::Args a = {};
    a.q = (const char *)q;
    a.qst = q_strides[0] * e;
    a.qsh = q_strides[1] * e;
    a.gain = q_gain;
    a.eps = eps;
    a.cos = cos_tab;
    a.sin = sin_tab;
    a.n_tab = cos_tab ? n_tab : 1;
    a.kr = (const char *)kr_pages;
    a.v = (const char *)v_pages;
    a.pages = num_pages;
    a.table = page_table;
    a.lens = seq_lens;
    a.cu = cu;
    a.scales = scales;
    a.T = (int)T;
    a.Bd = (int)Bd;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.G = (int)(Hq / Hkv);
    a.maxp = (int)max_pages;
    a.max_len = (int)max_len;
    a.W = (int)(W < (1 << 30) ? W : (1 << 30));
    a.S = (int)(S < (1 << 30) ? S : (1 << 30));
    a.shared = (int)shared_pages;
    a.out = (char *)out;
    a.po = (float *)workspace;
    a.pml = need ? (float *)workspace + T * Hq * p.slots() * d : nullptr;
    int st = HBA_OK;
#define HBA_PAGED(DT, D) st = paged::launch<DT, D>(a, p, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PAGED);
#undef HBA_PAGED
    return st;
}
