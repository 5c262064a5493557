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
//   decode_part    one token per sequence: memory-bound.  A wave takes a page of
//                  one KV head in operand order straight into registers (its
//                  heads are the 16 columns), the next one's loads in flight.
//                  Long sequences' pages are one list that the workgroups share
//                  evenly (even_kernel).
//   rows_part      128 rows (token, head) a workgroup over staged pages
//                  (hba_rows.h): parts of prompts, and the shared pages for the
//                  rows of the whole batch.
//   join_kernel    the parts of a row, by their maxima and sums.
//
// With shared pages, both parts of the work are one launch (shared_kernel): neither
// fills the card alone.
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
    int slots, slot0, part;             // parts of a row: how many, the first of these, pages of one of them
    char *out;                          // [T, Hq, D]
    // parts: [T, Hq, slots, D] sums, [T, Hq, slots, 2] maximum (log2 units) and sum; of even shares (slots of
    // them, part pages at least): [slots, 2, 16, D] and [slots, 2, 16, 2], see even_kernel
    float *po, *pml;
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

// gi: 16 heads of a KV head of sequence s; pages p0 .. p1 - 1 of its list.  Head i of
// the 16 writes part at + i step, or its row of the output (at < 0).
// Units of UK keys: a page, or half of one where a page's operands would fill the
// registers.  DW waves take the pages' units in turn.
template <int DT, int D> constexpr int UNIT = DT == 1 && D == 64 ? 64 : 32;
template <int D> struct DecodeLds {
    float o[4][16][D + 4], m[4][16], l[4][16];
};
template <int DT, int D, int DW>
__device__ __forceinline__ void decode_part(const Args &a, DecodeLds<D> &lds, int s, int gi, int p0, int p1,
                                            int64_t at, int step) {
    typedef typename Op<DT>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, UK = UNIT<DT, D>;
    constexpr int NKS = D / 32, NDT = D / 16, NH = UK / 32, UP = rows::PAGE / UK;
    typedef const __attribute__((address_space(4))) int32_t *uniform;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ct = (a.G + 15) / 16;
    const int g = gi / ct, c0 = gi % ct * 16;
    const int L = length(a, s);
    const Pages pg = page_list(a, L);
    const int u0 = p0 * UP, u1 = min(pg.n, p1) * UP;
    const int hl = c0 + l16, head = g * a.G + min(hl, a.G - 1);
    const char *kb = a.kr + (int64_t)g * rows::PAGE * D * ESZ, *vb = a.v + (int64_t)g * rows::PAGE * D * ESZ;
    const int64_t pstep = (int64_t)a.Hkv * rows::PAGE * D * ESZ;
    const uniform table = (uniform)(uintptr_t)(a.table + (int64_t)s * a.maxp);

    struct Unit {
        F k[2 * NH][NKS], v[NDT][NH];
    };
    // the logical page of unit u (the last one past the end), its place in the cache
    const auto logical = [&](int u) {
        const int i = min(u, u1 - 1) / UP;
        return i < pg.ns ? i : pg.w0 + i - pg.ns;
    };
    const auto place = [&](int u) { return max((int64_t)0, min((int64_t)table[logical(u)], a.pages - 1)); };
    const auto load = [&](Unit &x, int u, int64_t id) {
        const int h0 = UP == 1 ? 0 : u % UP;
        const char *kp = kb + id * pstep, *vp = vb + id * pstep;
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
                x.k[mt][ks] = Op<DT>::load(kp + (((2 * h0 + mt) * NKS + ks) * 64 + lane) * 8 * ESZ);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int h = 0; h < NH; ++h) x.v[dt][h] = Op<DT>::load(vp + ((dt * 2 + h0 + h) * 64 + lane) * 8 * ESZ);
    };
    int u = u0 + wave;
    Unit xa;
    int64_t next = 0;   // the place of unit u + DW
    if (u < u1) {
        load(xa, u, place(u));
        next = place(u + DW);
    }

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
    f32x4 O[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    const auto use = [&](Unit &x, int at) {
        const int j0 = logical(at) * rows::PAGE + (UP == 1 ? 0 : at % UP * UK);
        f32x4 S[2 * NH];
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt) {
            S[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                S[mt] = Mma16<DT>::mma(x.k[mt][ks], qh[ks], S[mt]);
                if constexpr (DT == 1) S[mt] = Mma16<DT>::mma(x.k[mt][ks], ql[ks], S[mt]);
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
                    float y[8];
                    Op<DT>::unpack(x.v[dt][h], y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = see[e] ? y[e] : 0.0f;
                    x.v[dt][h] = Op<DT>::pack(y);
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
            const F pf = Op<DT>::pack(p);   // bf16: a relative 2^-8 each at most; l has them as they are
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt] = Mma16<DT>::mma(x.v[dt][h], pf, O[dt]);
        }
    };
    if constexpr (DT == 0 && D == 128) {   // two units would fill the registers
#pragma unroll 1
        for (; u < u1; u += DW) {
            use(xa, u);
            if (u + DW >= u1) break;
            load(xa, u + DW, next);
            next = place(u + 2 * DW);
        }
    } else {
        Unit xb;
#pragma unroll 1
        for (; u < u1; u += 2 * DW) {
            if (u + DW < u1) {
                load(xb, u + DW, next);
                next = place(u + 2 * DW);
            }
            use(xa, u);
            if (u + DW >= u1) break;
            if (u + 2 * DW < u1) {
                load(xa, u + 2 * DW, next);
                next = place(u + 3 * DW);
            }
            use(xb, u + DW);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // the waves' sums meet in LDS: those of waves 4 and up fold into the first four's
    const auto put = [&](int w) {
        if (lg == 0) {
            lds.m[w][l16] = m;
            lds.l[w][l16] = l;
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4 *>(&lds.o[w][l16][16 * dt + 4 * lg]) = O[dt];
    };
    if constexpr (DW > 4) {
        if (wave >= 4) put(wave - 4);
        __syncthreads();
        if (wave < 4) {
            const float om = lds.m[wave][l16], ol = lds.l[wave][l16], mn = fmaxf(m, om);
            const float fa = m == -INFINITY ? 0.0f : ex2(m - mn), fb = om == -INFINITY ? 0.0f : ex2(om - mn);
            l = fmaf(ol, fb, l * fa);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                O[dt] = O[dt] * fa + *reinterpret_cast<const f32x4 *>(&lds.o[wave][l16][16 * dt + 4 * lg]) * fb;
            m = mn;
        }
    }
    if (wave < 4) put(wave);   // its own place: nobody else has read it
    __syncthreads();
    // thread (head, 4 elements)
    for (int x = threadIdx.x; x < 16 * D / 4; x += 64 * DW) {
        const int hc = x / (D / 4), e = x % (D / 4) * 4;
        if (c0 + hc >= a.G) break;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, lds.m[w][hc]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float ll = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            // a wave without keys, or with scores that are all -inf, has zeros
            const float f = lds.m[w][hc] == -INFINITY ? 0.0f : ex2(lds.m[w][hc] - mm);
            ll = fmaf(lds.l[w][hc], f, ll);
            o = o + *reinterpret_cast<const f32x4 *>(&lds.o[w][hc][e]) * f;
        }
        const int64_t row = (int64_t)s * a.Hq + g * a.G + c0 + hc;
        if (at < 0) {
            // nothing seen: 0; keys whose scores are all -inf: NaN, as a softmax of them
            const f32x4 r = L > 0 ? o / ll : f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (DT == 1)
                *reinterpret_cast<uint2 *>(a.out + (row * D + e) * 2) =
                    make_uint2(pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3]));
            else
                *reinterpret_cast<f32x4 *>(a.out + (row * D + e) * 4) = r;
        } else {
            const int64_t to = at + (int64_t)hc * step;
            *reinterpret_cast<f32x4 *>(a.po + to * D + e) = o;
            if (e == 0) {
                a.pml[2 * to] = mm;
                a.pml[2 * to + 1] = ll;
            }
        }
    }
}

constexpr int DW = 8;   // waves of a decode workgroup
// group: (sequence, KV head, 16 of its heads), part: a run of a.part pages.
// 64 sequences' windows of 1024 keys, 14 / 2 heads, d = 64: 11 us, 7 at a copy's rate.
// Eight waves, so that a window of 17 or 18 pages takes a wave two pages, or three:
// chains of round trips bound it.
template <int DT, int D, int DW>
__device__ __forceinline__ void decode_run(const Args &a, DecodeLds<D> &lds, int group, int part) {
    const int ct = (a.G + 15) / 16, ng = a.Hkv * ct, s = group / ng, gi = group % ng;
    const int64_t row = (int64_t)s * a.Hq + gi / ct * a.G + gi % ct * 16;
    decode_part<DT, D, DW>(a, lds, s, gi, part * a.part, (part + 1) * a.part,
                           a.slots == 1 ? -1 : row * a.slots + a.slot0 + part, a.slots);
}
template <int DT, int D> __global__ __launch_bounds__(64 * DW) void decode_kernel(const Args a) {
    __shared__ DecodeLds<D> lds;
    decode_run<DT, D, DW>(a, lds, blockIdx.x, blockIdx.y);
}

// Even shares.  All pages of all groups (a group: 16 heads of a sequence) make one
// list, in the order of sequences; workgroup w takes share w of it, whatever the
// sequences' lengths.  A group inside one share is written at once; of the others
// a share holds two at most, one that began before it (or with it) and one that
// ends after it: parts 2 w and 2 w + 1.
struct Shares {
    int units, per;   // pages of all groups, of one share
};
__device__ __forceinline__ int list_pages(const Args &a, int s) { return max(1, page_list(a, length(a, s)).n); }
__device__ __forceinline__ int groups_of(const Args &a) { return a.Hkv * ((a.G + 15) / 16); }
template <int NT> __device__ __forceinline__ Shares shares(const Args &a) {
    Shares x;
    x.units = ragged::total<NT>(a.Bd, [&](int s) { return list_pages(a, s); }) * groups_of(a);
    x.per = max(a.part, (x.units + a.slots - 1) / a.slots);
    return x;
}
template <int DT, int D> __global__ __launch_bounds__(64 * DW) void even_kernel(const Args a) {
    __shared__ DecodeLds<D> lds;
    const Shares sh = shares<64 * DW>(a);
    const int ng = groups_of(a), w = blockIdx.x;
    const int64_t u0 = (int64_t)w * sh.per;
    if (u0 >= sh.units) return;
    int left = (int)min((int64_t)sh.per, sh.units - u0), at;
    int s = ragged::find<64 * DW>((int)u0, a.Bd, [&](int i) { return list_pages(a, i) * ng; }, at);
    for (int part = 2 * w; left > 0 && s < a.Bd; part = 2 * w + 1) {
        const int n = list_pages(a, s), p0 = at % n, p1 = min(n, p0 + left);
        decode_part<DT, D, DW>(a, lds, s, at / n, p0, p1, p1 - p0 == n ? -1 : (int64_t)part * 16, 1);
        __syncthreads();   // lds is free again
        left -= p1 - p0;
        at += p1 - p0;
        if (at == n * ng) {
            at = 0;
            ++s;
        }
    }
}

// -------------------------------------------------------------------- rows ----
// The rows, of KV head g, of tokens before cu[0] or behind cu[Bd]: 0, by workgroups
// left over (there are some: no batch fills its last Bd tiles).
template <int DT, int D> __device__ __forceinline__ void zero_strays(const Args &a, int g, int w, int of) {
    constexpr int V = DT == 1 ? 8 : 4;   // elements of 16 bytes
    const int lo = max(0, min(a.T, a.cu[0])), hi = max(lo, min(a.T, a.cu[a.Bd]));
    const int64_t n = (int64_t)(lo + a.T - hi) * a.G * (D / V), step = (int64_t)of * (64 * rows::NW);
    for (int64_t i = (int64_t)w * (64 * rows::NW) + threadIdx.x; i < n; i += step) {
        const int64_t k = i / (D / V) / a.G, t = k < lo ? k : k - lo + hi, head = g * a.G + i / (D / V) % a.G;
        *reinterpret_cast<uint4 *>(a.out + ((t * a.Hq + head) * D + i % (D / V) * V) * (16 / V)) = uint4{0, 0, 0, 0};
    }
}

// SHARED: the rows of all tokens over the shared pages (x: 128-row tile); else the
// rows of one sequence's tokens over its own pages (x: tile of the ragged batch).
// g: KV head, z: part, a run of a.part pages.
template <int DT, int D, bool SHARED>
__device__ __forceinline__ void rows_part(const Args &a, char *smem, int x, int g, int z) {
    typedef typename Op<DT>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, NKS = D / 16, KT = rows::KEYS<DT, D>, TP = rows::PAGE / KT;
    constexpr bool LO = DT == 1;
    const int lane = threadIdx.x & 63, hf = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    rows::PageKV<DT, D> src;
    src.page = (int64_t)a.Hkv * rows::PAGE * D * ESZ;
    src.k = a.kr + (int64_t)g * rows::PAGE * D * ESZ;
    src.v = a.v + (int64_t)g * rows::PAGE * D * ESZ;
    src.pages = a.pages;
    const int it0 = z * a.part * TP;
    int s = 0, tile = x, first = 0, cnt = a.T, it1 = 0, ns = 0, wt0 = 0;
    if constexpr (SHARED) {   // every tile of the part, whatever the rows see of it: it can be staged at once
        src.table = a.table;
        src.len = a.shared * rows::PAGE;
        it1 = min(a.shared * TP, it0 + a.part * TP);
        rows::attend_begin(src, smem, it0, it1, 0, 0);
    } else {
        const auto tiles = [&](int i) {
            int f;
            return (ragged::tokens(a.cu, i, a.T, f) * a.G + rows::RT - 1) / rows::RT;
        };
        s = ragged::find(x, a.Bd, tiles, tile);
        if (s < 0) {
            if (a.slots == 1) {   // else the join does it
                const int used = ragged::total<64 * rows::NW>(a.Bd, tiles);
                zero_strays<DT, D>(a, g, x - used, gridDim.x - used);
            }
            return;
        }
        cnt = ragged::tokens(a.cu, s, a.T, first);
        src.table = a.table + (int64_t)s * a.maxp;
        src.len = length(a, s);
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
    const int64_t row = (int64_t)t * a.Hq + head, at = row * a.slots + a.slot0 + z;
    if constexpr (!SHARED) {
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
        const int nt = hi > 0 ? rows::tile_list<KT>(lo, hi, w.S, ns, wt0) : 0;
        it1 = min(nt, it0 + a.part * TP);
        if (it0 >= it1 && a.slots > 1) {   // nothing of the rows' keys in this part
            if (in && hf == 0) {
                a.pml[2 * at] = -INFINITY;
                a.pml[2 * at + 1] = 0.0f;
            }
            return;
        }
        rows::attend_begin(src, smem, it0, it1, ns, wt0);
    }
    F qh[NKS], ql[NKS];
    {
        float y[NKS][8];
        const char *q = a.q + (int64_t)t * a.qst + head * a.qsh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) Op<DT>::unpack(Op<DT>::load(q + (16 * ks + 8 * hf) * ESZ), y[ks]);
        const int64_t turn = max((int64_t)0, min((int64_t)pos, a.n_tab - 1)) * D;
        finish_q<D, 16>(y, 8 * hf, a.gain ? a.gain + head : nullptr, a.eps, a.cos ? a.cos + turn : nullptr,
                        a.sin ? a.sin + turn : nullptr, a.scales[sq] * LOG2E);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) split<DT>(y[ks], qh[ks], ql[ks]);
    }
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
        for (int dt = 0; dt < D / 32; ++dt) acc.O[dt] = f32x16{0.0f};
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

// 4 sequences, 1560 new tokens behind 1300 to 8500 keys, 14 heads, d = 64, bf16: 73 us,
// 27 at the rate of a large product.  Queries of two bf16 parts double q . k (3
// products for 2), exponentials and conversions as in the sliding-window kernel.
template <int DT, int D, bool SHARED>
__global__ __launch_bounds__(64 * rows::NW, (DT == 1 && D == 64 ? 3 : rows::WAVES<DT, D>)) void rows_kernel(
    const Args a) {
    extern __shared__ __align__(16) char smem[];
    rows_part<DT, D, SHARED>(a, smem, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The shared pages for all rows (the first nshared workgroups, which take longest)
// and every sequence's own pages for its newest token: 64 sequences, 8192 shared
// keys, d = 64: 14.5 us, and 5 of the join.
template <int DT, int D>
__global__ __launch_bounds__(64 * rows::NW, (rows::WAVES<DT, D>)) void shared_kernel(
    const Args a, const Args own, int ptiles, int nshared, int groups) {
    extern __shared__ __align__(16) char smem[];
    const int i = blockIdx.x;
    if (i < nshared)
        rows_part<DT, D, true>(a, smem, i % ptiles, i / ptiles % a.Hkv, i / (ptiles * a.Hkv));
    else
        decode_run<DT, D, rows::NW>(own, *reinterpret_cast<DecodeLds<D> *>(smem), (i - nshared) % groups,
                                    (i - nshared) / groups);
}

// out = sum of the parts' O 2^(m - max) over sum of their l 2^(m - max); a row
// without keys 0.  D / 4 threads a part, SG parts of a row at a time (all of a
// workgroup where a row has many parts, one where rows are many), each with sums
// of its own that LDS joins.  EVEN: the parts are those of even shares.
template <int DT, int D, int SG, bool EVEN>
__global__ __launch_bounds__(256) void join_kernel(const Args a, int64_t nrows) {
    constexpr int TP = D / 4, RB = 256 / (TP * SG);   // threads of a part, rows of a workgroup
    __shared__ float so[SG > 1 ? SG : 1][SG > 1 ? D : 1];
    __shared__ float sm[SG], sl[SG];
    const int x = threadIdx.x % TP * 4, sg = threadIdx.x / TP % SG;
    const int64_t row = (int64_t)blockIdx.x * RB + threadIdx.x / (TP * SG);
    if (row >= nrows) return;                         // SG > 1: the workgroup's one row
    int slots = a.slots, step = 1;                    // part p at first + p step, the row's first part at part0
    int64_t first_part = row * a.slots, part0 = first_part;
    if constexpr (EVEN) {
        static_assert(RB == 1, "the scans are a workgroup's");
        const Shares sh = shares<256>(a);
        const int s = (int)(row / a.Hq), h = (int)(row % a.Hq), ct = (a.G + 15) / 16, n = list_pages(a, s);
        const int before = ragged::total<256>(s, [&](int i) { return list_pages(a, i); }) * groups_of(a);
        const int u = before + (h / a.G * ct + h % a.G / 16) * n, w0 = u / sh.per, w1 = (u + n - 1) / sh.per;
        if (w0 == w1) return;                         // written already
        slots = w1 - w0 + 1;
        step = 32;
        first_part = (int64_t)w0 * 32 + h % a.G % 16;
        part0 = first_part + (w0 * sh.per < u ? 16 : 0);
    }
    const auto place = [&](int p) { return p ? first_part + (int64_t)p * step : part0; };
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    for (int i = sg; i < slots; i += 4 * SG) {      // four parts at a time
        float pm[4], pl[4];
        f32x4 px[4];
        float mn = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t p = place(min(i + e * SG, slots - 1));
            const bool in = i + e * SG < slots;
            pm[e] = in ? a.pml[2 * p] : -INFINITY;
            pl[e] = in ? a.pml[2 * p + 1] : 0.0f;
            px[e] = *reinterpret_cast<const f32x4 *>(a.po + p * D + x);
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
    // what the row sees: nothing, or a token of no sequence, gives 0, scores that are all -inf NaN
    const int t = (int)(row / a.Hq), s = a.cu ? ragged::sequence(a.cu, a.Bd, t) : t;
    int first = t, cnt = 1;
    if (a.cu) cnt = ragged::tokens(a.cu, s, a.T, first);
    const bool sees = t >= first && t - first < cnt && length(a, s) - cnt + t - first >= 0;
    const f32x4 r = sees ? o / l : f32x4{0.f, 0.f, 0.f, 0.f};
    char *to = a.out + (row * D + x) * (DT == 1 ? 2 : 4);
    if constexpr (DT == 1)
        *reinterpret_cast<uint2 *>(to) = make_uint2(pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3]));
    else
        *reinterpret_cast<f32x4 *>(to) = r;
}

// ------------------------------------------------------------------- plan ----
// How the rows' keys are cut into parts: runs of pages, so that long sequences have
// more of them than short ones, or even shares of everything.
struct Plan {
    int prefix, own;              // parts over the shared pages, and over each sequence's own, at most
    int prefix_pages, own_pages;  // pages of one
    int shares;                   // even shares (0: parts), of own_pages at least
    int64_t tiles, ptiles;        // 128-row tiles: of the ragged batch (at most), of all tokens
    int slots() const { return prefix + own; }
};
// `base` workgroups a part: parts of one page while they find CUs of their own, then
// of `least` pages as long as there are no more than `most` workgroups.
constexpr int CUS = 256;
static int parts_of(int64_t pages, int64_t base, int64_t most, int64_t least, int &per) {
    int64_t parts = most / base < pages / least ? most / base : pages / least;
    if (parts < CUS / base) parts = CUS / base;
    if (parts > pages) parts = pages;
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
    // A part of a prompt may span any number of windows.  (The parts cut the list of one
    // 128-row tile, which has W + 128 / G tokens and the sinks, so of a window's parts most are empty.)
    if (W > 0 && !one) keys = max_len;
    if (keys < 1) keys = 1;
    int64_t pages = (keys + KT - 1) / KT + 1 + (W > 0 ? (S + KT - 1) / KT : 0);
    const int64_t all = (max_len + KT - 1) / KT;
    if (pages > all) pages = all > 0 ? all : 1;
    p.ptiles = (T * G + rows::RT - 1) / rows::RT;
    const int64_t groups = Bd * Hkv * ((G + 15) / 16);
    if (!one) {
        p.tiles = p.ptiles + Bd;
        // 4 sequences, 1560 tokens, 9000 keys, d = 64: 72 us at 1024 workgroups, 110 at 512, 77 at 1536
        p.own = parts_of(pages, p.ptiles * Hkv, 1024, 8, p.own_pages);
    } else if (shared) {
        p.own = parts_of(pages, groups, 1024, 4, p.own_pages);
    } else if (pages > 32 && groups < 1024 && groups * pages < (1 << 30)) {
        // Up to 32 pages are 4 a wave and need no join; from 1024 groups on, the card's
        // workgroups even out by themselves.  24 sequences of 4000 to 32000 keys, 4 KV
        // heads, d = 128: 155 us (5.8 TB/s), and 188 in runs of pages, 11 a sequence.
        // Lengths that are alike have less to even out.  Shares and one workgroup a group,
        // d = 64: 8 groups of 2000, 4096 and 8192 keys 13, 12, 13 and 9, 12, 20 us; 128
        // groups 21, 31, 51 and 15, 23, 40; d = 128: 16 groups 14, 15, 21 and 14, 25, 46;
        // 256 groups 51, 102, 192 and 44, 96, 187.
        p.shares = (int)(groups * pages / 8 < CUS ? groups * pages / 8 + 1 : CUS);
        p.own = 1;
        p.own_pages = 8;
    } else {
        p.own = 1;
        p.own_pages = (int)pages;
    }
    // 64 sequences' 8192 shared keys, d = 64: 14.5 us at 256 workgroups, 20 at 512, 17.5 at 128
    if (shared) p.prefix = parts_of(shared, p.ptiles * Hkv, CUS, 1, p.prefix_pages);
    return p;
}
static size_t workspace(const Plan &p, int64_t T, int64_t Hq, int64_t d) {
    const int64_t parts = p.shares ? (int64_t)p.shares * 32 : p.slots() > 1 ? T * Hq * p.slots() : 0;
    return (size_t)parts * (d + 2) * 4;
}

template <int DT, int D> static int launch(Args a, const Plan &p, hipStream_t s) {
    constexpr size_t lds = 2 * rows::PageKV<DT, D>::BYTES;
    static_assert(sizeof(DecodeLds<D>) <= 65536 && lds <= 65536, "LDS without an attribute");
    const int64_t groups = (int64_t)a.Bd * a.Hkv * ((a.G + 15) / 16);
    a.slots = p.slots();
    if (p.shares) {
        a.slots = p.shares;
        a.part = p.own_pages;
        const int64_t nrows = (int64_t)a.T * a.Hq;
        if (!abi::launchable(nrows, 256)) return HBA_ERR_UNSUPPORTED;
        hipLaunchKernelGGL((even_kernel<DT, D>), dim3((unsigned)p.shares), dim3(64 * DW), 0, s, a);
        HBA_LAUNCH_CHECK();
        hipLaunchKernelGGL((join_kernel<DT, D, 1024 / D, true>), dim3((unsigned)nrows), dim3(256), 0, s, a, nrows);
        HBA_LAUNCH_CHECK();
        return HBA_OK;
    }
    const int64_t nrows = (int64_t)a.T * a.Hq, nshared = p.ptiles * a.Hkv * p.prefix;
    constexpr int SG = 1024 / D, RB = 1024 / D;   // parts at a time, or rows, of a join's workgroup
    const int64_t joins = a.slots > 8 ? nrows : (nrows + RB - 1) / RB;
    const bool fits = a.cu ? abi::launchable(p.tiles, 64 * rows::NW)
                    : p.prefix ? abi::launchable(nshared + groups * p.own, 64 * rows::NW)
                               : abi::launchable(groups, 64 * DW);
    if (!fits || (a.slots > 1 && !abi::launchable(joins, 256)))
        return HBA_ERR_UNSUPPORTED;
    Args own = a;
    own.slot0 = p.prefix;
    own.part = p.own_pages;
    a.part = p.prefix_pages;
    if (p.prefix && !a.cu) {
        const int64_t grid = nshared + groups * p.own;
        constexpr size_t both = lds > sizeof(DecodeLds<D>) ? lds : sizeof(DecodeLds<D>);
        hipLaunchKernelGGL((shared_kernel<DT, D>), dim3((unsigned)grid), dim3(64 * rows::NW), both, s, a, own,
                           (int)p.ptiles, (int)nshared, (int)groups);
    } else {
        if (p.prefix)
            hipLaunchKernelGGL((rows_kernel<DT, D, true>),
                               dim3((unsigned)p.ptiles, (unsigned)a.Hkv, (unsigned)p.prefix), dim3(64 * rows::NW), lds,
                               s, a);
        HBA_LAUNCH_CHECK();
        if (a.cu)
            hipLaunchKernelGGL((rows_kernel<DT, D, false>), dim3((unsigned)p.tiles, (unsigned)a.Hkv, (unsigned)p.own),
                               dim3(64 * rows::NW), lds, s, own);
        else
            hipLaunchKernelGGL((decode_kernel<DT, D>), dim3((unsigned)groups, (unsigned)p.own), dim3(64 * DW), 0, s,
                               own);
    }
    HBA_LAUNCH_CHECK();
    if (a.slots > 1) {
        if (a.slots > 8)
            hipLaunchKernelGGL((join_kernel<DT, D, SG, false>), dim3((unsigned)joins), dim3(256), 0, s, a, nrows);
        else
            hipLaunchKernelGGL((join_kernel<DT, D, 1, false>), dim3((unsigned)joins), dim3(256), 0, s, a, nrows);
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
    *bytes = paged::workspace(p, T, Hq, d);
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
    const size_t need = paged::workspace(p, T, Hq, d);
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
    a.pml = need ? (float *)workspace + need / 4 / (d + 2) * d : nullptr;
    int st = HBA_OK;
#define HBA_PAGED(DT, D) st = paged::launch<DT, D>(a, p, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PAGED);
#undef HBA_PAGED
    return st;
}
