// Attention of new tokens over the paged cache (kr_pages, v_pages; or their form in 4
// or 8 bits, hba_mx.h): the newest token of each sequence (decode), several (a part of
// a prompt), whole or through a causal window with sinks; and of a batch whose
// sequences share their first pages, whose keys are then read once for all.
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
// Over codes, decode_codes and mx::attend take the place of the products over rows, and
//   even_codes_kernel  shares a long decode's pages out (as even_kernel, and by whole parts
//                      where those are even enough),
//   rows_even_kernel   shares out the keys of all row tiles of parts of prompts.
//
// With shared pages, both parts of the work are one launch (shared_kernel): neither
// fills the card alone.
#pragma once

#include "hba_abi.h"
#include "hba_common.h"
#include "hba_mx.h"
#include "hba_ragged.h"
#include "hba_rows.h"

namespace hba {
namespace paged {

using rows::ex2;
using rows::LOG2E;
using rows::Op;

// FMT: what the cache holds.  0: rows in the queries' type; 4, 8: codes of as many bits.
template <int DT, int D, int FMT> constexpr int64_t HEAD_BYTES =   // of a page's KV head
    FMT ? mx::page_bytes(D, FMT) : (int64_t)rows::PAGE * D * (DT == 1 ? 2 : 4);
// How the rows' products are taken (rows::Op): codes are exact in bf16, so fp32 rows go in parts.
template <int DT, int FMT> constexpr int OPS = FMT && DT == 0 ? 2 : DT;

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
    int *records;                       // of even shares of codes, see even_codes_kernel
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

// ------------------------------------------------------------ decode, codes --
// QKNorm, rotation (cs, sn: the lane's; y: the elements half a head away) and scale of a
// lane's N consecutive elements x of a head; lanes 16 and (ALL) 32 away have the others.
template <int D, int N, bool ALL>
__device__ __forceinline__ void finish_group(float (&x)[N], const float (&y)[N], bool first_half, const float *gain,
                                             float eps, bool turn, const float (&cs)[N], const float (&sn)[N],
                                             float scale) {
    if (gain) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) ss = fmaf(x[e], x[e], ss);
        ss += rows::other_row(ss);
        if constexpr (ALL) ss += rows::other_half(ss);
        scale *= *gain / sqrtf(fmaxf(ss / (float)D, eps));
    }
    if (turn) {
        const float sign = first_half ? -1.0f : 1.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = x[e] * cs[e] + y[e] * (sign * sn[e]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] *= scale;
}

// decode_part's walk over codes.  A unit's codes are a few registers; they become
// operands as they are used.
//   keys, 4 bits   go to the matrix cores as they are, with their scales; the queries are
//                  e2m3 parts, whose products with e2m1 are summed like fp32's.  (e4m3
//                  products are not: they lose bits below 2^-14 of the largest.)
//   keys, 8 bits   bf16 by one instruction a pair, scales included; queries in bf16 parts
//   values         bf16, without their scales: a lane's eight tokens have eight in each
//                  group, which go into the weights instead (a power of two: nothing is
//                  rounded), a set of weights for each group.
// With 8 heads or less (NS = 2) the columns 8 .. 15 are the same heads again: their lanes
// make the weights of the other half of the groups.
// A key that is not seen has logit -infinity; its value's codes and scale are 0.  So
// what is not finite there has no effect, at no cost.
// Bound by memory: 24 sequences of 4000 to 32000 keys, 28 heads over 4, d = 128, 4 bits, 219 MB
// in 52 us with the join (a copy's rate: 42), another 24 in 28; 9 of 1000 to 9000 in 8 bits, fp32,
// 45 MB in 19 + 4.  Below some 20 MB by latency: 64 windows of 1024 in 8 bits 8.4 us, one
// sequence of 1500 keys 8.6 (page numbers, pages, products, join in LDS, one after the other).
template <int DT, int D, int DW, int FMT, int NS>
__device__ __forceinline__ void decode_codes(const Args &a, int s, int g, int head, int L, int p0, int p1,
                                             f32x4 (&O)[D / 16], float &m, float &l) {
    constexpr int ESZ = DT == 1 ? 2 : 4, UK = FMT == 8 && D == 128 ? 32 : 64;
    constexpr int NDT = D / 16, NG = D / mx::GROUP, NH = UK / 32, UP = rows::PAGE / UK, NL = NG / NS;
    constexpr int NP = DT == 1 ? 1 : 3;                  // bf16 parts of a weight
    constexpr int NQ = FMT == 8 ? (DT == 1 ? 2 : 3) : DT == 0 ? 6 : D == 128 ? 3 : 4;   // parts of a query
    constexpr int NM = FMT == 4 && D == 64 ? NQ / 2 : NQ;   // D = 64: two parts in one product's 128 elements
    constexpr int NKS = FMT == 8 ? D / 32 : 1;
    constexpr int E = D / 4, KP = D * FMT / 256;         // codes of a lane in a tile; its 16-byte pieces of 32 tokens
    typedef const __attribute__((address_space(4))) int32_t *uniform;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = FMT == 4 ? lg % NG : lg * E / mx::GROUP;   // the group of a lane's key elements
    const Pages pg = page_list(a, L);
    const int u0 = p0 * UP, u1 = min(pg.n, p1) * UP;
    const char *kb = a.kr + (int64_t)g * HEAD_BYTES<DT, D, FMT>, *vb = a.v + (int64_t)g * HEAD_BYTES<DT, D, FMT>;
    const int64_t pstep = (int64_t)a.Hkv * HEAD_BYTES<DT, D, FMT>;
    const uniform table = (uniform)(uintptr_t)(a.table + (int64_t)s * a.maxp);
    // a lane's offsets in a page: codes (of 4-bit keys at D = 64 the halves of a group), scales
    const uint32_t co = lane * 16, k64 = (l16 + 32 * kg) * 16, ko = (l16 + 16 * kg) * 4;
    const uint32_t vo = (lg * NG + (NS == 2 ? (l16 >> 3) * NL : 0)) * 8;

    struct Unit {
        mx::u32x4 k[FMT == 4 ? 2 * NH : NH * KP], v[NH * KP];
        mx::u32x2 vs[NH][NL];
        uint32_t ks;
    };
    const auto logical = [&](int u) {
        const int i = min(u, u1 - 1) / UP;
        return i < pg.ns ? i : pg.w0 + i - pg.ns;
    };
    const auto place = [&](int u) { return max((int64_t)0, min((int64_t)table[logical(u)], a.pages - 1)); };
    const auto load = [&](Unit &x, int u, int64_t id) {
        const int h0 = UP == 1 ? 0 : u % UP;
        constexpr int HB = (int)HEAD_BYTES<DT, D, FMT>, CB = (int)mx::code_bytes(D, FMT);
        const mx::Buffer kp = mx::buffer(kb + id * pstep, HB), vp = mx::buffer(vb + id * pstep, HB);
        const uint32_t from = co + h0 * (KP * 1024);
        if constexpr (FMT == 4 && D == 64) {
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const mx::u32x2 lo = mx::load8(kp, k64, mt / 2 * 1024 + mt % 2 * 8);
                const mx::u32x2 hi = mx::load8(kp, k64, mt / 2 * 1024 + mt % 2 * 8 + 256);
                x.k[mt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NH * KP; ++i) x.k[i] = mx::load16(kp, from, i * 1024);
        }
        x.ks = mx::load4(kp, ko, CB);
#pragma unroll
        for (int i = 0; i < NH * KP; ++i) x.v[i] = mx::load16(vp, from, i * 1024);
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int i = 0; i < NL; ++i) x.vs[h][i] = mx::load8(vp, vo + h0 * (32 * NG), CB + (h * 4 * NG + i) * 8);
    };
    // Wave 0 makes the query's operand for all (and takes the units' turns last).
    constexpr int NE = FMT == 4 ? 32 : E;                 // a lane's elements of the query, from `first` on
    constexpr int QR = FMT == 4 ? 6 * NM : 4 * NKS * NQ;  // registers of the operand
    __shared__ uint32_t qlds[QR][64];
    __shared__ int slds[2][64];
    const int first = FMT == 4 ? 32 * kg : E * lg;
    if (wave == 0) {
        float qx[NE], qy[NE], cs[NE], sn[NE];
        const char *row = a.q + (int64_t)s * a.qst + head * a.qsh;
        const int64_t pos = max((int64_t)0, min((int64_t)L - 1, a.n_tab - 1)) * D;
#pragma unroll
        for (int i = 0; i < NE / 8; ++i) {
            float t[8];
            Op<DT>::unpack(Op<DT>::load(row + (first + 8 * i) * ESZ), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) qx[8 * i + e] = t[e];
        }
        if (a.cos) {
#pragma unroll
            for (int i = 0; i < NE / 8; ++i) {
                float t[8];
                Op<DT>::unpack(Op<DT>::load(row + ((first + D / 2) % D + 8 * i) * ESZ), t);
#pragma unroll
                for (int e = 0; e < 8; ++e) qy[8 * i + e] = t[e];
            }
#pragma unroll
            for (int e = 0; e < NE; e += 4) {
                *reinterpret_cast<f32x4 *>(cs + e) = *reinterpret_cast<const mx::f32x4u *>(a.cos + pos + first + e);
                *reinterpret_cast<f32x4 *>(sn + e) = *reinterpret_cast<const mx::f32x4u *>(a.sin + pos + first + e);
            }
        }
        finish_group<D, NE, FMT == 8 || D == 128>(qx, qy, first < D / 2, a.gain ? a.gain + head : nullptr, a.eps,
                                                  a.cos != nullptr, cs, sn, a.scales[s] * LOG2E);
        if constexpr (FMT == 4) {
            const mx::Query6<NQ> r = mx::parts6<NQ>(qx);
            int qs[2] = {0, 0};
#pragma unroll
            for (int n = 0; n < NM; ++n) {
                mx::u32x6 w = r.q[n];
                int b = r.scale[n];
                if constexpr (D == 64) {   // elements 0 .. 63 and again, of the next part
                    b = lg < 2 ? r.scale[2 * n] : r.scale[2 * n + 1];
#pragma unroll
                    for (int i = 0; i < 6; ++i) w[i] = lg < 2 ? r.q[2 * n][i] : r.q[2 * n + 1][i];
                }
#pragma unroll
                for (int i = 0; i < 6; ++i) qlds[6 * n + i][lane] = w[i];
                qs[n / 4] |= b << (8 * (n % 4));
            }
            slds[0][lane] = qs[0];
            slds[1][lane] = qs[1];
        } else {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                float t[8];
                bf16x8 p[NQ];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = qx[8 * ks + e];
                rows::parts<NQ>(t, p);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const mx::u32x4 w = __builtin_bit_cast(mx::u32x4, p[n]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) qlds[4 * (ks * NQ + n) + i][lane] = w[i];
                }
            }
        }
    }
    // Three units: one is worked on while two are on their way.  Past the end the last one
    // is loaded again (it is in the cache): a load that some passes of the loop leave out
    // would make all of them wait for every load there is.
    int u = u0 + (wave + DW - 1) % DW;
    Unit xa, xb, xc;
    int64_t next = 0;   // the place of the unit that is loaded next
    if (u < u1) {
        __builtin_amdgcn_sched_barrier(0);
        load(xa, u, place(u));
        __builtin_amdgcn_sched_barrier(0);
        load(xb, min(u + DW, u1 - 1), place(u + DW));
        __builtin_amdgcn_sched_barrier(0);
        next = place(u + 2 * DW);
    }
    __syncthreads();
    mx::i32x8 q6[FMT == 4 ? NM : 1];
    int qs[2] = {0, 0};           // scales of the parts, a byte each
    bf16x8 q16[NKS][FMT == 8 ? NQ : 1];
    if constexpr (FMT == 4) {
#pragma unroll
        for (int n = 0; n < NM; ++n) {
            q6[n] = mx::i32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 6; ++i) q6[n][i] = (int)qlds[6 * n + i][lane];
        }
        qs[0] = slds[0][lane];
        qs[1] = slds[1][lane];
    } else {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                mx::u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = qlds[4 * (ks * NQ + n) + i][lane];
                q16[ks][n] = __builtin_bit_cast(bf16x8, w);
            }
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.0f;
    const auto use = [&](Unit &x, int at) {
        const int h0 = UP == 1 ? 0 : at % UP, j0 = logical(at) * rows::PAGE + h0 * UK;
        f32x4 S[2 * NH];
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt) S[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (FMT == 4) {
            // part by part over the tiles: a tile's sums wait for one another
            const auto part = [&](auto N) {
                constexpr int n = N.value;
                if constexpr (n < NM) {
                    S[0] = mx::product6<0, n % 4>(x.k[0], q6[n], S[0], x.ks, qs[n / 4]);
                    S[1] = mx::product6<1, n % 4>(x.k[1], q6[n], S[1], x.ks, qs[n / 4]);
                    S[2] = mx::product6<2, n % 4>(x.k[2], q6[n], S[2], x.ks, qs[n / 4]);
                    S[3] = mx::product6<3, n % 4>(x.k[3], q6[n], S[3], x.ks, qs[n / 4]);
                }
            };
            part(mx::number<0>());
            part(mx::number<1>());
            part(mx::number<2>());
            part(mx::number<3>());
            part(mx::number<4>());
            part(mx::number<5>());
        } else {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
                for (int mt = 0; mt < 2 * NH; ++mt) {
                    const float sc = __uint_as_float((x.ks >> (8 * (2 * h0 + mt)) & 255u) << 23);
                    const int w = 2 * (mt * NKS + ks);   // the first of the two words of 8 codes
                    const uint32_t c[2] = {x.k[w / 4][w % 4], x.k[w / 4][w % 4 + 1]};
                    const bf16x8 kf = mx::eight<8>(c, sc);
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        S[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q16[ks][n], S[mt], 0, 0, 0);
                }
        }
        // S[mt][e]: key j0 + 32 (mt / 2) + 8 lg + 4 (mt % 2) + e
        const bool whole = j0 + UK <= L && (j0 >= pg.lo || j0 + UK <= a.S);
        if (!whole) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const uint32_t bits = (uint32_t)(rows::seen_bits(pg.lo, L, a.S, j0 + 32 * h) >> (8 * lg));
                // four bits as four bytes
                const uint32_t see[2] = {((bits & 15u) * 0x00204081u & 0x01010101u) * 255u,
                                         ((bits >> 4 & 15u) * 0x00204081u & 0x01010101u) * 255u};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    S[2 * h + (e >> 2)][e & 3] = rows::keep(S[2 * h + (e >> 2)][e & 3], bits, e, -INFINITY);
#pragma unroll
                for (int i = 0; i < NL; ++i)
#pragma unroll
                    for (int w = 0; w < 2; ++w) x.vs[h][i][w] &= see[w];
                if constexpr (FMT == 8) {   // a code may be a NaN
#pragma unroll
                    for (int i = 0; i < KP; ++i)
#pragma unroll
                        for (int w = 0; w < 4; ++w) x.v[h * KP + i][w] &= see[w & 1];
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2 * NH; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, S[mt][e]);
        top = fmaxf(top, rows::other_row(top));
        top = fmaxf(top, rows::other_half(top));
        if (__ballot(top > m)) {
            const float mn = fmaxf(m, top), al = m == -INFINITY ? 0.0f : ex2(m - mn);
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
#pragma unroll
            for (int i = 0; i < NL; ++i) {   // the lane's i-th group
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = p[e] * mx::power(x.vs[h][i][e >> 2], e & 3);
                bf16x8 pf[NP];   // bf16 output: a relative 2^-8 each at most; l has them as they are
                rows::parts<NP>(y, pf);
#pragma unroll
                for (int k = 0; k < 2 * NS; ++k) {   // the columns of that group in each set
                    const int dt = 2 * (k / 2 * NL + i) + k % 2;
                    constexpr int W = FMT / 4;
                    const int w = dt * W;
                    const uint32_t c[2] = {x.v[h * KP + w / 4][w % 4], W == 2 ? x.v[h * KP + w / 4][w % 4 + W - 1] : 0u};
                    const bf16x8 vf = mx::eight<FMT>(c, 1.0f);
#pragma unroll
                    for (int n = 0; n < NP; ++n) O[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], O[dt], 0, 0, 0);
                }
            }
        }
    };
    const auto step = [&](Unit &now, Unit &free) {
        load(free, min(u + 2 * DW, u1 - 1), next);
        next = place(u + 3 * DW);
        __builtin_amdgcn_sched_barrier(0);
        use(now, u);
        __builtin_amdgcn_sched_barrier(0);
        u += DW;
        return u < u1;
    };
    if (u >= u1) return;
#pragma unroll 1
    while (step(xa, xc) && step(xb, xa) && step(xc, xb)) {}
}

// gi: 16 heads of a KV head of sequence s; pages p0 .. p1 - 1 of its list.  Head i of
// the 16 writes part at + i step, or its row of the output (at < 0).
// Units of UK keys: a page, or half of one where a page's operands would fill the
// registers.  DW waves take the pages' units in turn.
template <int DT, int D> constexpr int UNIT = DT == 1 && D == 64 ? 64 : 32;
template <int D> struct DecodeLds {
    float o[4][16][D + 4], m[4][16], l[4][16];
};
template <int DT, int D, int DW, int FMT, int NS>
__device__ __forceinline__ void decode_part(const Args &a, DecodeLds<D> &lds, int s, int gi, int p0, int p1,
                                            int64_t at, int step, int known = -1) {   // known: the length, if it is
    typedef typename Op<DT>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, UK = UNIT<DT, D>;
    constexpr int NKS = D / 32, NDT = D / 16, NH = UK / 32, UP = rows::PAGE / UK;
    typedef const __attribute__((address_space(4))) int32_t *uniform;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ct = (a.G + 15) / 16;
    const int g = gi / ct, c0 = gi % ct * 16;
    const int L = FMT != 0 && known >= 0 ? known : length(a, s);
    const int hr = NS == 2 ? l16 & 7 : l16;   // the lane's head of the 16 (or 8, twice)
    const int hl = c0 + hr, head = g * a.G + min(hl, a.G - 1);
    f32x4 O[NDT];
    float m, l;
    if constexpr (FMT != 0) {
        decode_codes<DT, D, DW, FMT, NS>(a, s, g, head, L, p0, p1, O, m, l);
    } else {
        const Pages pg = page_list(a, L);
        const int u0 = p0 * UP, u1 = min(pg.n, p1) * UP;
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
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.0f;
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
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // the waves' sums meet in LDS: those of waves 4 and up fold into the first four's
    const auto put = [&](int w) {
        if (lg == 0) {
            lds.m[w][hr] = m;
            lds.l[w][hr] = l;
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            if (NS == 2 && l16 >> 3 != dt / (NDT / 2)) continue;   // the other set has these columns
            *reinterpret_cast<f32x4 *>(&lds.o[w][hr][16 * dt + 4 * lg]) = O[dt];
        }
    };
    if constexpr (DW > 4) {
        if (wave >= 4) put(wave - 4);
        __syncthreads();
        if (wave < 4) {
            const float om = lds.m[wave][hr], ol = lds.l[wave][hr], mn = fmaxf(m, om);
            const float fa = m == -INFINITY ? 0.0f : ex2(m - mn), fb = om == -INFINITY ? 0.0f : ex2(om - mn);
            l = fmaf(ol, fb, l * fa);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                O[dt] = O[dt] * fa + *reinterpret_cast<const f32x4 *>(&lds.o[wave][hr][16 * dt + 4 * lg]) * fb;
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
template <int DT, int D, int DW, int FMT, int NS>
__device__ __forceinline__ void decode_run(const Args &a, DecodeLds<D> &lds, int group, int part) {
    const int ct = (a.G + 15) / 16, ng = a.Hkv * ct, s = group / ng, gi = group % ng;
    const int64_t row = (int64_t)s * a.Hq + gi / ct * a.G + gi % ct * 16;
    decode_part<DT, D, DW, FMT, NS>(a, lds, s, gi, part * a.part, (part + 1) * a.part,
                           a.slots == 1 ? -1 : row * a.slots + a.slot0 + part, a.slots);
}
template <int DT, int D, int FMT, int NS> __global__ __launch_bounds__(64 * DW) void decode_kernel(const Args a) {
    __shared__ DecodeLds<D> lds;
    decode_run<DT, D, DW, FMT, NS>(a, lds, blockIdx.x, blockIdx.y);
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
// The same for codes (at most MOST sequences), where a share's own work is short: what
// comes before each sequence is found once, in LDS, and for the join a group's first
// share writes down which parts are its own (records: [groups][2], the first one and how
// many, 0 if the group is done).  A second part costs a workgroup as much as
// EXTRA pages (5 us: its query, first loads and sums).  So where parts of up to so many
// pages more make no more of them than there are shares, each workgroup has one part.
constexpr int MOST = 1024, EXTRA = 16;
// The sums of count(i) over the sequences before each i, and over all, by a workgroup.
template <int NT, class F> __device__ __forceinline__ int sums_before(int Bd, int *before, const F &count) {
    __shared__ int wsum[NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int sum = 0;
    for (int base = 0; base < Bd; base += NT) {
        const int i = base + tid, n = i < Bd ? count(i) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o, 64);
            if (lane >= o) upto += x;
        }
        if (lane == 63) wsum[wave] = upto;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            if (w < wave) upto += wsum[w];
            all += wsum[w];
        }
        if (i < Bd) before[i] = sum + upto - n;
        sum += all;
        __syncthreads();
    }
    if (tid == 0) before[Bd] = sum;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sum);
}
template <int DT, int D, int FMT, int NS> __global__ __launch_bounds__(64 * DW) void even_codes_kernel(const Args a) {
    constexpr int NT = 64 * DW;
    __shared__ DecodeLds<D> lds;
    __shared__ int before[MOST + 1], pages[MOST], len[MOST], counts[EXTRA], found;
    const int tid = threadIdx.x, w = blockIdx.x, ng = groups_of(a);
    const auto find = [&](int64_t x) {   // the sequence with place x
        for (int i = tid; i < a.Bd; i += NT)
            if (x >= (int64_t)before[i] * ng && x < (int64_t)before[i + 1] * ng) found = i;
        __syncthreads();
        return __builtin_amdgcn_readfirstlane(found);
    };
    const int units = sums_before<NT>(a.Bd, before, [&](int i) {
        len[i] = length(a, i);
        return pages[i] = max(1, page_list(a, len[i]).n);
    }) * ng;
    int per = max(a.part, (units + a.slots - 1) / a.slots);
    {   // the parts there are at per + c pages
        static_assert(NT % EXTRA == 0 && NT / EXTRA <= 64, "a candidate's threads are lanes of a wave");
        const int c = tid / (NT / EXTRA);
        int n = 0;
        for (int i = tid % (NT / EXTRA); i < a.Bd; i += NT / EXTRA) n += (pages[i] + per + c - 1) / (per + c);
#pragma unroll
        for (int o = 1; o < NT / EXTRA; o <<= 1) n += __shfl_xor(n, o, 64);
        counts[c] = n * ng;
    }
    __syncthreads();
    int more = 0;
    while (more < EXTRA && counts[more] > a.slots) ++more;
    if (more < EXTRA) {
        per += more;
        const int parts = sums_before<NT>(a.Bd, before, [&](int i) { return (pages[i] + per - 1) / per; }) * ng;
        if (w >= parts) return;
        const int s = find(w), n = __builtin_amdgcn_readfirstlane(pages[s]), k = (n + per - 1) / per;
        const int x = w - __builtin_amdgcn_readfirstlane(before[s]) * ng, gi = x / k, z = x % k, run = (n + k - 1) / k;
        if (z == 0 && tid == 0) {
            a.records[2 * (s * ng + gi)] = 2 * w;
            a.records[2 * (s * ng + gi) + 1] = k == 1 ? 0 : k;
        }
        decode_part<DT, D, DW, FMT, NS>(a, lds, s, gi, z * run, (z + 1) * run, k == 1 ? -1 : (int64_t)w * 32, 1,
                                        __builtin_amdgcn_readfirstlane(len[s]));
        return;
    }
    const int64_t u0 = (int64_t)w * per, u1 = min(u0 + per, (int64_t)units);
    if (u0 >= units) return;
    int s = find(u0), left = (int)(u1 - u0), at = (int)u0 - __builtin_amdgcn_readfirstlane(before[s]) * ng;
    for (int part = 2 * w; left > 0 && s < a.Bd; part = 2 * w + 1) {
        const int n = __builtin_amdgcn_readfirstlane(pages[s]), gi = at / n, p0 = at % n, p1 = min(n, p0 + left);
        if (p0 == 0 && tid == 0) {
            a.records[2 * (s * ng + gi)] = part;
            a.records[2 * (s * ng + gi) + 1] = p1 == n ? 0 : (int)((u1 - left + n - 1) / per) - w + 1;
        }
        decode_part<DT, D, DW, FMT, NS>(a, lds, s, gi, p0, p1, p1 - p0 == n ? -1 : (int64_t)part * 16, 1,
                                        __builtin_amdgcn_readfirstlane(len[s]));
        __syncthreads();   // lds is free again
        left -= p1 - p0;
        at += p1 - p0;
        if (at == n * ng) {
            at = 0;
            ++s;
        }
    }
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
        decode_part<DT, D, DW, 0, 1>(a, lds, s, at / n, p0, p1, p1 - p0 == n ? -1 : (int64_t)part * 16, 1);
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

// finish_q for Rows6: x[s] are the elements 64 s + 32 hf .. of the row; cs, sn begin at 32 hf.
// The table's rows are loaded at once, in 16 bytes (wherever the tensor begins): an element at
// a time, each behind a branch, they were 12 us of a workgroup of 128 rows.
template <int D>
__device__ __forceinline__ void finish_rows(float (&x)[D / 64][32], int hf, const float *gain, float eps, const float *cs,
                                            const float *sn, float scale) {
    const auto norm = [&]() {
        if (gain) {
            float ss = 0.0f;
#pragma unroll
            for (int s = 0; s < D / 64; ++s)
#pragma unroll
                for (int e = 0; e < 32; ++e) ss = fmaf(x[s][e], x[s][e], ss);
            ss += rows::other_half(ss);
            scale *= *gain / sqrtf(fmaxf(ss / (float)D, eps));
        }
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
#pragma unroll
            for (int e = 0; e < 32; ++e) x[s][e] *= scale;
    };
    if (!cs) {
        norm();
        return;
    }
    constexpr int M = 2048 / D;   // elements at a time: 64 registers
    float first[2][D / 64][M];
    const auto load = [&](int e0, float (&to)[2][D / 64][M]) {
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
#pragma unroll
            for (int i = 0; i < M; i += 4) {
                *reinterpret_cast<f32x4 *>(&to[0][s][i]) = *reinterpret_cast<const mx::f32x4u *>(cs + 64 * s + e0 + i);
                *reinterpret_cast<f32x4 *>(&to[1][s][i]) = *reinterpret_cast<const mx::f32x4u *>(sn + 64 * s + e0 + i);
            }
    };
    const auto turn = [&](int e0, const float (&by)[2][D / 64][M]) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            float &lo = x[0][e0 + i];
            if constexpr (D == 64) {
                const float y = rows::other_half(lo);
                lo = lo * by[0][0][i] + y * (hf ? by[1][0][i] : -by[1][0][i]);
            } else {
                float &hi = x[1][e0 + i];
                const float y = lo * by[0][0][i] - hi * by[1][0][i];
                hi = hi * by[0][1][i] + lo * by[1][1][i];
                lo = y;
            }
        }
    };
    load(0, first);
    norm();
    turn(0, first);
    if constexpr (M < 32) {
        load(M, first);
        turn(M, first);
    }
}

// A row's query: operands of the product with bf16 or fp32 keys (h; fp32 ones of codes have
// all parts there), and with 4-bit codes (q6).
template <int DT, int D, int FMT> struct Queries {
    typedef typename Op<OPS<DT, FMT>>::F F;
    static constexpr int NKS = D / 16;
    F h[FMT == 4 ? 1 : NKS], l[FMT == 4 || OPS<DT, FMT> == 2 ? 1 : NKS];
    mx::Rows6<FMT == 4 ? D : 64, FMT != 4 ? 1 : DT == 1 ? 3 : 6> q6;
    __device__ __forceinline__ const auto &keys() const {
        if constexpr (FMT == 4) return q6;
        else return h;
    }
    // word w of the parts that are used
    static constexpr int HW = sizeof(h) / 4, WORDS = FMT == 4 ? decltype(q6)::WORDS : (sizeof(h) + (OPS<DT, FMT> == 2 ? 0 : sizeof(l))) / 4;
    __device__ __forceinline__ int &word(int w) {
        if constexpr (FMT == 4) return q6.word(w);
        else return w < HW ? reinterpret_cast<int *>(h)[w] : reinterpret_cast<int *>(l)[w - HW];
    }
};
template <int DT, int D, int FMT>
__device__ __forceinline__ void row_queries(const Args &a, int t, int head, int pos, int s, Queries<DT, D, FMT> &to) {
    constexpr int ESZ = DT == 1 ? 2 : 4, N = D / 16, OP = OPS<DT, FMT>;
    const int hf = (threadIdx.x & 63) >> 5;
    const char *q = a.q + (int64_t)t * a.qst + head * a.qsh;
    const int64_t turn = max((int64_t)0, min((int64_t)pos, a.n_tab - 1)) * D + (FMT == 4 ? 32 * hf : 0);
    const float *gain = a.gain ? a.gain + head : nullptr, *cs = a.cos ? a.cos + turn : nullptr;
    const float *sn = a.sin ? a.sin + turn : nullptr, scale = a.scales[s] * LOG2E;
    if constexpr (FMT == 4) {
        float y[D / 64][32];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float z[8];
            Op<DT>::unpack(Op<DT>::load(q + (64 * (i / 4) + 32 * hf + 8 * (i % 4)) * ESZ), z);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i / 4][8 * (i % 4) + e] = z[e];
        }
        finish_rows<D>(y, hf, gain, a.eps, cs, sn, scale);
        to.q6.set(y);
    } else {
        float y[N][8];
#pragma unroll
        for (int ks = 0; ks < N; ++ks) Op<DT>::unpack(Op<DT>::load(q + (16 * ks + 8 * hf) * ESZ), y[ks]);
        finish_q<D, 16>(y, 8 * hf, gain, a.eps, cs, sn, scale);
#pragma unroll
        for (int ks = 0; ks < N; ++ks) {
            if constexpr (OP == 2) to.h[ks] = Op<OP>::pack(y[ks]);
            else split<DT>(y[ks], to.h[ks], to.l[ks]);
        }
    }
}

template <int DT, int D, int FMT> struct RowSource { typedef mx::TileKV<OPS<DT, FMT>, D, FMT> T; };
template <int DT, int D> struct RowSource<DT, D, 0> { typedef rows::PageKV<DT, D> T; };
// SHARED: the rows of all tokens over the shared pages (x: 128-row tile); else the
// rows of one sequence's tokens over its own pages (x: tile of the ragged batch).
// g: KV head, z: part, a run of a.part pages.
template <int DT, int D, int FMT, bool SHARED>
__device__ __forceinline__ void rows_part(const Args &a, char *smem, int x, int g, int z) {
    typedef typename RowSource<DT, D, FMT>::T Source;
    constexpr int OP = OPS<DT, FMT>;
    typedef typename Op<OP>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, NKS = D / 16, KT = Source::KT, TP = rows::PAGE / KT;
    constexpr bool LO = OP != 0;
    const int lane = threadIdx.x & 63, hf = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Source src;
    src.page = (int64_t)a.Hkv * HEAD_BYTES<DT, D, FMT>;
    src.k = a.kr + (int64_t)g * HEAD_BYTES<DT, D, FMT>;
    src.v = a.v + (int64_t)g * HEAD_BYTES<DT, D, FMT>;
    src.pages = a.pages;
    if constexpr (FMT != 0) {
        src.expected = -1;   // no tile is
        src.by = 1;
    }
    const auto begin = [&](int it0, int it1, int ns, int wt0) {
        if constexpr (FMT == 0) {
            rows::attend_begin(src, smem, it0, it1, ns, wt0);
        } else {
            src.ns = ns;
            src.wt0 = wt0;
            src.from = it0;
            src.last = it1 - 1;
            if (it0 < it1) src.next(0);
        }
    };
    const int it0 = z * a.part * TP;
    int s = 0, tile = x, first = 0, cnt = a.T, it1 = 0, ns = 0, wt0 = 0;
    if constexpr (SHARED) {   // every tile of the part, whatever the rows see of it: it can be staged at once
        src.table = a.table;
        src.len = a.shared * rows::PAGE;
        it1 = min(a.shared * TP, it0 + a.part * TP);
        begin(it0, it1, 0, 0);
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
        begin(it0, it1, ns, wt0);
    }
    Queries<DT, D, FMT> q;
    if constexpr (FMT == 0) {
        float y[NKS][8];
        const char *qp = a.q + (int64_t)t * a.qst + head * a.qsh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) Op<DT>::unpack(Op<DT>::load(qp + (16 * ks + 8 * hf) * ESZ), y[ks]);
        const int64_t turn = max((int64_t)0, min((int64_t)pos, a.n_tab - 1)) * D;
        finish_q<D, 16>(y, 8 * hf, a.gain ? a.gain + head : nullptr, a.eps, a.cos ? a.cos + turn : nullptr,
                        a.sin ? a.sin + turn : nullptr, a.scales[sq] * LOG2E);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) split<DT>(y[ks], q.h[ks], q.l[ks]);
    } else {
        row_queries(a, t, head, pos, sq, q);
    }
    rows::RowAcc<OP, D> acc;
    if constexpr (FMT == 0) rows::attend<OP, D, LO>(src, smem, q.h, q.l, 1.0f, it0, it1, ns, wt0, w, acc);
    else mx::attend<OP, D>(src, smem, q.keys(), q.l, it1 - it0, w, acc);
    float l = acc.l + rows::other_half(acc.l);
    const bool valid = w.hi > 0;
    if (__ballot(valid && (rows::any_bad<D>(acc.O) || !rows::finite(l)))) {
        if constexpr (FMT == 0) rows::attend_each<OP, D, LO>(src, q.h, q.l, 1.0f, it0, it1, ns, wt0, w, acc);
        else mx::attend_each<OP, D>(src, q.keys(), q.l, it1 - it0, w, acc);
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

// Over rows (FMT 0): 4 sequences, 1560 new tokens behind 1300 to 8500 keys, 14 heads, d = 64,
// bf16: 73 us, 27 at the rate of a large product.  Queries of two bf16 parts double q . k (3
// products for 2), exponentials and conversions as in the sliding-window kernel.  Over codes:
// `plan` has figures.  Registers are spilled, around the keys' loop or in it, at d = 128 (bf16, 4
// bits 18, 8 bits 105 of them; fp32, 8 bits 37) and by fp32 over 8 bits at d = 64 (58).
template <int DT, int D, int FMT, bool SHARED>
__global__ __launch_bounds__(64 * rows::NW, (DT == 1 && D == 64 && FMT != 8 ? 3 : rows::WAVES<DT, D>)) void rows_kernel(
    const Args a) {
    extern __shared__ __align__(16) char smem[];
    rows_part<DT, D, FMT, SHARED>(a, smem, blockIdx.x, blockIdx.y, blockIdx.z);
}

// ---------------------------------------------------------- rows, even shares ----
// Parts of prompts over codes.  All (128-row tile of a KV head, tile of its keys) make one
// list; each workgroup takes an even share of it, as decode's do, whatever the
// sequences' lengths.  SETS sets of four waves work on the same rows and take the key
// tiles in turn, each with buffers of its own, and join in LDS: as many waves as the
// registers leave room for, without their parts in memory.  (1560 tokens behind 1300 to 8500
// keys, 14 heads over 2, d = 64, 4 bits: 67 us and 5 for the join, 458 TFLOP/s, where 1024
// workgroups of a run of keys each took 71 and 8; 650 TFLOP/s at four times the tokens.  Three
// sets have 168 registers, too few: 96.  A window of 1024 in 8 bits, d = 128, 550 tokens: 38 and
// 6, by runs 69 with the join.  No spills of more than 7 registers, but 94 in bf16 over 4 bits at
// d = 128: 278 us for 1560 tokens behind 8000 keys, 28 heads over 4, by runs 316.)  Of a SIMD's
// time vector instructions have 60%, half of it exponentials and their rounding to bf16, and the
// matrix cores 30%; a piece's beginning and end are 10 us.
constexpr int TILES = 2048;    // row tiles of a KV head, at most
template <int DT, int D, int FMT> constexpr int SETS = DT == 0 && D == 128 ? 1 : 2;
// What a piece costs besides its keys, in tiles of keys (6 us, and 0.7 a tile; 10 and 0.9 at 32
// keys a tile).  Not counted, the workgroups with most pieces took half as long again.
template <int KT> constexpr int BEGIN = 512 / KT;
// What the tile of sequence s, of length L with cnt new tokens, sees: keys lo .. hi - 1 and sinks.
__device__ __forceinline__ void tile_sees(const Args &a, int L, int cnt, int tile, int &lo, int &hi) {
    const int r0 = tile * rows::RT, r1 = min(r0 + rows::RT, cnt * a.G) - 1;
    hi = max(0, L - cnt + r1 / a.G + 1);
    lo = a.W > 0 ? max(0, max(0, L - cnt + r0 / a.G) + 1 - a.W) : 0;
}
// A piece of the list, in LDS: what is needed again after its keys would spill in registers.
struct Piece {
    int s, tile, g, p0, p1, part;    // sequence, its row tile, KV head, key tiles p0 .. p1 - 1, part (-1: all keys)
    int first, count, len;           // of the sequence: its first new token, their number, all keys
    int next, at, left, head;        // where the next piece begins, and how many key tiles are left
    int tiles, per;                  // row tiles of a KV head, key tiles of a workgroup
};
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The kernel's first argument, read once more for the same reason.
__device__ __forceinline__ const Args &again() {
    uint64_t p = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm("" : "+s"(p));
    return *(const Args *)reinterpret_cast<const __attribute__((address_space(4))) Args *>(p);
}
template <int DT, int D, int FMT, int SETS>
__device__ __forceinline__ void rows_codes(const Args &a, char *smem, const Piece &job) {
    const int s = uniform(job.s), tile = uniform(job.tile), g = uniform(job.g), p0 = uniform(job.p0), p1 = uniform(job.p1);
    typedef typename RowSource<DT, D, FMT>::T Source;
    constexpr int OP = OPS<DT, FMT>;
    typedef typename Op<OP>::F F;
    constexpr int ESZ = DT == 1 ? 2 : 4, NKS = D / 16, KT = Source::KT;
    const int lane = threadIdx.x & 63, hf = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % rows::NW;
    const int set = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / rows::NW;
    const int first = uniform(job.first), cnt = uniform(job.count), L = uniform(job.len);
    int lo, hi, ns = 0, wt0 = 0;
    tile_sees(a, L, cnt, tile, lo, hi);
    const int nt = hi > 0 ? rows::tile_list<KT>(lo, hi, a.W > 0 ? a.S : 0, ns, wt0) : 0;
    Source src;
    src.page = (int64_t)a.Hkv * HEAD_BYTES<DT, D, FMT>;
    src.k = a.kr + (int64_t)g * HEAD_BYTES<DT, D, FMT>;
    src.v = a.v + (int64_t)g * HEAD_BYTES<DT, D, FMT>;
    src.pages = a.pages;
    src.table = a.table + (int64_t)s * a.maxp;
    src.len = L;
    src.expected = -1;
    src.ns = ns;
    src.wt0 = wt0;
    src.from = p0 + set;
    src.by = SETS;
    src.last = min(p1, nt) - 1;
    const int n = nt > 0 ? (p1 - p0 + SETS - 1) / SETS : 0;
    char *mine = smem + set * (2 * Source::BYTES);
    if (n > 0) src.next(0);

    const int nr = cnt * a.G, r = tile * rows::RT + wave * rows::RW + (lane & 31);
    const bool in = r < nr;
    const int t = first + min(r, nr - 1) / a.G, head = g * a.G + min(r, nr - 1) % a.G, pos = L - cnt + t - first;
    rows::Sees w;
    w.S = a.W > 0 ? a.S : 0;
    w.hi = in && pos >= 0 ? pos + 1 : 0;
    w.lo = a.W > 0 ? max(0, pos + 1 - a.W) : 0;
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
    // Set 0 makes the queries for all.
    Queries<DT, D, FMT> q;
    if (set == 0) row_queries(a, t, head, pos, s, q);
    if constexpr (SETS > 1) {
        static_assert(q.WORDS * 1024 <= SETS * 2 * Source::BYTES, "before the tiles, in their place");
        int *at = reinterpret_cast<int *>(smem) + (threadIdx.x & 255);
        if (set == 0) {
#pragma unroll
            for (int i = 0; i < q.WORDS; ++i) at[i * 256] = q.word(i);
        }
        __syncthreads();
        if (set > 0) {
#pragma unroll
            for (int i = 0; i < q.WORDS; ++i) q.word(i) = at[i * 256];
        }
        __syncthreads();
    }
    rows::RowAcc<OP, D> acc;
    mx::attend<OP, D>(src, mine, q.keys(), q.l, n, w, acc);
    float l = acc.l + rows::other_half(acc.l);
    const bool valid = w.hi > 0;
    if (__ballot(valid && (rows::any_bad<D>(acc.O) || !rows::finite(l)))) {
        mx::attend_each<OP, D>(src, q.keys(), q.l, n, w, acc);
        l = acc.l + rows::other_half(acc.l);
    }
    if (!valid) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) acc.O[dt] = f32x16{0.0f};
        acc.m = -INFINITY;
        l = 0.0f;
    }
    if constexpr (SETS > 1) {   // into set 0, 32 columns at a time
        __shared__ float ml[SETS][rows::RT][2];
        const int row = wave * rows::RW + (lane & 31);
        if (hf == 0) {
            ml[set][row][0] = acc.m;
            ml[set][row][1] = l;
        }
        __syncthreads();
        float f[SETS], top = acc.m;
#pragma unroll
        for (int i = 0; i < SETS; ++i) top = fmaxf(top, ml[i][row][0]);
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            // a set without keys has zeros; scores that are all -inf have them too, and l 0
            f[i] = ml[i][row][0] == -INFINITY ? 0.0f : ex2(ml[i][row][0] - top);
            l = fmaf(ml[i][row][1], ml[i][row][0] == -INFINITY ? 1.0f : f[i], l);
        }
        acc.m = top;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
            f32x4 *buf = reinterpret_cast<f32x4 *>(smem) + wave * 256 + lane;
            if (set > 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    buf[(set - 1) * 1024 + i * 64] =
                        f32x4{acc.O[dt][4 * i], acc.O[dt][4 * i + 1], acc.O[dt][4 * i + 2], acc.O[dt][4 * i + 3]};
            }
            __syncthreads();
            if (set == 0) {
                acc.O[dt] = acc.O[dt] * f[0];
#pragma unroll
                for (int j = 1; j < SETS; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 x = buf[(j - 1) * 1024 + i * 64] * f[j];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc.O[dt][4 * i + e] += x[e];
                    }
            }
            __syncthreads();
        }
    }
    if (set == 0) {
        const Args &b = again();
        const int part = uniform(job.part), k = wave * rows::RW + (lane & 31), cnt = uniform(job.count);
        const int r = uniform(job.tile) * rows::RT + k;
        if (r < cnt * b.G) {
            if (part < 0) {
                const int64_t row = (int64_t)(uniform(job.first) + r / b.G) * b.Hq + uniform(job.g) * b.G + r % b.G;
                const bool valid = uniform(job.len) - cnt + r / b.G >= 0;
                rows::store_rows<DT, D>(b.out + row * D * ESZ, acc.O, valid ? 1.0f / l : 0.0f);
            } else {
                const int64_t at = (int64_t)part * rows::RT + k;
                rows::store_rows<0, D>(reinterpret_cast<char *>(b.po + at * D), acc.O, 1.0f);
                if (hf == 0) {
                    b.pml[2 * at] = acc.m;
                    b.pml[2 * at + 1] = l;
                }
            }
        }
    }
}
// records: the number of row tiles, then from [4] on four for each (KV head, row tile of
// `tiles`): the first part, how many (0: done), sequence, tile of the sequence.
template <int DT, int D, int FMT>
__global__ __launch_bounds__((256 * SETS<DT, D, FMT>)) void rows_even_kernel(const Args a, int tiles) {
    constexpr int NS = SETS<DT, D, FMT>, NT = 256 * NS, KT = RowSource<DT, D, FMT>::T::KT;
    extern __shared__ __align__(16) char smem[];
    __shared__ int before[MOST + 1], upto[TILES + 1], first[MOST], count[MOST], len[MOST];
    __shared__ Piece job;
    const int tid = threadIdx.x, w = blockIdx.x;
    const int nt = min(tiles, sums_before<NT>(a.Bd, before, [&](int i) {
        len[i] = length(a, i);
        count[i] = ragged::tokens(a.cu, i, a.T, first[i]);
        return (count[i] * a.G + rows::RT - 1) / rows::RT;
    }));
    const auto sequence = [&](int tile) {   // the last one that begins at the tile or before: it has tiles
        int lo = 0, hi = again().Bd - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= tile) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    const int U = sums_before<NT>(nt, upto, [&](int i) {
        const int s = sequence(i);
        int lo, hi, ns, wt0;
        tile_sees(a, len[s], count[s], i - before[s], lo, hi);
        return BEGIN<KT> + max(1, hi > 0 ? rows::tile_list<KT>(lo, hi, a.W > 0 ? a.S : 0, ns, wt0) : 0);
    });
    const int64_t units = (int64_t)U * a.Hkv;
    const int per = (int)max((int64_t)(BEGIN<KT> + 2 * NS), (units + a.slots - 1) / a.slots);
    if (w == 0 && tid == 0) a.records[0] = nt;
    const int64_t u0 = (int64_t)w * per, u1 = min(u0 + per, units);
    if (tid == 0) job.left = 0;
    __syncthreads();
    for (int i = tid; i < nt && u0 < units; i += NT) {
        const int at = (int)(u0 % U) - upto[i];
        if (at < 0 || at >= upto[i + 1] - upto[i]) continue;
        job.next = i;
        job.at = at;
        job.left = (int)(u1 - u0);
        job.head = (int)(u0 / U);
        job.tiles = nt;
        job.per = per;
    }
    __syncthreads();
    for (int turn = 0; uniform(job.left) > 0; turn = 1) {
        __syncthreads();
        if (tid == 0) {
            const Args &b = again();
            const int i = job.next, n = upto[i + 1] - upto[i] - BEGIN<KT>, at = job.at, to = min(n + BEGIN<KT>, at + job.left);
            const int p0 = max(0, at - BEGIN<KT>), p1 = max(0, to - BEGIN<KT>);   // p1 0: the next workgroup has the first keys
            const int g = job.head, s = sequence(i), tile = i - before[s], part = 2 * (int)blockIdx.x + turn;
            if (p0 == 0 && p1 > 0) {
                int *r = b.records + 4 + ((int64_t)g * tiles + i) * 4;
                r[0] = part;
                r[1] = p1 == n ? 0 : 2 + (n - p1 - 1) / job.per;
                r[2] = s;
                r[3] = tile;
            }
            job.s = s;
            job.tile = tile;
            job.g = g;
            job.first = first[s];
            job.count = count[s];
            job.len = len[s];
            job.p0 = p0;
            job.p1 = p1;
            job.part = p0 == 0 && p1 == n ? -1 : part;
            const bool end = p1 == n && i + 1 == job.tiles;
            job.next = end ? 0 : i + (p1 == n);
            job.at = p1 == n ? 0 : to;
            job.head = g + end;
            job.left -= to - at;
        }
        __syncthreads();
        if (uniform(job.p1) == 0) break;
        rows_codes<DT, D, FMT, NS>(a, smem, job);
    }
    if (tid < 256)
        for (int g = 0; g < again().Hkv; ++g) zero_strays<DT, D>(again(), g, blockIdx.x, gridDim.x);
}
// The parts of a row tile's 128 rows, as join_kernel.
template <int DT, int D> __global__ __launch_bounds__(256) void rows_join_kernel(const Args a, int tiles) {
    constexpr int TP = D / 4;
    const int i = blockIdx.x, g = blockIdx.y;
    if (i >= a.records[0]) return;
    const int *rec = a.records + 4 + ((int64_t)g * tiles + i) * 4;
    const int parts = rec[1], w0 = rec[0] / 2, s = rec[2], tile = rec[3];
    if (parts == 0) return;
    int first;
    const int cnt = ragged::tokens(a.cu, s, a.T, first), L = length(a, s);
    const int x = threadIdx.x % TP * 4, k = blockIdx.z * (256 / TP) + threadIdx.x / TP, r = tile * rows::RT + k;
    if (r >= cnt * a.G) return;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    for (int p = 0; p < parts; p += 4) {
        float pm[4], pl[4];
        f32x4 px[4];
        float mn = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int q = min(p + e, parts - 1);
            const int64_t at = (int64_t)(q == 0 ? rec[0] : 2 * (w0 + q)) * rows::RT + k;
            pm[e] = p + e < parts ? a.pml[2 * at] : -INFINITY;
            pl[e] = p + e < parts ? a.pml[2 * at + 1] : 0.0f;
            px[e] = *reinterpret_cast<const f32x4 *>(a.po + at * D + x);
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
    const int t = first + r / a.G;
    const int64_t row = (int64_t)t * a.Hq + g * a.G + r % a.G;
    const f32x4 y = L - cnt + r / a.G >= 0 ? o / l : f32x4{0.f, 0.f, 0.f, 0.f};   // it sees nothing: 0
    char *to = a.out + (row * D + x) * (DT == 1 ? 2 : 4);
    if constexpr (DT == 1)
        *reinterpret_cast<uint2 *>(to) = make_uint2(pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3]));
    else
        *reinterpret_cast<f32x4 *>(to) = y;
}
// The shared pages for all rows (the first nshared workgroups, which take longest)
// and every sequence's own pages for its newest token: 64 sequences, 8192 shared
// keys, d = 64: 14.5 us, and 5 of the join.
template <int DT, int D, int FMT, int NS>
__global__ __launch_bounds__(64 * rows::NW, (rows::WAVES<DT, D>)) void shared_kernel(
    const Args a, const Args own, int ptiles, int nshared, int groups) {
    extern __shared__ __align__(16) char smem[];
    const int i = blockIdx.x;
    if (i < nshared)
        rows_part<DT, D, FMT, true>(a, smem, i % ptiles, i / ptiles % a.Hkv, i / (ptiles * a.Hkv));
    else
        decode_run<DT, D, rows::NW, FMT, NS>(own, *reinterpret_cast<DecodeLds<D> *>(smem), (i - nshared) % groups,
                                    (i - nshared) / groups);
}

// out = sum of the parts' O 2^(m - max) over sum of their l 2^(m - max); a row
// without keys 0.  D / 4 threads a part, SG parts of a row at a time (all of a
// workgroup where a row has many parts, one where rows are many), each with sums
// of its own that LDS joins.  EVEN: the parts are those of even shares (2: written down).
template <int DT, int D, int SG, int EVEN>
__global__ __launch_bounds__(256) void join_kernel(const Args a, int64_t nrows) {
    constexpr int TP = D / 4, RB = 256 / (TP * SG);   // threads of a part, rows of a workgroup
    __shared__ float so[SG > 1 ? SG : 1][SG > 1 ? D : 1];
    __shared__ float sm[SG], sl[SG];
    const int x = threadIdx.x % TP * 4, sg = threadIdx.x / TP % SG;
    const int64_t row = (int64_t)blockIdx.x * RB + threadIdx.x / (TP * SG);
    if (row >= nrows) return;                         // SG > 1: the workgroup's one row
    int slots = a.slots, step = 1;                    // part p at first + p step, the row's first part at part0
    int64_t first_part = row * a.slots, part0 = first_part;
    if constexpr (EVEN == 2) {
        const int s = (int)(row / a.Hq), h = (int)(row % a.Hq), ct = (a.G + 15) / 16, hc = h % a.G;
        const int *r = a.records + 2 * ((s * a.Hkv + h / a.G) * ct + hc / 16);
        slots = r[1];
        if (slots == 0) return;                       // written already
        step = 32;
        first_part = (int64_t)(r[0] / 2) * 32 + hc % 16;
        part0 = (int64_t)r[0] * 16 + hc % 16;
    } else if constexpr (EVEN) {
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
    const bool sees = EVEN == 2 || (t >= first && t - first < cnt && length(a, s) - cnt + t - first >= 0);
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
    bool even_rows;               // shares of row tiles' lists of keys
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
                 int64_t max_len, int64_t d, int bits) {   // bits: of the cache's codes, or 0
    Plan p = {};
    const int64_t G = Hq / Hkv, KT = rows::PAGE;
    // A window or sinks past every length are every key, and no sum below overflows.
    W = W < max_len ? W : max_len;
    S = S < max_len ? S : max_len;
    int64_t keys = max_len - shared * KT;
    if (W > 0 && W < keys) keys = W;
    // A part of a prompt may span any number of windows.  (The parts cut the list of one
    // 128-row tile, which has W + 128 / G tokens and the sinks, so of a window's parts most are empty.)
    if (W > 0 && !one) keys = max_len;
    if (bits && W > 0 && !one && W + rows::RT / G + 1 < max_len) keys = W + rows::RT / G + 1;   // that list
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
        // Shares of codes where there are enough keys for them: a share begins and ends in 20 us, a
        // run in 12, but at d = 128 those of 8-bit keys spill.  Shares and runs, bf16, d = 64, 4 bits:
        // 1560 tokens behind 1000, 2500, 8000 keys 35, 45, 66 and 35, 49, 77 us, 4900 in 16 sequences
        // 82 and 99, a window of 1024 in those 76 and 52; 5 tokens behind 16000 keys 25 and 18, 16
        // times 1 to 6 behind 4000 23 and 26; in 8 bits 1560 tokens alone, behind 1000 and 8000 keys
        // 26, 35, 71 and 19, 34, 101, the windows 80 and 74, the 5 tokens 25 and 17.  d = 128, 8 bits:
        // 5 tokens behind 16000 keys 34 and 40, 8 times 1 to 6 behind 1600 30 and 48; 3 windows of
        // 1024 44 and 68 (fp32 70 and 61), 64 of 1 to 6 tokens 52 and 81.  d = 128, 4 bits, bf16 (and
        // fp32): 1560 tokens behind 1000, 2500, 8000 keys 84, 126, 278 and 85, 133, 316 (132, 240, 631
        // and 160, 278, 702), alone 71 and 64 (103 and 122), 4900 in 16 sequences 321 and 296 (661 and
        // 763), a window of 1024 in those 189 and 149 (320 and 348); 5 tokens behind 16000 keys 38 and
        // 27 (50 and 51), 16 times 1 to 6 behind 4000 46 and 54 (76 and 116), 8 times behind 1600 34
        // and 30 (45 and 52).  fp32, d = 64, 4 bits (8 bits): 45, 64, 138 and 47, 71, 150 (47, 69, 155
        // and 50, 82, 181); 5 tokens 33 and 20 (33 and 21), 16 times 31 and 34 (32 and 40).  So bf16's
        // borders cost fp32 at d = 128 up to a fifth where it stays in runs, and bf16 in 4 bits a
        // twelfth where many tokens are shared out.
        // (And what LDS holds, the join's grid, sums in 32 bits.)
        const int64_t all_pages = p.tiles * Hkv * pages;
        const bool enough = bits && (bits == 8 && d == 128 ? all_pages >= 512 : pages > 32 && all_pages >= 2048);
        if (enough && !shared && Bd <= MOST && p.tiles <= TILES && p.tiles * Hkv <= (1 << 19) &&
            p.tiles * pages < (1 << 29) / Hkv) {
            const int64_t shares = p.tiles * Hkv * pages / 2 + 1;   // of 4 tiles of 32 keys at least
            p.even_rows = true;
            p.shares = (int)(shares < CUS ? shares : CUS);
        }
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
static size_t parts_bytes(const Plan &p, int64_t T, int64_t Hq, int64_t d) {
    const int64_t parts = p.even_rows ? (int64_t)p.shares * 2 * rows::RT
                          : p.shares  ? (int64_t)p.shares * 32
                                      : (p.slots() > 1 ? T * Hq * p.slots() : 0);
    return (size_t)parts * (d + 2) * 4;
}
static size_t workspace(const Plan &p, int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, bool codes) {
    const size_t records = p.even_rows           ? (size_t)(1 + p.tiles * Hkv) * 16
                           : codes && p.shares   ? (size_t)(Bd * Hkv * ((Hq / Hkv + 15) / 16) * 8)
                                                 : 0;
    return parts_bytes(p, T, Hq, d) + records;
}

// NS: sets of columns, 2 where a KV head of a cache in 4 or 8 bits has 8 query heads at most
template <int DT, int D, int FMT, int NS> static int launch(Args a, const Plan &p, hipStream_t s) {
    constexpr size_t lds = 2 * RowSource<DT, D, FMT>::T::BYTES;
    static_assert(sizeof(DecodeLds<D>) <= 65536 && lds <= 65536, "LDS without an attribute");
    const int64_t groups = (int64_t)a.Bd * a.Hkv * ((a.G + 15) / 16);
    a.slots = p.slots();
    if constexpr (FMT != 0) {
        if (p.even_rows) {
            constexpr int bytes = SETS<DT, D, FMT> * 2 * RowSource<DT, D, FMT>::T::BYTES;
            static_assert(bytes >= (SETS<DT, D, FMT> - 1) * 16384, "the sets join in the tiles' place");
            a.slots = p.shares;
            if (hipFuncSetAttribute(reinterpret_cast<const void *>(rows_even_kernel<DT, D, FMT>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
                return HBA_ERR_LAUNCH;
            hipLaunchKernelGGL((rows_even_kernel<DT, D, FMT>), dim3((unsigned)p.shares), dim3(256 * SETS<DT, D, FMT>), bytes, s,
                               a, (int)p.tiles);
            HBA_LAUNCH_CHECK();
            hipLaunchKernelGGL((rows_join_kernel<DT, D>), dim3((unsigned)p.tiles, (unsigned)a.Hkv, rows::RT * D / 1024),
                               dim3(256), 0, s, a, (int)p.tiles);
            HBA_LAUNCH_CHECK();
            return HBA_OK;
        }
    }
    if (p.shares) {
        a.slots = p.shares;
        a.part = p.own_pages;
        const int64_t nrows = (int64_t)a.T * a.Hq;
        if (!abi::launchable(nrows, 256)) return HBA_ERR_UNSUPPORTED;
        if constexpr (FMT == 0)
            hipLaunchKernelGGL((even_kernel<DT, D>), dim3((unsigned)p.shares), dim3(64 * DW), 0, s, a);
        else
            hipLaunchKernelGGL((even_codes_kernel<DT, D, FMT, NS>), dim3((unsigned)p.shares), dim3(64 * DW), 0, s, a);
        HBA_LAUNCH_CHECK();
        hipLaunchKernelGGL((join_kernel<DT, D, 1024 / D, FMT == 0 ? 1 : 2>), dim3((unsigned)nrows), dim3(256), 0, s, a,
                           nrows);
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
        hipLaunchKernelGGL((shared_kernel<DT, D, FMT, NS>), dim3((unsigned)grid), dim3(64 * rows::NW), both, s, a, own,
                           (int)p.ptiles, (int)nshared, (int)groups);
    } else {
        if (p.prefix)
            hipLaunchKernelGGL((rows_kernel<DT, D, FMT, true>),
                               dim3((unsigned)p.ptiles, (unsigned)a.Hkv, (unsigned)p.prefix), dim3(64 * rows::NW), lds,
                               s, a);
        HBA_LAUNCH_CHECK();
        if (a.cu)
            hipLaunchKernelGGL((rows_kernel<DT, D, FMT, false>), dim3((unsigned)p.tiles, (unsigned)a.Hkv, (unsigned)p.own),
                               dim3(64 * rows::NW), lds, s, own);
        else
            hipLaunchKernelGGL((decode_kernel<DT, D, FMT, NS>), dim3((unsigned)groups, (unsigned)p.own), dim3(64 * DW), 0, s,
                               own);
    }
    HBA_LAUNCH_CHECK();
    if (a.slots > 1) {
        if (a.slots > 8)
            hipLaunchKernelGGL((join_kernel<DT, D, SG, 0>), dim3((unsigned)joins), dim3(256), 0, s, a, nrows);
        else
            hipLaunchKernelGGL((join_kernel<DT, D, 1, 0>), dim3((unsigned)joins), dim3(256), 0, s, a, nrows);
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
    if (max_len > (1 << 30) || max_pages > (1 << 24) || shared > max_pages || T > (1 << 30) || Hq > (1 << 30) ||
        Bd > 0x7fffffff || Hkv > 65535)
        return HBA_ERR_UNSUPPORTED;   // (before they are multiplied)
    if (T * Hq > (1 << 30) || Bd * (Hq + 16 * Hkv) > 0x7fffffff) return HBA_ERR_UNSUPPORTED;
    return HBA_OK;
}

// Checks an entry point's arguments and fills in the kernels' (strides and pages in bytes).
static int setup(Args &a, Plan &p, int dtype, const void *q, const int64_t q_strides[2], const float *q_gain, float eps,
                 const float *cos_tab, const float *sin_tab, int64_t n_tab, const void *kr_pages, const void *v_pages,
                 int64_t num_pages, const int32_t *page_table, int64_t max_pages, const int32_t *seq_lens,
                 const float *scales, const int32_t *cu, int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d,
                 int64_t Bk, int64_t W, int64_t S, int64_t shared_pages, int64_t max_len, void *workspace,
                 size_t ws_bytes, void *out, int bits) {
    if (int st = abi::check_dtype_dim(dtype, d)) return st;
    if (Bk != rows::PAGE) return HBA_ERR_UNSUPPORTED;
    if (int st = check(T, Bd, Hq, Hkv, d, W, S, shared_pages, cu == nullptr, max_len, max_pages)) return st;
    if (!q || !q_strides || !kr_pages || !v_pages || !page_table || !seq_lens || !scales || !out || num_pages <= 0 ||
        !cos_tab != !sin_tab || (cos_tab && n_tab <= 0))
        return HBA_ERR_INVALID_ARG;
    const int64_t e = abi::elem_size(dtype), al = 16 / e;
    if (!abi::aligned16(q) || q_strides[0] % al || q_strides[1] % al || !abi::aligned16(kr_pages) ||
        !abi::aligned16(v_pages) || !abi::aligned16(out))
        return HBA_ERR_UNSUPPORTED;
    p = plan(T, Bd, Hq, Hkv, W, S, shared_pages, cu == nullptr, max_len, d, bits);
    const size_t need = paged::workspace(p, T, Bd, Hq, Hkv, d, bits != 0), parts = parts_bytes(p, T, Hq, d);
    if (need && (!workspace || ws_bytes < need)) return HBA_ERR_INVALID_ARG;
    if (need && !abi::aligned16(workspace)) return HBA_ERR_UNSUPPORTED;
    a = {};
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
    a.pml = need ? (float *)workspace + parts / 4 / (d + 2) * d : nullptr;
    a.records = need ? (int *)((char *)workspace + parts) : nullptr;
    return HBA_OK;
}

}  // namespace paged
}  // namespace hba
