// The paged cache in 4 or 8 bits (hba_mx.h): writing new tokens into it, and reading
// tokens back as rows.
//
//   append_kernel   QKNorm, the rotation at each token's position, quantised keys and
//                   values into their pages
//   read_kernel     the last tokens of every sequence as rows of fp32 or bf16
#include "hba_abi.h"
#include "hba_common.h"
#include "hba_mx.h"
#include "hba_ragged.h"

namespace hba {
namespace mx {

constexpr int HALF = 32;                // (2^5) tokens of half a page, whose codes lie apart from the other half's

struct AppendArgs {
    const char *k, *v;                  // [T, Hkv, D]; byte strides of token and head
    int64_t kst, ksh, vst, vsh;
    const int32_t *cu;                  // nullptr: one token per sequence
    int T, Bd, Hkv, maxp;
    const float *gain, *cos, *sin;      // nullptr: no norm, no rotation
    float eps;
    int64_t n_tab, pages;               // positions at/after n_tab are not appended
    const int32_t *table, *lens;
    char *kp, *vp;
};

// Tokens of sequence s and those of them that lie in its pages: positions first ..
// last - 1, from place c0 of the batch on.  (Not in them: positions below 0, past the
// page table or the rotation tables.)
struct Span {
    int from, n, c0, first, last;
    // Runs of 2^n tokens, each from a multiple of 2^n on, that they touch.
    __device__ __forceinline__ int runs(int n) const { return last > first ? ((last - 1) >> n) - (first >> n) + 1 : 0; }
};
__device__ __forceinline__ Span span(const int32_t *cu, const int32_t *lens, int T, int64_t most, int s) {
    Span x;
    if (cu) {
        x.n = ragged::tokens(cu, s, T, x.from);
    } else {
        x.from = s;
        x.n = 1;
    }
    x.c0 = x.from;
    const int64_t L = lens[s];
    int64_t first = L - x.n;
    if (first < 0) {
        x.c0 += (int)min(-first, (int64_t)x.n);
        first = 0;
    }
    x.first = (int)min(first, most);
    x.last = (int)max((int64_t)x.first, min(L, most));
    return x;
}

// The scale of a group whose largest magnitude has the bits `big`: the smallest 2^(b - 127)
// that takes it to at most 1.75 2^EMAX (e2m1 7, of which 6 is left; e4m3 448).  Of the
// energy of normal values e2m1 then loses 1.25% (with the limit 6 1.33%, with 8 1.32%,
// with the better of two scales in each group 1.245%).
template <int F> __device__ __forceinline__ int scale_byte(uint32_t big) {
    constexpr int EMAX = F == 4 ? 2 : 8;
    const int b = (int)(big >> 23) - EMAX + ((big & 0x7fffffu) > 0x600000u);
    // (over 1.75 2^127 the nearest code would stand for 2^128, which fp32 has not)
    return big == 0 ? 0 : big > 0x7f600000u ? 255 : max(b, 1);
}
// Four elements of such a group as codes (rounded to nearest, ties to even), F / 2 bytes.
template <int F> __device__ __forceinline__ uint32_t four(const float (&x)[4], int b) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    if (b == 0 || b == 255) return 0;
    const float to = __uint_as_float((uint32_t)(254 - b) << 23);   // b is at most 252
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = x[i] * to;   // exact, or far below the smallest code
    if constexpr (F == 4) {
        const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], 1.0f, 0);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1) & 0xffffu;
    } else {
        const s16x2 w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, y[0], y[1], 1.0f, false);
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, y[2], y[3], 1.0f, true));
    }
}
// Of 8 lanes that all call it (16 with the last step): the value of the lane 1 away, 2 away, in
// the other four, in the other eight, once those that share a value have been taken together.
template <int STEP> __device__ __forceinline__ uint32_t partner(uint32_t x) {
    constexpr int CTRL = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 4 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int STEP> __device__ __forceinline__ double partner(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)partner<STEP>((uint32_t)(b >> 32)) << 32 | partner<STEP>((uint32_t)b)));
}
// 1 / sqrt(x) to 64 bits' last place or two: each step takes an error e to 5 / 16 e^3.
__device__ __forceinline__ double inverse_root(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double e = fma(-x * y, y, 1.0);
        y = fma(y * e, fma(0.375, e, 0.5), y);
    }
    return x == (double)INFINITY ? 0.0 : y;
}
// The largest magnitude's bits over the 8 lanes of a group (32 elements, 4 each); a NaN's
// are above all.
__device__ __forceinline__ uint32_t largest(const float (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    m = max(m, partner<1>(m));
    m = max(m, partner<2>(m));
    return max(m, partner<4>(m));
}
// Four elements as they lie in memory, and as fp32.
template <int DT> struct Four {
    uint2 w;
    __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const {
        x[0] = __uint_as_float(w.x << 16);
        x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16);
        x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
};
template <> struct Four<0> {
    float4 w;
    __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const {
        x[0] = w.x;
        x[1] = w.y;
        x[2] = w.z;
        x[3] = w.w;
    }
};

// One workgroup per (half of a page that gets tokens, KV head): twice as many as pages, and
// half the rows one after the other in each.  D / 8 lanes a row, each with 4
// elements of its first half and the 4 that they are rotated with.  The norm and the
// rotation run in 64 bits (at half a rate that nothing here needs) and are rounded to
// 32 once: next to a border between two codes the last bit of an fp32 sum would decide
// which one it is, and a key's code would depend on the order of that sum.  (12800 tokens, 4
// KV heads, d = 128, 4 bits: 15.2 us for 33 MB, 6.3 at a copy's rate; 8.7 us of it are vector
// instructions, the rest where each workgroup looks for its sequence and waits for its rows.
// All workgroups at once, 7 waves a SIMD, rather than two rows' loads in flight in 4: 18.5.)
// Codes go to LDS in the page's order (the values' a byte each, by columns) and from
// there in whole 16-byte pieces.  Two tokens' values share a byte (F = 4): where only
// some of a piece's tokens are new, the others are read and put back, by the one
// workgroup that writes this half.
template <int DT, int D, int F> __global__ __launch_bounds__(256, (DT == 0 && D == 128 ? 5 : 7)) void append_kernel(const AppendArgs a) {
    typedef Place<D, F> At;
    constexpr int TPH = D / 8, RPP = 256 / TPH, NP = HALF / RPP, ESZ = DT == 1 ? 2 : 4, NG = D / GROUP;
    constexpr int CB = (int)code_bytes(D, F), VS = HALF + 4;
    __shared__ __align__(16) uint8_t kcodes[CB / 2];
    __shared__ __align__(16) uint8_t vcodes[D * VS];
    __shared__ uint8_t scales[4 * D];   // as in the page, with the first half's: the keys', then the values'
    const int tid = threadIdx.x, g = blockIdx.x / 8 % a.Hkv, slot = blockIdx.x / 8 / a.Hkv * 8 + blockIdx.x % 8;
    const int64_t most = min((int64_t)a.maxp * 64, a.n_tab);
    int s, tile = 0;
    if (a.cu) {
        s = ragged::find(slot, a.Bd, [&](int i) { return span(a.cu, a.lens, a.T, most, i).runs(5); }, tile);
        if (s < 0) return;
    } else {
        s = slot;
        if (s >= a.Bd) return;
    }
    const Span x = span(a.cu, a.lens, a.T, most, s);
    if (x.last <= x.first) return;
    const int half = x.first / HALF + tile, p0 = half * HALF, h = half % 2;
    const int ja = max(x.first - p0, 0), jb = min(x.last - p0, HALF);   // its new tokens
    const int64_t page = a.table[(int64_t)s * a.maxp + half / 2];
    if (page < 0 || page >= a.pages) return;                          // not a page of this cache
    char *kp = a.kp + (page * a.Hkv + g) * page_bytes(D, F), *vp = a.vp + (page * a.Hkv + g) * page_bytes(D, F);
    const int jl = tid % TPH, t0 = 4 * jl;
    const double gain = a.gain ? (double)a.gain[g] : 0.0;
#pragma unroll 1
    for (int pass = 0; pass < NP; ++pass) {
        if (pass * RPP >= jb || pass * RPP + RPP <= ja) continue;     // uniform
        // (a row that is not new stands for the nearest one that is)
        const int j = pass * RPP + tid / TPH, pos = p0 + min(max(j, ja), jb - 1);
        const int64_t tok = x.c0 + (pos - x.first);
        const char *kr = a.k + tok * a.kst + g * a.ksh, *vr = a.v + tok * a.vst + g * a.vsh;
        Four<DT> kx[2], vx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            kx[i].load(kr + (t0 + i * (D / 2)) * ESZ);
            vx[i].load(vr + (t0 + i * (D / 2)) * ESZ);
        }
        float cs[2][4], sn[2][4];
        if (a.cos) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t at = (int64_t)pos * D + t0 + i * (D / 2);
                const f32x4 c = *reinterpret_cast<const f32x4u *>(a.cos + at), s = *reinterpret_cast<const f32x4u *>(a.sin + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    cs[i][e] = c[e];
                    sn[i][e] = s[e];
                }
            }
        }
        float y[2][4], v[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            kx[i].get(y[i]);
            vx[i].get(v[i]);
        }
        if (a.gain || a.cos) {
            double z[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[i][e] = (double)y[i][e];
            if (a.gain) {
                double ss = 0.0;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fma(z[i][e], z[i][e], ss);
                ss += partner<1>(ss);
                ss += partner<2>(ss);
                ss += partner<4>(ss);
                if constexpr (TPH == 16) ss += partner<8>(ss);
                const double ms = ss * (1.0 / D);
                const double f = gain * inverse_root(ms < (double)a.eps ? (double)a.eps : ms);   // (a maximum would lose a NaN)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[i][e] *= f;
            }
            if (a.cos) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double lo = z[0][e], hi = z[1][e];
                    z[0][e] = fma(lo, (double)cs[0][e], -(hi * (double)sn[0][e]));
                    z[1][e] = fma(hi, (double)cs[1][e], lo * (double)sn[1][e]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[i][e] = (float)z[i][e];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = t0 + i * (D / 2), grp = t / GROUP;
            const int kb = scale_byte<F>(largest(y[i])), vb = scale_byte<F>(largest(v[i]));
            const uint32_t kc = four<F>(y[i], kb), vc = four<F>(v[i], vb);
            if constexpr (F == 4) *reinterpret_cast<uint16_t *>(kcodes + At::key(j, t)) = (uint16_t)kc;
            else *reinterpret_cast<uint32_t *>(kcodes + At::key(j, t)) = kc;
#pragma unroll
            for (int e = 0; e < 4; ++e) vcodes[(t + e) * VS + j] = (uint8_t)(F == 4 ? vc >> (4 * e) & 15u : vc >> (8 * e));
            if (jl % 8 == 0) {
                scales[At::key_scale(j, grp) - CB] = (uint8_t)kb;
                scales[2 * D + At::val_scale(j, grp) - CB] = (uint8_t)vb;
            }
        }
    }
    __syncthreads();
    char *kh = kp + h * (CB / 2), *vh = vp + h * (CB / 2);
    for (int c = tid; c < CB / 32; c += 256) {
        // keys: 8 bytes are of one token
        constexpr int TB = D / 4 * F / 8;   // bytes of a lane in a tile
        const int lane = c % 64, b0 = c / 64 * 16;
        bool in[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int mt = (b0 + 8 * i) / TB, l16 = lane % 16;
            const int j = 8 * (l16 >> 2) + 4 * mt + (l16 & 3);
            in[i] = j >= ja && j < jb;
        }
        const u32x4 w = *reinterpret_cast<const u32x4 *>(kcodes + 16 * c);
        if (in[0] && in[1]) {
            *reinterpret_cast<u32x4 *>(kh + 16 * c) = w;
        } else {
            if (in[0]) *reinterpret_cast<u32x2 *>(kh + 16 * c) = u32x2{w[0], w[1]};
            if (in[1]) *reinterpret_cast<u32x2 *>(kh + 16 * c + 8) = u32x2{w[2], w[3]};
        }
        // values: eight tokens of 4 columns, or 2
        const int j0 = 8 * (lane / 16);
        if (j0 + 8 <= ja || j0 >= jb) continue;
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 16 / F; ++i) {
            const uint32_t *col = reinterpret_cast<const uint32_t *>(vcodes + (16 * (16 / F * (c / 64) + i) + lane % 16) * VS + j0);
            if constexpr (F == 4) {
                uint32_t lo = col[0], hi = col[1];
                lo = (lo | lo >> 4) & 0x00ff00ffu;
                hi = (hi | hi >> 4) & 0x00ff00ffu;
                v[i] = ((lo | lo >> 8) & 0xffffu) | (hi | hi >> 8) << 16;
            } else {
                v[2 * i] = col[0];
                v[2 * i + 1] = col[1];
            }
        }
        if (j0 < ja || j0 + 8 > jb) {       // the other tokens' codes stay
            const int lo = max(ja - j0, 0) * F, hi = min(jb - j0, 8) * F;   // bits of the new ones
            const uint64_t m = (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~((1ull << lo) - 1);
            const u32x4 old = *reinterpret_cast<const u32x4 *>(vh + 16 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t mi = F == 4 || i % 2 == 0 ? (uint32_t)m : (uint32_t)(m >> 32);
                v[i] = (v[i] & mi) | (old[i] & ~mi);
            }
        }
        *reinterpret_cast<u32x4 *>(vh + 16 * c) = v;
    }
    for (int c = tid; c < D; c += 256) {
        const int l = c / 2, mt = c % 2, jk = 8 * (l % 16 >> 2) + 4 * mt + (l & 3), jv = c / (8 * NG) * 8 + c % 8;
        if (jk >= ja && jk < jb) kp[CB + l * 4 + 2 * h + mt] = (char)scales[l * 4 + mt];
        if (jv >= ja && jv < jb) vp[CB + h * D + c] = (char)scales[2 * D + c];
    }
}

struct ReadArgs {
    const char *kp, *vp;
    const int32_t *cu, *table, *lens;
    int T, Bd, Hkv, maxp;
    int64_t pages;
    char *k, *v;                        // [T, Hkv, D]
    int run;                            // a workgroup's tokens are 2^run: half a page or all of it
};

// n rows of zeros, the i-th at place at(i) of the batch.
template <int DT, int D, class At> __device__ __forceinline__ void zero_rows(const ReadArgs &a, int g, int n, const At &at) {
    constexpr int ESZ = DT == 1 ? 2 : 4, C = D * ESZ / 16;
    for (int64_t i = threadIdx.x; i < (int64_t)n * C; i += 256) {
        const int64_t to = ((at((int)(i / C)) * a.Hkv + g) * D) * ESZ + i % C * 16;
        *reinterpret_cast<uint4 *>(a.k + to) = uint4{0, 0, 0, 0};
        *reinterpret_cast<uint4 *>(a.v + to) = uint4{0, 0, 0, 0};
    }
}

// Half h of a page: its tokens ja .. jb - 1 to rows at + ja .. of the batch.
template <int DT, int D, int F>
__device__ __forceinline__ void read_half(const ReadArgs &a, const char *kp, const char *vp, int h, int g, int64_t at, int ja,
                                          int jb, typename St<DT>::T *krows, typename St<DT>::T *vrows) {
    constexpr int ESZ = DT == 1 ? 2 : 4, NG = D / GROUP, CB = (int)code_bytes(D, F), RS = D + 16 / ESZ;
    constexpr int TB = D / 4 * F / 8, N8 = 32 / F / 2;    // bytes of a lane in a key tile; runs of 8 codes in a piece
    const int tid = threadIdx.x;
    const char *kh = kp + h * (CB / 2), *vh = vp + h * (CB / 2);
    for (int c = tid; c < CB / 32; c += 256) {
        const int lane = c % 64, l16 = lane % 16, lg = lane / 16;
        const u32x4 kw = *reinterpret_cast<const u32x4 *>(kh + 16 * c), vw = *reinterpret_cast<const u32x4 *>(vh + 16 * c);
        const uint32_t ks = *reinterpret_cast<const uint32_t *>(kp + CB + (l16 + 16 * (lg * (D / 4) / GROUP)) * 4) >> (16 * h);
        u32x2 vs[N8];
#pragma unroll
        for (int r = 0; r < N8; ++r)
            vs[r] = *reinterpret_cast<const u32x2 *>(vp + CB + ((4 * h + lg) * NG + (N8 * (c / 64) + r) / 2) * 8);
        // keys: runs of 8 elements of a token
#pragma unroll
        for (int r = 0; r < N8; ++r) {
            const int b = c / 64 * 16 + r * F, mt = b / TB, t = D / 4 * lg + b % TB * 8 / F;
            const float scale = power(ks, mt);
            const uint32_t w[2] = {kw[F == 4 ? r : 2 * r], kw[F == 4 ? r : 2 * r + 1]};
            typename St<DT>::T *to = krows + (8 * (l16 >> 2) + 4 * mt + (l16 & 3)) * RS + t;
            if constexpr (DT == 1) {
                *reinterpret_cast<u32x4 *>(to) = __builtin_bit_cast(u32x4, eight<F>(w, scale));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x2 x = pair<F>(w[i], scale, F == 4 ? 2 * i : 0), y = pair<F>(w[i], scale, F == 4 ? 2 * i + 1 : 1);
                    *reinterpret_cast<f32x4 *>(to + 4 * i) = f32x4{x[0], x[1], y[0], y[1]};
                }
            }
        }
        // values: runs of 8 tokens of a column.  bf16 ones in twos: lanes l and l ^ 1, of two columns,
        // have the even and the odd token of both.
#pragma unroll
        for (int r = 0; r < N8; ++r) {
            const int t = 16 * (N8 * (c / 64) + r) + l16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = vw[F == 4 ? r : 2 * r + (i >> 1)];
                const int p = F == 4 ? i : i & 1;
                const float s0 = power(vs[r][i >> 1], 2 * (i & 1)), s1 = power(vs[r][i >> 1], 2 * (i & 1) + 1);
                if constexpr (DT == 1) {
                    const uint32_t lo = __builtin_bit_cast(uint32_t, two<F>(w, s0, p));
                    const uint32_t hi = __builtin_bit_cast(uint32_t, two<F>(w, s1, p));
                    const uint32_t mine = __builtin_amdgcn_perm(hi, lo, 0x07060100), other = partner<1>(mine);
                    const int odd = l16 & 1;
                    *reinterpret_cast<uint32_t *>(vrows + (8 * lg + 2 * i + odd) * RS + t - odd) =
                        __builtin_amdgcn_perm(other, mine, odd ? 0x03020706 : 0x05040100);
                } else {
                    vrows[(8 * lg + 2 * i) * RS + t] = pair<F>(w, s0, p)[0];
                    vrows[(8 * lg + 2 * i + 1) * RS + t] = pair<F>(w, s1, p)[1];
                }
            }
        }
    }
    __syncthreads();
    constexpr int C = D * ESZ / 16;
    for (int i = ja * C + tid; i < jb * C; i += 256) {
        const int64_t to = (((at + i / C) * a.Hkv + g) * D) * ESZ + i % C * 16;
        const int from = i / C * RS + i % C * (16 / ESZ);
        *reinterpret_cast<uint4 *>(a.k + to) = *reinterpret_cast<const uint4 *>(krows + from);
        *reinterpret_cast<uint4 *>(a.v + to) = *reinterpret_cast<const uint4 *>(vrows + from);
    }
}

// One workgroup per (half of a page that holds some of the tokens, KV head).  Keys and values go
// through LDS as rows, so that whole rows are written.  Tokens that lie in no page give
// 0: those of a sequence are tiles behind its pages', those of no sequence (before
// cu[0], behind cu[Bd]) are left to the workgroups that have nothing else.  A workgroup's search
// for its sequence is worth a whole page's work where there are enough of those: by pages and by
// halves, bf16, 94000 tokens, 2 KV heads, d = 64, 8 bits 14.8 us (4.9 TB/s) and 16.6, 40000 8.3 and
// 9.5, 12800 5.3 and 5.3, 3000 4.4 and 4.0; 4 heads, d = 128, 4 bits, 40000 tokens 19.0 and 20.2,
// 12800 9.0 and 9.3, 3000 5.7 and 5.1.  (Keys and values an element at a time instead of packed in
// words: 17.5 for the first, 12.6 for 12800 tokens of the second.)
template <int DT, int D, int F> __global__ __launch_bounds__(256) void read_kernel(const ReadArgs a) {
    typedef typename St<DT>::T T;
    constexpr int RS = D + (DT == 1 ? 8 : 4);
    __shared__ __align__(16) T krows[HALF * RS], vrows[HALF * RS];
    const int g = blockIdx.y;
    const int64_t most = (int64_t)a.maxp * 64;
    const auto tiles = [&](int i) {
        const Span x = span(a.cu, a.lens, a.T, most, i);
        return x.runs(a.run) + (x.n - (x.last - x.first) + 63) / 64;
    };
    int tile = 0, s = blockIdx.x;
    if (a.cu) {
        s = ragged::find(blockIdx.x, a.Bd, tiles, tile);
        if (s < 0) {
            const int used = ragged::total<256>(a.Bd, tiles), w = blockIdx.x - used, of = gridDim.x - used;
            const int lo = max(0, min(a.T, a.cu[0])), hi = max(lo, min(a.T, a.cu[a.Bd]));
            const int n = lo + a.T - hi, per = (n + of - 1) / of, i0 = min((int64_t)w * per, (int64_t)n);
            zero_rows<DT, D>(a, g, min(per, n - i0), [&](int i) { return (int64_t)(i0 + i < lo ? i0 + i : i0 + i - lo + hi); });
            return;
        }
    }
    const Span x = span(a.cu, a.lens, a.T, most, s);
    const int np = x.runs(a.run), run = (x.first >> a.run) + tile;
    if (tile >= np) {
        const int front = x.c0 - x.from, have = x.last - x.first, i0 = (tile - np) * 64;
        zero_rows<DT, D>(a, g, min(64, x.n - have - i0),
                         [&](int i) { return (int64_t)(i0 + i < front ? x.from + i0 + i : x.from + i0 + i + have); });
        return;
    }
    const int64_t page = a.table[(int64_t)s * a.maxp + (run << a.run) / 64];
    if (page < 0 || page >= a.pages) {                    // not a page of this cache
        const int ja = max(x.first, run << a.run), jb = min((int64_t)x.last, ((int64_t)run + 1) << a.run);
        zero_rows<DT, D>(a, g, jb - ja, [&](int i) { return (int64_t)x.c0 + ja + i - x.first; });
        return;
    }
    const char *kp = a.kp + (page * a.Hkv + g) * page_bytes(D, F), *vp = a.vp + (page * a.Hkv + g) * page_bytes(D, F);
    for (int i = 0; i < (1 << a.run); i += HALF) {
        const int p0 = (run << a.run) + i, h = p0 / HALF % 2, ja = max(x.first - p0, 0), jb = min(x.last - p0, HALF);
        if (ja >= jb) continue;
        const int64_t at = (int64_t)x.c0 + p0 - x.first;   // the place of the half's token 0
        __syncthreads();                                   // the rows of the other half are written
        read_half<DT, D, F>(a, kp, vp, h, g, at, ja, jb, krows, vrows);
    }
}

static int check(int64_t T, int64_t Bd, int64_t Hkv, int64_t d, int64_t Bk, int64_t bits, int64_t max_pages,
                 int64_t num_pages, const int32_t *cu) {
    if (d != 64 && d != 128) return HBA_ERR_UNSUPPORTED;
    if (T < 0 || Bd <= 0 || Hkv <= 0 || max_pages <= 0 || num_pages <= 0 || (!cu && T != Bd)) return HBA_ERR_INVALID_ARG;
    if (Bk != 64 || (bits != 4 && bits != 8)) return HBA_ERR_UNSUPPORTED;
    if (T > (1 << 30) || Bd > (1 << 24) || Hkv > 65535 || max_pages > (1 << 24)) return HBA_ERR_UNSUPPORTED;
    return HBA_OK;
}

}  // namespace mx
}  // namespace hba

using namespace hba;

#define HBA_DISPATCH_BITS(dtype, d, bits, M)            \
    do {                                                \
        if ((dtype) == HBA_DTYPE_F32) {                 \
            if ((d) == 64 && (bits) == 4) M(0, 64, 4);  \
            else if ((d) == 64) M(0, 64, 8);            \
            else if ((bits) == 4) M(0, 128, 4);         \
            else M(0, 128, 8);                          \
        } else {                                        \
            if ((d) == 64 && (bits) == 4) M(1, 64, 4);  \
            else if ((d) == 64) M(1, 64, 8);            \
            else if ((bits) == 4) M(1, 128, 4);         \
            else M(1, 128, 8);                          \
        }                                               \
    } while (0)

extern "C" int hba_kv_append_mx(int dtype, const void *k, const int64_t k_strides[2], const void *v,
                                const int64_t v_strides[2], const int32_t *cu, int64_t T, const float *k_gain, float eps,
                                const float *cos_tab, const float *sin_tab, int64_t n_tab, const int32_t *page_table,
                                int64_t max_pages, const int32_t *seq_lens, int64_t Bd, int64_t Hkv, int64_t d,
                                int64_t Bk, int64_t bits, int64_t num_pages, void *k_pages, void *v_pages,
                                void *stream) {
    if (int st = abi::check_dtype_dim(dtype, d)) return st;
    if (int st = mx::check(T, Bd, Hkv, d, Bk, bits, max_pages, num_pages, cu)) return st;
    if (!k || !k_strides || !v || !v_strides || !page_table || !seq_lens || !k_pages || !v_pages || !cos_tab != !sin_tab ||
        (cos_tab && n_tab <= 0))
        return HBA_ERR_INVALID_ARG;
    const int64_t e = abi::elem_size(dtype), al = 16 / e;
    if (!abi::aligned16(k) || !abi::aligned16(v) || k_strides[0] % al || k_strides[1] % al || v_strides[0] % al ||
        v_strides[1] % al || !abi::aligned16(k_pages) || !abi::aligned16(v_pages))
        return HBA_ERR_UNSUPPORTED;
    if (T == 0) return HBA_OK;
    mx::AppendArgs a = {};
    a.k = (const char *)k;
    a.v = (const char *)v;
    a.kst = k_strides[0] * e;
    a.ksh = k_strides[1] * e;
    a.vst = v_strides[0] * e;
    a.vsh = v_strides[1] * e;
    a.cu = cu;
    a.T = (int)T;
    a.Bd = (int)Bd;
    a.Hkv = (int)Hkv;
    a.maxp = (int)max_pages;
    a.gain = k_gain;
    a.cos = cos_tab;
    a.sin = sin_tab;
    a.eps = eps;
    a.n_tab = cos_tab ? n_tab : INT64_MAX;
    a.pages = num_pages;
    a.table = page_table;
    a.lens = seq_lens;
    a.kp = (char *)k_pages;
    a.vp = (char *)v_pages;
    // c tokens touch at most c and at most c / 32 + 2 halves of pages
    const int64_t slots = !cu || T < T / mx::HALF + 2 * Bd ? T : T / mx::HALF + 2 * Bd, blocks = (slots + 7) / 8 * 8 * Hkv;
    if (!abi::launchable(blocks, 256)) return HBA_ERR_UNSUPPORTED;
#define HBA_APPEND_MX(DT, D, F) \
    hipLaunchKernelGGL((mx::append_kernel<DT, D, F>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
    HBA_DISPATCH_BITS(dtype, d, bits, HBA_APPEND_MX);
#undef HBA_APPEND_MX
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_kv_read_mx(int dtype, const void *k_pages, const void *v_pages, int64_t num_pages,
                              const int32_t *page_table, int64_t max_pages, const int32_t *seq_lens, const int32_t *cu,
                              int64_t T, int64_t Bd, int64_t Hkv, int64_t d, int64_t Bk, int64_t bits, void *k, void *v,
                              void *stream) {
    if (int st = abi::check_dtype_dim(dtype, d)) return st;
    if (int st = mx::check(T, Bd, Hkv, d, Bk, bits, max_pages, num_pages, cu)) return st;
    if (!k_pages || !v_pages || !page_table || !seq_lens || !k || !v) return HBA_ERR_INVALID_ARG;
    if (!abi::aligned16(k) || !abi::aligned16(v) || !abi::aligned16(k_pages) || !abi::aligned16(v_pages))
        return HBA_ERR_UNSUPPORTED;
    if (T == 0) return HBA_OK;
    mx::ReadArgs a = {};
    a.kp = (const char *)k_pages;
    a.vp = (const char *)v_pages;
    a.cu = cu;
    a.table = page_table;
    a.lens = seq_lens;
    a.T = (int)T;
    a.Bd = (int)Bd;
    a.Hkv = (int)Hkv;
    a.maxp = (int)max_pages;
    a.pages = num_pages;
    a.k = (char *)k;
    a.v = (char *)v;
    // A sequence's c tokens are at most c tiles, and at most c / 32 + 3: halves of pages, and those
    // in none.  One workgroup more, for tokens of no sequence.
    a.run = (T >> 5) * Hkv > 2048 ? 6 : 5;
    const int64_t tiles = (T >> a.run) + 3 * Bd, slots = !cu ? Bd : (T < tiles ? T : tiles) + 1;
    if (!abi::launchable(slots, 256)) return HBA_ERR_UNSUPPORTED;
#define HBA_READ_MX(DT, D, F)                                                                                      \
    hipLaunchKernelGGL((mx::read_kernel<DT, D, F>), dim3((unsigned)slots, (unsigned)Hkv), dim3(256), 0,            \
                       (hipStream_t)stream, a)
    HBA_DISPATCH_BITS(dtype, d, bits, HBA_READ_MX);
#undef HBA_READ_MX
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}
