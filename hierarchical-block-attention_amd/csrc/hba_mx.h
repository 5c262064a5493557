// The paged cache in 4 or 8 bits: what a page holds, and how it becomes operands.
//
// A page (64 tokens of one KV head, D elements each) is 64 D F / 8 bytes of codes
// and 2 D bytes of scales.  Codes are e2m1 (F = 4) or e4m3 (F = 8); the elements
// 32 g .. 32 g + 31 of a token share the scale 2^(b - 127), b a byte (b = 255, codes 0:
// they are NaN).  A value has at most 4 bits of mantissa, so it is exact in bf16 (from 2^-130
// on: the smallest codes of F = 8 at b < 3 are rounded to bf16's last step, 2^-133), and one
// instruction makes two of them from their codes and scale.
//
// The order is that of the decode kernel's MFMA tiles (16 keys; the tile and row of
// a key, and the lane of a value, as in the bf16 pages, hba_common.h).  Lane
// L = l16 + 16 lg has of every tile of keys the D/4 neighbours from D/4 lg on (at
// D = 128 a group with its scale), of every 32 values 8 tokens in each column
// 16 dt + l16; its codes are a stream of bytes,
//   keys    byte (mt D/4 + t % (D/4)) F / 8, lg = t / (D/4),
//   values  of half h: byte (dt 8 + e) F / 8
// stored as 16-byte pieces: byte x of lane L at (x / 16 * 64 + L) * 16 + x % 16, so
// that a wave loads whole KBs (values: half h begins at piece h D F / 256).  With
// F = 4 the even element, or token, has a byte's low half.  The scales: a key's at
// (l16 + 16 g) 4 + mt, so that a lane's four tiles are one word; a value's at
// ((h 4 + lg) D/32 + g) 8 + e, so that a lane's eight tokens are two.
#pragma once

#include "hba_common.h"
#include "hba_rows.h"

namespace hba {
namespace mx {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
using hba::f32x16;
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // of a table that may begin anywhere
template <int N> struct number {
    static constexpr int value = N;
};

constexpr int GROUP = 32;
constexpr int64_t code_bytes(int64_t d, int bits) { return 64 * d * bits / 8; }
constexpr int64_t page_bytes(int64_t d, int bits) { return code_bytes(d, bits) + 2 * d; }

// Bytes of key j's element t and of its group's scale, of value j's.
template <int D, int F> struct Place {
    static __host__ __device__ __forceinline__ int piece(int x, int lane) { return (x / 16 * 64 + lane) * 16 + x % 16; }
    static __host__ __device__ __forceinline__ int tile(int j) { return 2 * (j >> 5) + ((j >> 2) & 1); }
    static __host__ __device__ __forceinline__ int row(int j) { return 4 * ((j & 31) >> 3) + (j & 3); }
    static __host__ __device__ __forceinline__ int key(int j, int t) {
        return piece((tile(j) * (D / 4) + t % (D / 4)) * F / 8, row(j) + 16 * (t / (D / 4)));
    }
    static __host__ __device__ __forceinline__ int key_scale(int j, int g) {
        return (int)code_bytes(D, F) + (row(j) + 16 * g) * 4 + tile(j);
    }
    static __host__ __device__ __forceinline__ int val(int j, int t) {
        return (j >> 5) * (D * F / 256) * 1024 + piece(((t >> 4) * 8 + (j & 7)) * F / 8, (t & 15) + 16 * ((j & 31) >> 3));
    }
    static __host__ __device__ __forceinline__ int val_scale(int j, int g) {
        return (int)code_bytes(D, F) + ((j >> 3) * (D / GROUP) + g) * 8 + (j & 7);
    }
};

// Byte k of four as the power of two that it stands for.  (255 gives infinity here:
// its group's codes are 0, and 0 times infinity the NaN it stands for.)
__device__ __forceinline__ float power(uint32_t w, int k) {
    return __uint_as_float((k == 0 ? w << 23 : k == 1 ? w << 15 : k == 2 ? w << 7 : w >> 1) & 0x7f800000u);
}

// Two codes times a power of two: codes 2 i, 2 i + 1 of a word.
template <int F> __device__ __forceinline__ bf16x2 two(uint32_t w, float scale, int i) {
    if constexpr (F == 4)
        return i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)
               : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)
               : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    else
        return i == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)
                      : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
}
// Eight of them as an operand: 32 bits (F = 4) or 64 from word w on.
template <int F> __device__ __forceinline__ bf16x8 eight(const uint32_t *w, float scale) {
    bf16x2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = F == 4 ? two<F>(w[0], scale, i) : two<F>(w[i >> 1], scale, i & 1);
    const auto a = __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3), b = __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// c + a 16x16 product over 128 elements: e2m1 codes with byte KB of ks as their scale
// (lane l: row l % 16, elements 32 (l / 16) ..), e2m3 with byte QB of qs (columns).
template <int KB, int QB> __device__ __forceinline__ f32x4 product6(u32x4 k, i32x8 q, f32x4 c, int ks, int qs) {
    const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, c, 4, 2, KB, ks, QB, qs);
}
// Codes 2 i, 2 i + 1 of a word times a power of two, in fp32 (exact).
template <int F> __device__ __forceinline__ f32x2 pair(uint32_t w, float scale, int i) {
    if constexpr (F == 4)
        return i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0)
               : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1)
               : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2)
                        : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    else
        return i == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false)
                      : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
}
// One code (the low F bits) as fp32, exact.
template <int F> __device__ __forceinline__ float one(uint32_t code, float scale) {
    f32x2 r;
    if constexpr (F == 4) r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0);
    else r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code, scale, false);
    return r[0];
}

// `bytes` of memory from a wave-uniform address on, for loads at a lane's 32-bit offset: no
// 64-bit addresses in vector registers, whose reuse would have to wait for loads.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const char *p, int bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32 |
                       (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a);
    return __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)u, 0, bytes, 0x00027000);
}
__device__ __forceinline__ u32x4 load16(Buffer b, uint32_t lane, uint32_t at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, lane + at, 0, 0));
}
__device__ __forceinline__ u32x2 load8(Buffer b, uint32_t lane, uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(b, lane + at, 0, 0));
}
__device__ __forceinline__ uint32_t load4(Buffer b, uint32_t lane, uint32_t at) {
    return __builtin_amdgcn_raw_buffer_load_b32(b, lane + at, 0, 0);
}

// c + a 32x32 product over 64 elements: e2m1 codes with byte KB of ks as their scale (lane
// l: row l % 32, elements 32 (l / 32) ..), e2m3 with byte QB of qs (columns).
template <int KB, int QB> __device__ __forceinline__ f32x16 product6(u32x4 k, i32x8 q, f32x16 c, int ks, int qs) {
    const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, q, c, 4, 2, KB, ks, QB, qs);
}
// 32 elements as e2m3 with the scale f, and back.  The conversions write their results over
// several cycles: these must not lie where an operand does, as the compiler places them where
// the operand is needed no more (the scale of a query's last part, whose elements then were of
// other scales: 0.5% off the outputs of bf16 at d = 128).  So the operands stay in use; the build
// looks for others.  (Conversions of two elements may lie there: the compiler places results of
// theirs on their codes and scales in all of read_kernel's forms, whose rows are the definition's
// bit for bit.)
template <bool LAST> __device__ __forceinline__ u32x6 to6(f32x16 even, f32x16 odd, float f) {
    u32x6 r = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, f);
    asm volatile("" : "+v"(r) : "v"(f));
    if (LAST) asm volatile("" : "+v"(r) : "v"(even), "v"(odd));   // (else they are used again)
    return r;
}
__device__ __forceinline__ f32x32 from6(u32x6 x, float f) {
    f32x32 r = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(x, f);
    asm volatile("" : "+v"(r) : "v"(x), "v"(f));
    return r;
}
// A query's 32 elements of a group as N parts of e2m3 (6 bits), each with a power of two
// of its own: the largest magnitude goes to (3.75, 7.5], what the rounding leaves (1/4 of
// the first unit at most) times 2^4, of every later one times 2^5.  N parts leave at most
// 2^-(5 N - 1.1) of the largest magnitude (3 of bf16 queries: 2^-13.9).
template <int N> struct Query6 {
    u32x6 q[N];
    int scale[N];   // bytes
};
template <int N> __device__ __forceinline__ Query6<N> parts6(const float (&y)[32]) {
    Query6<N> r;
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) big = max(big, __float_as_uint(y[e]) & 0x7fffffffu);
    const int b = (int)(big >> 23) - 2 + ((big & 0x7fffffu) > 0x700000u);
    const bool bad = big >= 0x7f800000u;   // 255 makes every logit NaN
    f32x16 x[2];                           // even and odd elements, as the conversion takes them
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e & 1][e >> 1] = bad ? 0.0f : y[e];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        r.scale[n] = bad ? 255 : max(n == 0 ? b : b + 1 - 5 * n, 1);
        const float f = __uint_as_float((uint32_t)(bad ? 127 : r.scale[n]) << 23);
        if (n == N - 1) {
            r.q[n] = to6<true>(x[0], x[1], f);
        } else {
            r.q[n] = to6<false>(x[0], x[1], f);
            const f32x32 back = from6(r.q[n], f);
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e & 1][e >> 1] -= back[e];
        }
    }
    return r;
}
// The columns of a 32x32 product: lane l has column l % 32, and of every 64 elements
// those 32 (l / 32) .. + 31, in N parts.
template <int D, int N> struct Rows6 {
    i32x8 q[D / 64][N];
    int qs[D / 64][2];   // scales, a byte each
    // x[s]: the elements 64 s + 32 (l / 32) .. of the column
    __device__ __forceinline__ void set(const float (&x)[D / 64][32]) {
#pragma unroll
        for (int s = 0; s < D / 64; ++s) {
            const Query6<N> r = parts6<N>(x[s]);
            qs[s][0] = qs[s][1] = 0;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                q[s][n] = i32x8{(int)r.q[n][0], (int)r.q[n][1], (int)r.q[n][2], (int)r.q[n][3], (int)r.q[n][4],
                                (int)r.q[n][5], 0, 0};
                qs[s][n / 4] |= r.scale[n] << (8 * (n % 4));
            }
        }
    }
    // word w of what it holds
    static constexpr int SCALES = (N + 3) / 4, WORDS = D / 64 * (6 * N + SCALES);
    __device__ __forceinline__ int &word(int w) {
        const int s = w / (6 * N + SCALES), i = w % (6 * N + SCALES);
        return i < 6 * N ? reinterpret_cast<int *>(&q[s][i / 6])[i % 6] : qs[s][i - 6 * N];
    }
    // element e of x[s] again
    __device__ __forceinline__ void get(int s, float (&x)[32]) const {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0.0f;
#pragma unroll
        for (int n = N - 1; n >= 0; --n) {
            const u32x6 w = {(uint32_t)q[s][n][0], (uint32_t)q[s][n][1], (uint32_t)q[s][n][2],
                             (uint32_t)q[s][n][3], (uint32_t)q[s][n][4], (uint32_t)q[s][n][5]};
            const uint32_t b = (uint32_t)qs[s][n / 4] >> (8 * (n % 4)) & 255u;
            const f32x32 y = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, __uint_as_float(b << 23));   // (not from6: it would spill; the build looks here too)
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] += y[e];
        }
    }
};

// ------------------------------------------------------------ staged tiles --
// Keys and values of one KV head, for attend: a tile's codes are loaded into
// registers while the tile before it is worked on.  Values, and keys of 8 bits, become
// the bf16 tile that rows::PageKV stages; keys of 4 bits stay codes (CODES), with their
// scales behind them, and the queries are Rows6.  A thread has 16 codes of the keys and
// 16 of the values: of a key, half a group at most; of the values, eight tokens in two
// columns of a group.
template <int DT, int D, int F> struct TileKV {
    typedef typename rows::Op<DT>::F Q;    // the queries' operand
    typedef rows::PageKV<1, D> Bf16;
    typedef Place<D, F> At;
    static constexpr bool CODES = F == 4;
    static constexpr int KT = Bf16::KT, TP = Bf16::TP, NG = D / GROUP, NB = 16 * F / 8;   // NB: a thread's bytes of codes
    static constexpr int KEYB = CODES ? KT * D / 2 + 256 : KT * D * 2, BYTES = KEYB + KT * D * 2;
    const char *k, *v;            // the KV head's place in page 0
    int64_t page;                 // bytes from page to page
    const int32_t *table;
    int len;
    int64_t pages;
    int half;                     // the place in its page of the tile that is staged next
    int expected;                 // the tile after it, and (in all lanes) its page's number as it lies in the table
    uint32_t number;
    uint32_t kc[NB / 4], vc[NB / 4], ks, vs[2];   // its codes and scales
    // The tiles: of a list (place i < ns: sinks, tile i; else tile wt0 + i - ns) the places from,
    // from + by .. last.
    int ns, wt0, from, by, last;

    __device__ __forceinline__ int tile(int it) const {
        const int i = min(from + it * by, last);
        return i < ns ? i : wt0 + i - ns;
    }
    __device__ __forceinline__ bool past(int it) const { return from + it * by > last; }
    __device__ __forceinline__ int64_t at(int lp) const {
        typedef const __attribute__((address_space(4))) int32_t *uniform;
        const int p = ((uniform)(uintptr_t)table)[__builtin_amdgcn_readfirstlane(lp)];
        return p < 0 ? 0 : (p < pages ? p : pages - 1);   // never outside the cache
    }
    // The thread's 16 codes q = thread / 64 of its lane's stream in this tile: a tile of
    // 16 keys (D = 64) or half of one (128); columns 32 g .. of 32 tokens.
    static __device__ __forceinline__ int unit() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % rows::NW; }
    static __device__ __forceinline__ void get(uint32_t (&to)[NB / 4], Buffer b, uint32_t lane, uint32_t at) {
        if constexpr (F == 4) {
            const u32x2 x = load8(b, lane, at);
            __builtin_memcpy(to, &x, sizeof x);
        } else {
            const u32x4 x = load16(b, lane, at);
            __builtin_memcpy(to, &x, sizeof x);
        }
    }
    // Page numbers come a tile ahead, and by vector loads: a scalar load would be waited for
    // with the next LDS read.
    __device__ __forceinline__ void next(int it) {
        const int tile = this->tile(it), after = this->tile(it + 1);
        constexpr int HB = (int)page_bytes(D, F), CB = (int)code_bytes(D, F);
        const int p = __builtin_amdgcn_readfirstlane((int)number);
        const int64_t id = tile == expected ? max((int64_t)0, min((int64_t)p, pages - 1)) : at(tile / TP);
        expected = after;
        number = load4(buffer((const char *)table, 0x7fffffff), after / TP * 4, 0);
        half = tile % TP;
        const int q = unit(), lane = threadIdx.x & 63, lg = lane >> 4, x = q * NB;
        const uint32_t first = half * (4 * NB) * 64 + x / 16 * 1024 + x % 16;
        const Buffer kp = buffer(k + id * page, HB), vp = buffer(v + id * page, HB);
        get(kc, kp, lane * 16, first);
        get(vc, vp, lane * 16, first);
        // the scales: as they lie there, for a tile of codes
        ks = load4(kp, (CODES ? lane % (16 * NG) : (lane & 15) + 16 * (lg * (D / 4) / GROUP)) * 4, CB);
        const int h = D == 64 ? q >> 1 : half, vg = D == 64 ? q & 1 : q;
        const u32x2 s = load8(vp, lg * (NG * 8), CB + (h * 4 * NG + vg) * 8);
        vs[0] = s[0];
        vs[1] = s[1];
    }
    __device__ __forceinline__ void stage(int it, uint32_t lds) {
        const int tile = this->tile(it);
        typedef __attribute__((address_space(3))) u32x4 *out;
        const int q = unit(), lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
        if constexpr (CODES) {
            const int x = q * NB;
            *(__attribute__((address_space(3))) u32x2 *)(uintptr_t)(lds + (x / 16 * 64 + lane) * 16 + x % 16) = u32x2{kc[0], kc[1]};
            // the tile's scales in the low bytes, by all waves alike
            *(__attribute__((address_space(3))) uint32_t *)(uintptr_t)(lds + KT * D / 2 + lane % (16 * NG) * 4) = ks >> (16 * half);
        } else {
            const int mt = D == 64 ? q : q >> 1, t0 = D / 4 * lg + (D == 64 ? 0 : 16 * (q & 1));   // key tile here, first element
            const int pt = D == 64 ? mt : 2 * half + mt;                                           // and in its page
            const float sc = __uint_as_float((ks >> (8 * pt) & 255u) << 23);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int t = t0 + 8 * c;
                *(out)(uintptr_t)(lds + ((mt * (D / 32) + (t >> 5)) * 64 + l16 + 16 * ((t >> 3) & 3)) * 16) =
                    __builtin_bit_cast(u32x4, eight<F>(kc + c * (F / 4), sc));
            }
        }
        const int h = D == 64 ? q >> 1 : 0, g = D == 64 ? q & 1 : q;
        const int left = len - tile * KT - 32 * h - 8 * lg;   // of the thread's eight tokens, those of the sequence
        if (tile * KT + KT > len) {                           // the same for the workgroup
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int n = left - 4 * w;
                const uint32_t m = n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1;
                vs[w] &= m;
                if constexpr (F == 8) {                       // a code may be a NaN
                    vc[w] &= m;
                    vc[2 + w] &= m;
                }
            }
        }
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = power(vs[e >> 2], e & 3);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // tokens 2 i and 2 i + 1 have a scale each
                const uint32_t w = vc[F == 4 ? c : 2 * c + (i >> 1)];
                const int p = F == 4 ? i : i & 1;
                const uint32_t lo = __builtin_bit_cast(uint32_t, two<F>(w, s[2 * i], p));
                const uint32_t hi = __builtin_bit_cast(uint32_t, two<F>(w, s[2 * i + 1], p));
                r[i] = __builtin_amdgcn_perm(hi, lo, 0x07060100);
            }
            *(out)(uintptr_t)(lds + KEYB + (((2 * g + c) * (KT / 32) + h) * 64 + lane) * 16) = r;
        }
    }
    static __device__ __forceinline__ int key(int r, int hf) { return Bf16::key(r, hf); }
    static __device__ __forceinline__ bf16x8 vf(const char *t, int kt, int dt, int u, int lane) {
        const int x = 32 * dt + (lane & 31);
        return rows::Op<1>::load(t + KEYB + (((x >> 4) * (KT / 32) + kt) * 64 + (x & 15) + 16 * (2 * u + (lane >> 5))) * 16);
    }
    // Operands of 32 keys (in PageKV's order), and c + their products with the queries.
    struct Keys {
        u32x4 k[CODES ? D / 64 : D / 16];
        int scale[CODES ? D / 64 : 1];
    };
    static __device__ __forceinline__ Keys keys(const char *t, int kt, int lane) {
        Keys r;
        if constexpr (CODES) {
            const int x = lane & 31, hf = lane >> 5, l16 = 8 * (x >> 4) + 4 * ((x >> 2) & 1) + (x & 3), odd = (x >> 3) & 1;
#pragma unroll
            for (int s = 0; s < D / 64; ++s) {
                const int g = 2 * s + hf;
                if constexpr (D == 64) {   // a group is the pieces' halves in two places
                    const char *p = t + kt * 1024 + (l16 + 32 * g) * 16 + 8 * odd;
                    const u32x2 lo = *reinterpret_cast<const u32x2 *>(p), hi = *reinterpret_cast<const u32x2 *>(p + 256);
                    r.k[s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
                } else {
                    r.k[s] = *reinterpret_cast<const u32x4 *>(t + (odd * 64 + l16 + 16 * g) * 16);
                }
                r.scale[s] = (int)(*reinterpret_cast<const uint32_t *>(t + KT * D / 2 + (l16 + 16 * g) * 4) >> (8 * odd));
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) r.k[ks] = __builtin_bit_cast(u32x4, Bf16::kf(t, kt, ks, lane));
        }
        return r;
    }
    static __device__ __forceinline__ f32x16 logits(const Keys &k, int, const Q (&q)[D / 16], const Q *qlo, f32x16 c) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const bf16x8 kf = __builtin_bit_cast(bf16x8, k.k[ks]);
            c = rows::Op<DT>::mma(kf, q[ks], c);
            if constexpr (DT == 1) c = rows::Op<DT>::mma(kf, qlo[ks], c);
        }
        return c;
    }
    template <int N> static __device__ __forceinline__ f32x16 logits(const Keys &k, int kt, const Rows6<D, N> &q, const Q *, f32x16 c) {
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
            c = kt == 0 ? products<0>(k.k[s], q.q[s], c, k.scale[s], q.qs[s]) : products<2>(k.k[s], q.q[s], c, k.scale[s], q.qs[s]);
        return c;
    }
    template <int KB, int N> static __device__ __forceinline__ f32x16 products(u32x4 k, const i32x8 (&q)[N], f32x16 c, int ks,
                                                                               const int (&qs)[2]) {
        c = product6<KB, 0>(k, q[0], c, ks, qs[0]);
        if constexpr (N > 1) c = product6<KB, 1>(k, q[1], c, ks, qs[0]);
        if constexpr (N > 2) c = product6<KB, 2>(k, q[2], c, ks, qs[0]);
        if constexpr (N > 3) c = product6<KB, 3>(k, q[3], c, ks, qs[0]);
        if constexpr (N > 4) c = product6<KB, 0>(k, q[4], c, ks, qs[1]);
        if constexpr (N > 5) c = product6<KB, 1>(k, q[5], c, ks, qs[1]);
        return c;
    }
    // one key, for attend_each
    static __device__ __forceinline__ float value(const char *p, int at_code, int at_scale, int odd) {
        const uint32_t c = (uint8_t)p[at_code];
        return one<F>(F == 4 ? c >> (4 * odd) : c, __uint_as_float((uint32_t)(uint8_t)p[at_scale] << 23));
    }
    template <int N> __device__ __forceinline__ float dot(const Rows6<D, N> &q, const Q *, int j, int hf) const {
        const char *p = k + at(j / rows::PAGE) * page;
        const int jp = j % rows::PAGE;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < D / 64; ++s) {
            float x[32];
            q.get(s, x);
            const int g = 2 * s + hf;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                sum = fmaf(x[e], value(p, At::key(jp, 32 * g + e), At::key_scale(jp, g), e & 1), sum);
                if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);   // few registers, not speed
            }
        }
        return sum + rows::other_half(sum);
    }
    __device__ __forceinline__ float dot(const Q (&q)[D / 16], const Q *qlo, int j, int hf) const {
        const char *p = k + at(j / rows::PAGE) * page;
        float sum = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            float a[8], b[8];
            rows::Op<DT>::unpack(q[ks], a);
            if constexpr (DT == 1) rows::Op<DT>::unpack(qlo[ks], b);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = 16 * ks + 8 * hf + e, jp = j % rows::PAGE;
                const float x = value(p, At::key(jp, t), At::key_scale(jp, t / GROUP), e & 1);
                sum = fmaf(a[e], x, sum);
                if constexpr (DT == 1) sum = fmaf(b[e], x, sum);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return sum + rows::other_half(sum);
    }
    __device__ __forceinline__ void add(f32x16 (&o)[D / 32], int j, float w, int hf) const {
        const char *p = v + at(j / rows::PAGE) * page;
        const int jp = j % rows::PAGE;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = 32 * dt + 8 * (r >> 2) + 4 * hf + (r & 3);
                o[dt][r] = fmaf(w, value(p, At::val(jp, t), At::val_scale(jp, t / GROUP), jp & 1), o[dt][r]);
                if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
    }
};

// One pass of a group of NW waves over n of src's tiles, whose first are in registers (next(0)):
// the queries are in log2 units, in parts.  All groups of the workgroup call it with the same n.
// The logits count from a reference of the row's own, O and l are sums of 2^(s - m):
// m is 0 as long as no row of the wave leaves +-BAND (fp32 and bf16 hold 2^-126 .. 2^127 with the
// same number of bits, and the products begin at 0 without a register; a row whose largest weight
// is 2^-BAND loses weights below 2^-94 of it, and values below 2^-94 lose bits; what overflows
// goes to attend_each), else the largest logit when it was last set.  All the tile's logits are taken before the first
// exponential: the next 32 keys' matrix products run beside the exponentials of these.
constexpr float BAND = 32.0f, ABOVE = 0x1p40f;   // ABOVE: a sum over a tile's keys that sets m anew
template <int DT, int D, class Src, class Keys>
__device__ __forceinline__ void attend(Src &src, char *smem, const Keys &q, const typename Src::Q *qlo, int n,
                                       const rows::Sees &w, rows::RowAcc<DT, D> &a) {
    typedef rows::Op<DT> Op;
    constexpr int NDT = D / 32, KT = Src::KT, SUBS = KT / 32;
    const int lane = threadIdx.x & 63, hf = lane >> 5;
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) a.O[dt] = zero;
    a.m = -INFINITY;
    a.l = 0.0f;
    float shift = 0.0f;    // -m, or 0 while nothing is seen
    bool plain = true;     // it is 0 in all lanes
    const uint32_t lds = lds_offset(smem);
    if (n > 0) {
        src.stage(0, lds);
        src.next(1);
    }
#pragma unroll 1
    for (int it = 0; it < n; ++it) {
        __syncthreads();   // this tile is staged, and the other buffer is read no more
        const int cur = it & 1, j0 = src.tile(it) * KT;
        const char *t = smem + cur * Src::BYTES;
        const auto blind = [&](int j, int n) { return j >= w.hi_max || (j + n <= w.lo_min && j >= w.S); };
        const bool skip = src.past(it) || blind(j0, KT);   // nothing the wave's rows see
        f32x16 s[SUBS];
        if (!skip) {
            typename Src::Keys k[SUBS];
#pragma unroll
            for (int i = 0; i < SUBS; ++i) k[i] = src.keys(t, i, lane);
            if (plain) {
#pragma unroll
                for (int i = 0; i < SUBS; ++i) s[i] = src.logits(k[i], i, q, qlo, zero);
            } else {
#pragma unroll
                for (int i = 0; i < SUBS; ++i) s[i] = src.logits(k[i], i, q, qlo, zero + shift);
            }
        }
        if (it + 1 < n) {   // beside the products
            src.stage(it + 1, lds + (cur ^ 1) * Src::BYTES);
            src.next(it + 2);
        }
        if (skip) continue;
#pragma unroll
        for (int i = 0; i < SUBS; ++i) {
            const int jh = j0 + 32 * i;
            if (blind(jh, 32)) continue;
            bf16x8 vk[2][NDT];   // while the products and exponentials take their time
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) vk[u][dt] = src.vf(t, i, dt, u, lane);
            __builtin_amdgcn_sched_barrier(0);
            if (!(jh + 32 <= w.hi_min && (jh >= w.lo_max || jh + 32 <= w.S))) {
                const uint64_t see = rows::seen_bits(w.lo, w.hi, w.S, jh) >> Src::key(0, hf);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[i][r] = rows::keep(s[i][r], see, Src::key(r, 0), -INFINITY);
            }
            typename Op::F p[2];
            const auto weights = [&]() {   // as operands, and this half's sum of them
                float sum = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = rows::ex2(s[i][8 * u + e]);
                    p[u] = Op::pack(x);
                    if constexpr (DT == 1) {
                        sum = Op::sum(p[u], sum);
                    } else {   // the parts have all their bits
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum += x[e];
                    }
                }
                return sum;
            };
            float sum = weights();
            if (__ballot(!(sum <= ABOVE) || a.m == -INFINITY)) {
                float mx = s[i][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[i][r]);
                mx = fmaxf(a.m, fmaxf(mx, rows::other_half(mx)) - shift);
                if (fabsf(mx) <= BAND) mx = 0.0f;
                const float al = a.m == -INFINITY ? 0.0f : rows::ex2(a.m - mx);   // nothing to rescale yet
                a.l *= al;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) a.O[dt][r] *= al;
                a.m = mx;
                const float by = mx == -INFINITY ? 0.0f : -mx;   // rows that still see nothing: 2^-inf
#pragma unroll
                for (int k = i; k < SUBS; ++k) s[k] = s[k] + (by - shift);
                shift = by;
                plain = !__ballot(!(shift == 0.0f));
                sum = weights();
            }
            a.l += sum;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) a.O[dt] = Op::mma(vk[u][dt], p[u], a.O[dt]);
        }
    }
    __syncthreads();
}

// attend, one key at a time: for rows that came out non-finite.  Each lane adds the visible
// keys only, so nothing of a masked key reaches its row.
template <int DT, int D, class Src, class Keys>
__device__ __forceinline__ void attend_each(const Src &src, const Keys &q, const typename Src::Q *qlo, int n,
                                            const rows::Sees &w, rows::RowAcc<DT, D> &a) {
    const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) a.O[dt] = f32x16{0.0f};
    a.m = -INFINITY;
    a.l = 0.0f;
#pragma unroll 1
    for (int it = 0; it < n && !src.past(it); ++it) {
        const int j0 = src.tile(it) * Src::KT;
#pragma unroll 1
        for (int j = j0; j < min(j0 + Src::KT, w.hi_max); ++j) {
            const float s = src.dot(q, qlo, j, hf);
            if (!(j < w.hi && (j >= w.lo || j < w.S))) continue;
            if (s != s) {   // a NaN makes the row NaN
                a.l = s;
                continue;
            }
            const float mn = fmaxf(a.m, s), al = a.m == -INFINITY ? 0.0f : rows::ex2(a.m - mn);
            const float p = mn == -INFINITY ? 0.0f : rows::ex2(s - mn);   // +inf: inf - inf, a NaN
            a.l = fmaf(a.l, al, hf ? 0.0f : p);
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) a.O[dt][r] *= al;
            a.m = mn;
            src.add(a.O, j, p, hf);
        }
    }
}

}  // namespace mx
}  // namespace hba
