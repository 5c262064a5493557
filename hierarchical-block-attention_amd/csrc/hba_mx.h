// The paged cache in 4 or 8 bits: what a page holds, and how it becomes operands.
//
// A page (64 tokens of one KV head, D elements each) is 64 D F / 8 bytes of codes
// and 2 D bytes of scales.  Codes are e2m1 (F = 4) or e4m3 (F = 8); the elements
// 32 g .. 32 g + 31 of a token share the scale 2^(b - 127), b a byte (b = 255, codes 0:
// they are NaN).  A value has at most 4 bits of mantissa, so it is exact in bf16, and one
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

// ------------------------------------------------------------ staged tiles --
// Keys and values of one KV head, for rows::attend: a tile's codes are loaded into
// registers while the tile before it is worked on, and become the bf16 tile that
// rows::PageKV stages.  A thread has 16 codes of the keys and 16 of the values: of a
// key, half a group at most; of the values, eight tokens in two columns of a group.
template <int DT, int D, int F> struct TileKV {
    typedef typename rows::Op<DT>::F Q;    // the queries' operand
    typedef rows::PageKV<1, D> Bf16;
    typedef Place<D, F> At;
    static constexpr int KT = Bf16::KT, TP = Bf16::TP, HALF = Bf16::HALF, BYTES = Bf16::BYTES;
    static constexpr int NG = D / GROUP, NB = 16 * F / 8;   // a thread's bytes of codes
    static constexpr bool TAIL = false;                     // stage clears what lies behind the sequence
    const char *k, *v;            // the KV head's place in page 0
    int64_t page;                 // bytes from page to page
    const int32_t *table;
    int len;
    int64_t pages;
    int64_t id;                   // the page of the tile that is staged next
    int half;                     // and the tile's place in it
    uint32_t kc[NB / 4], vc[NB / 4], ks, vs[2];   // its codes and scales

    __device__ __forceinline__ int64_t at(int lp) const {
        typedef const __attribute__((address_space(4))) int32_t *uniform;
        const int p = ((uniform)(uintptr_t)table)[__builtin_amdgcn_readfirstlane(lp)];
        return p < 0 ? 0 : (p < pages ? p : pages - 1);   // never outside the cache
    }
    // The thread's 16 codes q = thread / 64 of its lane's stream in this tile: a tile of
    // 16 keys (D = 64) or half of one (128); columns 32 g .. of 32 tokens.
    static __device__ __forceinline__ int unit() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
    template <class T> static __device__ __forceinline__ void get(uint32_t (&to)[NB / 4], const char *p) {
        const T x = *reinterpret_cast<const T *>(p);
        __builtin_memcpy(to, &x, sizeof x);
    }
    __device__ __forceinline__ void next(int tile) {
        typedef __attribute__((ext_vector_type(NB / 4))) uint32_t V;
        id = at(tile / TP);
        half = tile % TP;
        const int q = unit(), lane = threadIdx.x & 63, x = q * NB, first = half * (4 * NB) * 64;
        const char *kp = k + id * page, *vp = v + id * page;
        get<V>(kc, kp + first + (x / 16 * 64 + lane) * 16 + x % 16);
        get<V>(vc, vp + first + (x / 16 * 64 + lane) * 16 + x % 16);
        const int g = (lane >> 4) * (D / 4) / GROUP;
        ks = *reinterpret_cast<const uint32_t *>(kp + code_bytes(D, F) + ((lane & 15) + 16 * g) * 4);
        const int h = D == 64 ? q >> 1 : half, vg = D == 64 ? q & 1 : q;
        const u32x2 s = *reinterpret_cast<const u32x2 *>(vp + code_bytes(D, F) + ((h * 4 + (lane >> 4)) * NG + vg) * 8);
        vs[0] = s[0];
        vs[1] = s[1];
    }
    __device__ __forceinline__ void stage(int tile, uint32_t lds) {
        typedef __attribute__((address_space(3))) u32x4 *out;
        const int q = unit(), lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
        const int mt = D == 64 ? q : q >> 1, t0 = D / 4 * lg + (D == 64 ? 0 : 16 * (q & 1));   // key tile here, first element
        const int pt = D == 64 ? mt : 2 * half + mt;                                           // and in its page
        const float sc = __uint_as_float((ks >> (8 * pt) & 255u) << 23);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int t = t0 + 8 * c;
            *(out)(uintptr_t)(lds + ((mt * (D / 32) + (t >> 5)) * 64 + l16 + 16 * ((t >> 3) & 3)) * 16) =
                __builtin_bit_cast(u32x4, eight<F>(kc + c * (F / 4), sc));
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
            *(out)(uintptr_t)(lds + HALF + (((2 * g + c) * (KT / 32) + h) * 64 + lane) * 16) = r;
        }
    }
    static __device__ __forceinline__ int key(int r, int hf) { return Bf16::key(r, hf); }
    static __device__ __forceinline__ bf16x8 kf(const char *t, int kt, int ks, int lane) { return Bf16::kf(t, kt, ks, lane); }
    static __device__ __forceinline__ bf16x8 vf(const char *t, int kt, int dt, int u, int lane) {
        return Bf16::vf(t, kt, dt, u, lane);
    }
    // one key, for attend_each
    static __device__ __forceinline__ float value(const char *p, int at_code, int at_scale, int odd) {
        const uint32_t c = (uint8_t)p[at_code];
        return one<F>(F == 4 ? c >> (4 * odd) : c, __uint_as_float((uint32_t)(uint8_t)p[at_scale] << 23));
    }
    template <bool LO> __device__ __forceinline__ float dot(const Q (&q)[D / 16], const Q *qlo, int j, int hf) const {
        const char *p = k + at(j / rows::PAGE) * page;
        float sum = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            float a[8], b[8];
            rows::Op<DT>::unpack(q[ks], a);
            if constexpr (DT == 1 && LO) rows::Op<DT>::unpack(qlo[ks], b);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = 16 * ks + 8 * hf + e, jp = j % rows::PAGE;
                const float x = value(p, At::key(jp, t), At::key_scale(jp, t / GROUP), e & 1);
                sum = fmaf(a[e], x, sum);
                if constexpr (DT == 1 && LO) sum = fmaf(b[e], x, sum);
            }
            __builtin_amdgcn_sched_barrier(0);   // few registers, not speed
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

}  // namespace mx
}  // namespace hba
