// Attention of a tile of query rows to tiles of keys, shared by the sliding-window
// and the paged-cache kernels (bf16 and fp32, head dim 64 / 128).
//
// A wave holds 32 query rows as the columns of S^T = K . Q^T on 32x32 MFMA
// tiles: lane l has column l % 32, and of each 32-key tile the 16 keys of its
// half l / 32.  Row maxima and sums are then in-lane but for one exchange
// between the halves, and the probabilities are already the B operand of
// O^T += V^T . P^T: nothing moves between lanes.  The rows of one KV head's
// query heads are flattened (row r = token r / G, head r % G), so every group
// size fills the tiles and the heads of a group share the staged keys.
//
// Softmax: a shift m and the sums O and l in fp32, in units of log2.  m is a maximum
// of the row, but not of the newest tiles: a tile's probabilities are taken
// with the m there is, and only where their sum passes 2^16 (far from any
// range's end), or nothing was seen before, the wave takes the tile's maximum as
// m, rescales and does the tile once more.  So most tiles compute no maximum.
//
// Masked keys have probability 0; a NaN or infinity of V in a masked place
// would still spoil 0 * V.  Whether that happened shows in the result, so a
// workgroup whose rows come out non-finite computes them once more key by key,
// where a masked key takes no part (attend_each).  Finite inputs pay nothing but
// the check of the result; values behind a sequence in its last page, which may be
// anything, are cleared in LDS first.
#pragma once

#include "hba_common.h"
#include "hba_dma.h"

namespace hba {
namespace rows {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4r __attribute__((ext_vector_type(4)));

constexpr int PAGE = 64;          // tokens of a cache page
// Keys per staged tile: 8 KB of keys and as much of values, but 32 keys at least,
// so that two buffers leave LDS for as many workgroups as the registers do.
template <int DT, int D> constexpr int KEYS = D * (DT == 1 ? 2 : 4) <= 128 ? 64 : 32;
constexpr int NW = 4;             // waves per workgroup
constexpr int RW = 32;            // query rows per wave
constexpr int RT = NW * RW;       // query rows per workgroup
// Waves per SIMD that a row kernel's registers leave room for.  At two or more the
// compiler also keeps the MFMA results in the registers that vector instructions
// read, without a move each.
template <int DT, int D> constexpr int WAVES = DT == 1 ? 2 : (D == 64 ? 2 : 1);
constexpr float LOG2E = 1.4426950408889634f;
constexpr float MOST = 65536.0f;  // sum of a tile's probabilities that calls for a new maximum

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// The thread's place among the NW waves that stage tiles together (a workgroup may
// have two such groups, for halves of the keys).
__device__ __forceinline__ int thread() { return threadIdx.x % (64 * NW); }

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Operand fragments of a 16-deep step: 8 elements of one row or column, lane l
// those of its half, elements 8 (l / 32) .. + 7.  mma adds a 32x32 product.
// Lane l of the result: column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4.
// fp32 takes eight 2-deep steps: in step e half h supplies element 8 h + e.
template <int DT> struct Op;
template <> struct Op<1> {
    typedef bf16x8 F;
    static __device__ __forceinline__ f32x16 mma(F a, F b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    // the probabilities enter the product in bf16, as the matrix cores take them: a
    // relative 2^-8 each at most, which averages out over a row's keys
    static __device__ __forceinline__ F pack(const float (&x)[8]) {
        F r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (__bf16)x[e];
        return r;
    }
    static __device__ __forceinline__ F load(const void *p) {
        return __builtin_bit_cast(F, *reinterpret_cast<const u32x4r *>(p));
    }
    static __device__ __forceinline__ void unpack(F f, float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)f[e];
    }
    // acc + the sum of f's elements, two at a time
    static __device__ __forceinline__ float sum(F f, float acc) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(f, f, 0, 1), one, acc, false);
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(f, f, 2, 3), one, acc, false);
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(f, f, 4, 5), one, acc, false);
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(f, f, 6, 7), one, acc, false);
    }
};
template <> struct Op<0> {
    typedef f32x8 F;
    static __device__ __forceinline__ f32x16 mma(F a, F b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ F pack(const float (&x)[8]) {
        F r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = x[e];
        return r;
    }
    static __device__ __forceinline__ F load(const void *p) {
        const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ void unpack(F f, float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f[e];
    }
    static __device__ __forceinline__ float sum(F f, float acc) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc += f[e];
        return acc;
    }
};

// Elements 8u .. 8u+7 of a 32x32 result as the operand of the step over its
// rows' u-th half.
template <int DT> __device__ __forceinline__ typename Op<DT>::F half16(const f32x16 &p, int u) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[8 * u + e];
    return Op<DT>::pack(x);
}

// ------------------------------------------------------------ staged rows --
// R rows of D elements in LDS, 16-byte chunk c of row r at place c ^ swz(r) of its
// row, swz(r) = 2 (r % 4) + r / 4 % 2: eight rows' chunks c lie in eight
// different places (an operand along the rows reads those in one LDS cycle), and
// so do the chunk pairs 2c, 2c + 1 of four rows r, r + 1 .. (a transposed operand).
template <int DT, int D> struct Tile {
    typedef typename St<DT>::T T;
    typedef typename Op<DT>::F F;
    static constexpr int ESZ = DT == 1 ? 2 : 4;
    static constexpr int NCH = D * ESZ / 16;          // chunks per row
    static constexpr int ROWB = D * ESZ;              // bytes per row

    static constexpr int RPI = 64 * NW / NCH;         // rows that the workgroup stages at once (a multiple of 8)

    static __device__ __forceinline__ int swz(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }
    static __device__ __forceinline__ int at(int r, int c) { return r * ROWB + ((c ^ swz(r)) * 16); }

    // Row r, elements 16 ks + 8 (lane / 32) .. + 7.
    static __device__ __forceinline__ F row(const char *t, int r, int ks, int hf) {
        if constexpr (DT == 1) {
            return Op<1>::load(t + at(r, 2 * ks + hf));
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(t + at(r, 4 * ks + 2 * hf));
            const f32x4 b = *reinterpret_cast<const f32x4 *>(t + at(r, 4 * ks + 2 * hf + 1));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Column 32 dt + lane % 32 over rows r0 + 4 hf + 0..3 and r0 + 8 + 4 hf + 0..3: the
    // rows that registers 8u .. 8u+7 of a result hold, r0 = 32 tile + 16 u.
    static __device__ __forceinline__ F col(const char *t, int r0, int dt, int lane) {
        const int hf = lane >> 5;
        if constexpr (DT == 1) {
            const int r = r0 + 4 * hf + ((lane & 15) >> 2);
            const int x = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            const int c = x >> 3, o = (x & 7) * 2;
            return ld_tr8(reinterpret_cast<const bf16_t *>(t + at(r, c) + o),
                          reinterpret_cast<const bf16_t *>(t + at(r + 8, c) + o));
        } else {
            const int x = 32 * dt + (lane & 31), c = x >> 2, o = (x & 3) * 4;
            F f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                f[e] = *reinterpret_cast<const float *>(t + at(r0 + 4 * hf + (e & 3) + 8 * (e >> 2), c) + o);
            return f;
        }
    }
    // The thread's first chunk of a staging pass, as an offset from the first row.
    static __device__ __forceinline__ uint32_t offset(int64_t bytes) {
        const int r = thread() / NCH;
        return (uint32_t)(r * (int)bytes) + ((thread() % NCH) ^ swz(r)) * 16;
    }
    // Stage rows j0 .. j0 + R - 1 of a strided array (`bytes` from row to row, off =
    // offset(bytes)); rows past `last` read row `last`.  Called by all NW waves.
    template <int R>
    static __device__ __forceinline__ void stage(const char *base, int64_t bytes, uint32_t off, int j0, int last,
                                                 uint32_t lds) {
        const int wave = __builtin_amdgcn_readfirstlane(thread() >> 6);
        if (j0 + R - 1 <= last) {
            const char *p = base + j0 * bytes;
#pragma unroll
            for (int i = 0; i < R / RPI; ++i) dma16s(p + i * RPI * bytes, off, lds + (i * NW + wave) * 1024);
        } else {
            const int r = thread() / NCH, c = (thread() % NCH) ^ swz(r);
#pragma unroll
            for (int i = 0; i < R / RPI; ++i)
                dma16(base + (int64_t)min(j0 + r + i * RPI, last) * bytes + c * 16, lds + (i * NW + wave) * 1024);
        }
    }
};

// Keys and values of one KV head as strided rows.
template <int DT, int D, int KEYS_ = KEYS<DT, D>> struct DenseKV {
    typedef typename Op<DT>::F F;
    typedef Tile<DT, D> TL;
    static constexpr int KT = KEYS_, BYTES = 2 * KT * TL::ROWB;   // a staged tile: keys, then values
    static constexpr bool TAIL = false;               // no rows past `last` are read
    const char *k, *v;
    int64_t kb, vb;                                   // bytes from row to row
    int last;                                         // the last row that may be read
    uint32_t ko, vo;                                  // TL::offset of kb, vb

    __device__ __forceinline__ void next(int) {}
    __device__ __forceinline__ void stage(int tile, uint32_t lds) const {
        TL::template stage<KT>(k, kb, ko, tile * KT, last, lds);
        TL::template stage<KT>(v, vb, vo, tile * KT, last, lds + KT * TL::ROWB);
    }
    // the key (of 32) that register r of half hf holds
    static __device__ __forceinline__ int key(int r, int hf) { return 8 * (r >> 2) + 4 * hf + (r & 3); }
    static __device__ __forceinline__ F kf(const char *t, int kt, int ks, int lane) {
        return TL::row(t, 32 * kt + (lane & 31), ks, lane >> 5);
    }
    static __device__ __forceinline__ F vf(const char *t, int kt, int dt, int u, int lane) {
        return TL::col(t + KT * TL::ROWB, 32 * kt + 16 * u, dt, lane);
    }
    template <bool LO>
    __device__ __forceinline__ float dot(const F (&q)[D / 16], const F *, int j, int hf) const;
    __device__ __forceinline__ void add(f32x16 (&o)[D / 32], int j, float p, int hf) const;
};

// Keys and values of one KV head in 64-token pages (page_key_off, page_val_off):
// a tile is a page or half of one as it lies in memory (the tokens of a half are
// a run of the keys and every other KB of the values).  Row l % 32 of a key operand is the
// token for which the result's registers 8u .. 8u+7 of half h are the tokens
// 16 u + 8 h .. + 7, the order in which the pages hold values.
template <int DT, int D> struct PageKV {
    typedef typename Op<DT>::F F;
    static constexpr int KT = KEYS<DT, D>, TP = PAGE / KT;   // tiles of a page
    static constexpr int ESZ = DT == 1 ? 2 : 4, HALF = KT * D * ESZ, BYTES = 2 * HALF;
    const char *k, *v;            // the KV head's place in page 0
    int64_t page;                 // bytes from page to page
    const int32_t *table;         // the sequence's pages
    int len;                      // its keys: what lies behind them in a page may be anything
    int64_t pages;                // pages there are
    static constexpr bool TAIL = true;
    int64_t id;                   // the page of the tile that is staged next
    int half;                     // and the tile's place in it

    // A scalar load: a vector load's wait would be one for the DMA before it as well.
    __device__ __forceinline__ int64_t at(int lp) const {
        typedef const __attribute__((address_space(4))) int32_t *uniform;
        const int p = ((uniform)(uintptr_t)table)[__builtin_amdgcn_readfirstlane(lp)];
        return p < 0 ? 0 : (p < pages ? p : pages - 1);   // never outside the cache
    }
    __device__ __forceinline__ void next(int tile) {
        id = at(tile / TP);
        half = tile % TP;
    }
    __device__ __forceinline__ void stage(int, uint32_t lds) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t off = (threadIdx.x & 63) * 16;
        const char *kp = k + id * page + half * HALF, *vp = v + id * page + half * 512 * ESZ;
#pragma unroll
        for (int i = 0; i < HALF / 1024 / NW; ++i) {
            const int c = (i * NW + wave) * 1024;
            dma16s(kp + c, off, lds + c);
            // chunk run dt * 2 + half of a page becomes run dt of a half tile
            dma16s(vp + (TP == 1 ? c : c / (512 * ESZ) * (1024 * ESZ) + c % (512 * ESZ)), off, lds + HALF + c);
        }
    }
    static __device__ __forceinline__ int key(int r, int hf) {
        return 16 * (r >> 3) + 8 * hf + 4 * ((r >> 2) & 1) + (r & 3);
    }
    static __device__ __forceinline__ F kf(const char *t, int kt, int ks, int lane) {
        const int r = lane & 31, l16 = 8 * (r >> 4) + 4 * ((r >> 2) & 1) + (r & 3), mt = 2 * kt + ((r >> 3) & 1);
        return Op<DT>::load(t + ((mt * (D / 32) + (ks >> 1)) * 64 + l16 + 16 * (2 * (ks & 1) + (lane >> 5))) * 8 * ESZ);
    }
    static __device__ __forceinline__ F vf(const char *t, int kt, int dt, int u, int lane) {
        const int x = 32 * dt + (lane & 31);
        return Op<DT>::load(t + HALF + (((x >> 4) * (KT / 32) + kt) * 64 + (x & 15) + 16 * (2 * u + (lane >> 5))) * 8 * ESZ);
    }
    // Clears the values at and past place n of a staged tile: a weight of 0 would make
    // NaN of a NaN there.  A chunk of 8 is as many keys of one column (see vf).
    static __device__ __forceinline__ void clear(char *t, int n) {
        typedef typename St<DT>::T T;
        for (int c = threadIdx.x; c < KT * D / 8; c += 64 * NW) {
            const int first = n - (32 * (c / 64 % (KT / 32)) + 8 * (c % 64 / 16));   // the chunk's first to clear
            T *p = reinterpret_cast<T *>(t + HALF) + 8 * c;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= first) St<DT>::st(p, e, 0.0f);
        }
    }
    // one key, for attend_each
    __device__ __forceinline__ float dot_one(const F (&q)[D / 16], int j, int hf) const {
        const char *t = k + at(j / PAGE) * page;
        float sum = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            float a[8], b[8];
            Op<DT>::unpack(q[ks], a);
            Op<DT>::unpack(Op<DT>::load(t + page_key_off(j % PAGE, 16 * ks + 8 * hf, D) * ESZ), b);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(a[e], b[e], sum);
        }
        return sum + other_half(sum);
    }
    template <bool LO> __device__ __forceinline__ float dot(const F (&q)[D / 16], const F *qlo, int j, int hf) const {
        float s = dot_one(q, j, hf);
        if constexpr (LO) s += dot_one(*reinterpret_cast<const F(*)[D / 16]>(qlo), j, hf);
        return s;
    }
    __device__ __forceinline__ void add(f32x16 (&o)[D / 32], int j, float p, int hf) const {
        typedef typename St<DT>::T T;
        const T *t = reinterpret_cast<const T *>(v + at(j / PAGE) * page);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                o[dt][r] = fmaf(p, St<DT>::ld(t, page_val_off(j % PAGE, 32 * dt + 8 * (r >> 2) + 4 * hf + (r & 3))),
                                o[dt][r]);
    }
};

// A 32-column result, columns as rows of memory: registers 4g .. 4g+3 of block dt
// are elements 32 dt + 8 g + 4 hf + 0..3.
template <int DT, int D>
__device__ __forceinline__ void store_rows(char *p, const f32x16 (&o)[D / 32], float f) {
    const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = 32 * dt + 8 * g + 4 * hf;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = o[dt][4 * g + i] * f;
            if constexpr (DT == 1)
                *reinterpret_cast<uint2 *>(p + 2 * e) = make_uint2(pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3]));
            else
                *reinterpret_cast<float4 *>(p + 4 * e) = make_float4(x[0], x[1], x[2], x[3]);
        }
}

template <int D> __device__ __forceinline__ bool any_bad(const f32x16 (&o)[D / 32]) {
    float x = 0.0f;   // 0 * finite is 0, 0 * anything else NaN
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) x = fmaf(0.0f, o[dt][r], x);
    return !(x == 0.0f);
}

// The first n of 64 bits.
__device__ __forceinline__ uint64_t first_bits(int n) {
    return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}
// Places lo .. hi - 1 and those below both s and hi, of the 64 from j0.
__device__ __forceinline__ uint64_t seen_bits(int lo, int hi, int s, int j0) {
    return (first_bits(hi - j0) & ~first_bits(lo - j0)) | first_bits(min(s, hi) - j0);
}
// x where bit b of the mask is set, else `other`: two instructions (a bit field
// extract, a bitwise select).
__device__ __forceinline__ float keep(float x, uint64_t bits, int b, float other) {
    const uint32_t w = b < 32 ? (uint32_t)bits : (uint32_t)(bits >> 32);
    const uint32_t t = (uint32_t)((int32_t)(w << (31 - (b & 31))) >> 31);
    return __uint_as_float((__float_as_uint(x) & t) | (__float_as_uint(other) & ~t));
}

// What a row (a lane's column) and its wave see: keys j < hi with j >= lo or
// j < S.  The wave's bounds cover its valid rows.
struct Sees {
    int lo, hi, S;
    int lo_min, lo_max, hi_min, hi_max;
};

template <int DT, int D> struct RowAcc {
    f32x16 O[D / 32];
    float m, l;       // running maximum (log2 units; -inf: nothing seen yet), and this half's part of the sum
    float le;         // that part before the operands' rounding, of attend<.., SEP> only (else it is l)
};

// Stages the first of tiles it0 .. it1 - 1 of a list (tile it < ns: sinks, tile it;
// else tile wt0 + it - ns): attend goes on from there.  What a kernel loads in
// between comes while the tile does.
template <class Src>
__device__ __forceinline__ void attend_begin(Src &src, char *smem, int it0, int it1, int ns, int wt0) {
    const auto tile = [&](int it) { return it < ns ? it : wt0 + it - ns; };
    if (it0 >= it1) return;
    src.next(tile(it0));
    src.stage(tile(it0), lds_offset(smem));
    src.next(tile(min(it0 + 1, it1 - 1)));
}

// One pass of the workgroup's rows over the tiles.  c: logits to log2
// units.  LO: the queries come as two parts in log2 units already (c = 1); their
// products then start from -m instead of 0.  Every wave of the workgroup calls
// it; it leaves no wave reading LDS.
// ONE: of each tile the wave takes the 32 keys `which` only (another one has the rest).
// SEP: the sum of the probabilities as they are, too.  O is divided by the sum of the
// rounded ones, which its own weights are; a log-sum-exp from that would put a row's
// gradients off by up to a bf16 rounding (2^-8) in common.
template <int DT, int D, bool LO, bool ONE = false, bool SEP = false, class Src>
__device__ __forceinline__ void attend(Src &src, char *smem, const typename Op<DT>::F (&q)[D / 16],
                                       const typename Op<DT>::F *qlo, float c, int it0, int it1, int ns, int wt0,
                                       const Sees &w, RowAcc<DT, D> &a, int which = 0) {
    typedef typename Op<DT>::F F;
    constexpr int NKS = D / 16, NDT = D / 32, KT = Src::KT;
    const int lane = threadIdx.x & 63, hf = lane >> 5;
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) a.O[dt] = zero;
    a.m = -INFINITY;
    a.l = a.le = 0.0f;
    float shift = 0.0f;   // -m, or 0 while nothing is seen
    const uint32_t lds = lds_offset(smem);
    const auto tile = [&](int it) { return it < ns ? it : wt0 + it - ns; };
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
        wait_vm<0>();
        __syncthreads();   // this tile is staged, and the other buffer is read no more
        const int cur = (it - it0) & 1, nx = it + 1;
        if (nx < it1) {
            src.stage(tile(nx), lds + (cur ^ 1) * Src::BYTES);
            src.next(tile(min(nx + 1, it1 - 1)));
        }
        const int j0 = tile(it) * KT;
        if constexpr (Src::TAIL) {
            if (j0 + KT > src.len) {   // the same for the workgroup
                src.clear(smem + cur * Src::BYTES, src.len - j0);
                __syncthreads();
            }
        }
        if (j0 >= w.hi_max || (j0 + KT <= w.lo_min && j0 >= w.S)) continue;   // nothing the wave's rows see
        const char *t = smem + cur * Src::BYTES;
#pragma unroll
        for (int i = 0; i < (ONE ? 1 : KT / 32); ++i) {   // 32 keys at a time: fewer registers, and halves that no row sees cost nothing
            const int kt = ONE ? which : i, jh = j0 + 32 * kt;
            if (jh >= w.hi_max || (jh + 32 <= w.lo_min && jh >= w.S)) continue;
            f32x16 s = zero;
            if constexpr (LO) s = s + shift;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const F kf = src.kf(t, kt, ks, lane);
                s = Op<DT>::mma(kf, q[ks], s);
                if constexpr (LO) s = Op<DT>::mma(kf, qlo[ks], s);
            }
            if (!(jh + 32 <= w.hi_min && (jh >= w.lo_max || jh + 32 <= w.S))) {
                const uint64_t see = seen_bits(w.lo, w.hi, w.S, jh) >> Src::key(0, hf);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = keep(s[r], see, Src::key(r, 0), -INFINITY);
            }
            // probabilities 2^(c s + by) as operands, and this half's sum of them
            F p[2];
            struct Sums {
                float rounded, whole;
            };
            const auto weights = [&](float by) {
                Sums sum = {0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] = ex2(LO ? s[8 * u + e] : fmaf(s[8 * u + e], c, by));
                    if constexpr (SEP) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum.whole += x[e];
                    }
                    p[u] = Op<DT>::pack(x);
                    sum.rounded = Op<DT>::sum(p[u], sum.rounded);
                }
                return sum;
            };
            Sums sum = weights(shift);
            // A new maximum.  (A row that sees nothing, as those behind a tile's last have
            // nothing to see, has none and keeps its wave here: exponentials twice.)
            if (__ballot(!(sum.rounded <= MOST) || a.m == -INFINITY)) {
                float mx = s[0];
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
                mx = fmaxf(mx, other_half(mx));
                mx = fmaxf(a.m, LO ? mx - shift : mx * c);
                const float al = a.m == -INFINITY ? 0.0f : ex2(a.m - mx);   // nothing to rescale yet
                a.l *= al;
                if constexpr (SEP) a.le *= al;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) a.O[dt][r] *= al;
                a.m = mx;
                const float by = mx == -INFINITY ? 0.0f : -mx;   // rows that still see nothing: 2^-inf
                if constexpr (LO) s = s + (by - shift);
                shift = by;
                sum = weights(shift);
            }
            a.l += sum.rounded;
            if constexpr (SEP) a.le += sum.whole;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) a.O[dt] = Op<DT>::mma(src.vf(t, kt, dt, u, lane), p[u], a.O[dt]);
        }
    }
    __syncthreads();
}

// Sum over both halves of a fragment pair: the dot product of two rows.
template <int DT, int D>
__device__ __forceinline__ float dot_rows(const typename Op<DT>::F (&x)[D / 16], const char *p, int hf) {
    float sum = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        float u[8], y[8];
        Op<DT>::unpack(x[ks], u);
        Op<DT>::unpack(Op<DT>::load(p + (16 * ks + 8 * hf) * Tile<DT, D>::ESZ), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(u[e], y[e], sum);
        __builtin_amdgcn_sched_barrier(0);   // few registers, not speed: see attend_each
    }
    return sum + other_half(sum);
}

// o += f * (row p) on the elements 32 dt + 8 g + 4 hf + i of registers 4 g + i.
template <int DT, int D>
__device__ __forceinline__ void add_row(f32x16 (&o)[D / 32], const char *p, float f, int hf) {
    typedef typename St<DT>::T T;
    const T *x = reinterpret_cast<const T *>(p);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = fmaf(f, St<DT>::ld(x, 32 * dt + 8 * (r >> 2) + 4 * hf + (r & 3)), o[dt][r]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int DT, int D, int KT>
template <bool LO>
__device__ __forceinline__ float DenseKV<DT, D, KT>::dot(const F (&q)[D / 16], const F *, int j, int hf) const {
    return dot_rows<DT, D>(q, k + (int64_t)min(j, last) * kb, hf);
}
template <int DT, int D, int KT>
__device__ __forceinline__ void DenseKV<DT, D, KT>::add(f32x16 (&o)[D / 32], int j, float p, int hf) const {
    add_row<DT, D>(o, v + (int64_t)min(j, last) * vb, p, hf);
}

// attend, one key at a time: for rows that came out non-finite.  Each lane adds
// the visible keys only, so nothing of a masked key reaches its row.  It is kept
// from loading ahead: its registers would cost the kernels that hold it waves.
template <int DT, int D, bool LO, class Src>
__device__ __forceinline__ void attend_each(const Src &src, const typename Op<DT>::F (&q)[D / 16],
                                         const typename Op<DT>::F *qlo, float c, int it0, int it1, int ns, int wt0,
                                         const Sees &w, RowAcc<DT, D> &a) {
    const int hf = (threadIdx.x & 63) >> 5;
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) a.O[dt] = zero;
    a.m = -INFINITY;
    a.l = 0.0f;
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
        const int j0 = (it < ns ? it : wt0 + it - ns) * Src::KT;
#pragma unroll 1
        for (int j = j0; j < min(j0 + Src::KT, w.hi_max); ++j) {
            float s = src.template dot<LO>(q, qlo, j, hf) * c;
            if (!(j < w.hi && (j >= w.lo || j < w.S))) continue;
            if (s != s) {   // a NaN makes the row NaN
                a.l = s;
                continue;
            }
            const float mn = fmaxf(a.m, s), al = a.m == -INFINITY ? 0.0f : ex2(a.m - mn);
            const float p = mn == -INFINITY ? 0.0f : ex2(s - mn);   // +inf: inf - inf, a NaN
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

// The list of KT-key tiles that rows with first visible key lo (the smallest),
// one past the last hi (the largest) and S sinks see: ns tiles of sinks, then
// tiles wt0 ...; returns how many.
template <int KT> __device__ __forceinline__ int tile_list(int lo, int hi, int S, int &ns, int &wt0) {
    wt0 = lo / KT;
    ns = min((min(S, hi) + KT - 1) / KT, wt0);
    const int wt1 = (hi + KT - 1) / KT;
    return ns + max(wt1 - wt0, 0);
}

}  // namespace rows
}  // namespace hba
