// Key preparation, slot summaries, super-summaries and the paged-cache append.
//
//   prep_keys        QKNorm(k) -> kc, RoPE(kc) -> kr, V^T -> vt
//                    (_HeadRMSNorm.forward src/hba/attention.py:88-94,
//                     apply_rope src/hba/attention.py:40-44)
//   summarize        SlotSummarizer.summarize src/hba/summarizer.py:34-42
//   build_super      build_super src/hba/attention.py:202-214
//   kv_append        decode-cache append (no reference counterpart)
//   kv_append_advance  the decode loop's append: token, page summary when it
//                    fills a page, seq_lens += 1 and the new length's scale
//   kv_append_ragged any number of tokens per sequence, and the summaries of
//                    every page they fill
//
// All of these are HBM-bound elementwise / tiny-GEMM work: one thread per key
// row (prep), d/8 lanes per key row (append), one workgroup per 64-key block
// (summaries).
#include "hba_common.h"
#include "hba_abi.h"
#include "hba_generic.h"
#include "hba_ragged.h"

namespace hba {

// ------------------------------------------------------------- row I/O ----
// Rows are d-contiguous and 16-byte aligned (checked by the host entry points).
template <int DT, int D>
__device__ __forceinline__ void load_row(const typename St<DT>::T *p, float (&x)[D]) {
    if constexpr (DT == 1) {
        const uint4 *q = reinterpret_cast<const uint4 *>(p);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            uint4 u = q[c];
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[8 * c + 2 * e] = __uint_as_float(w[e] << 16);
                x[8 * c + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    } else {
        const float4 *q = reinterpret_cast<const float4 *>(p);
#pragma unroll
        for (int c = 0; c < D / 4; ++c) {
            float4 u = q[c];
            x[4 * c] = u.x;
            x[4 * c + 1] = u.y;
            x[4 * c + 2] = u.z;
            x[4 * c + 3] = u.w;
        }
    }
}

template <int DT, int D>
__device__ __forceinline__ void store_row(typename St<DT>::T *p, const float (&x)[D]) {
    if constexpr (DT == 1) {
        uint4 *q = reinterpret_cast<uint4 *>(p);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = (uint32_t)f2bf(x[8 * c + 2 * e]) | ((uint32_t)f2bf(x[8 * c + 2 * e + 1]) << 16);
            q[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        float4 *q = reinterpret_cast<float4 *>(p);
#pragma unroll
        for (int c = 0; c < D / 4; ++c) q[c] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
    }
}

// 8 consecutive elements (16 bytes of bf16, 32 of fp32; 16-byte aligned)
template <int DT>
__device__ __forceinline__ void load8(const typename St<DT>::T *p, float (&x)[8]) {
    if constexpr (DT == 1) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    } else {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], c = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
    }
}

template <int DT>
__device__ __forceinline__ void store8(typename St<DT>::T *p, const float (&x)[8]) {
    if constexpr (DT == 1) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (uint32_t)f2bf(x[2 * e]) | ((uint32_t)f2bf(x[2 * e + 1]) << 16);
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        float4 *q = reinterpret_cast<float4 *>(p);
        q[0] = make_float4(x[0], x[1], x[2], x[3]);
        q[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// --------------------------------------------------------------- kernels ----
// One workgroup per (batch, KV head, 64-key tile); D/8 lanes per key row, 8
// elements each, so that every row load and store is one coalesced 16-byte
// access per lane.  QKNorm's sum of squares runs in the declared order
// (sequential FMA over the row, as qknorm_row) as a chain through the row's
// lanes: lane c continues the sum of lane c-1 (row_shr:1 DPP move); the
// rotation's partner elements (rotate-half) come from lane c ^ (D/16).  The
// values are transposed through LDS, so that vt rows are written as 8
// consecutive keys per lane.
// kb (optional): the tile's kc rows as floats, row stride D + 1, for a
// summary of the block in the same workgroup.  256 threads.
template <int DT, int D>
__device__ __forceinline__ void prep_tile(
    const typename St<DT>::T *__restrict__ k, int64_t ksb, int64_t ksn, int64_t ksh,
    const typename St<DT>::T *__restrict__ v, int64_t vsb, int64_t vsn, int64_t vsh,
    const float *__restrict__ kgain, float eps, const float *__restrict__ cosT,
    const float *__restrict__ sinT, int64_t n, int64_t Hkv, int64_t tile, int64_t bg,
    typename St<DT>::T *__restrict__ kc, typename St<DT>::T *__restrict__ kr,
    typename St<DT>::T *__restrict__ vt, float *__restrict__ kb) {
    using T = typename St<DT>::T;
    constexpr int TPH = D / 8;          // lanes per key row
    constexpr int RPP = 256 / TPH;      // rows per pass
    __shared__ float vs[D][65];         // the tile's values (exact in fp32), key-minor
    const int tid = threadIdx.x;
    const int64_t b = bg / Hkv, g = bg % Hkv;
    const int jl = tid % TPH, t0 = 8 * jl;
    const bool lo = t0 < D / 2;
    const float gn = kgain ? kgain[g] : 0.0f;
#pragma unroll 1
    for (int pass = 0; pass < 64 / RPP; ++pass) {
        const int r = pass * RPP + tid / TPH;
        const int64_t j = tile * 64 + r;
        const bool act = j < n;
        const int64_t jj = act ? j : 0;
        float x[8];
        load8<DT>(k + b * ksb + jj * ksn + g * ksh + t0, x);
        if (kgain) {
            float run = 0.0f;
#pragma unroll
            for (int step = 0; step < TPH; ++step) {
                const float in = __builtin_bit_cast(
                    float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, run), 0x111, 0xf, 0xf, false));
                if (jl == step) {
                    float a = (jl == 0) ? 0.0f : in;
#pragma unroll
                    for (int u = 0; u < 8; ++u) a = fmaf(x[u], x[u], a);
                    run = a;
                }
            }
            const float ss = __shfl(run, (tid & 63) | (TPH - 1), 64);   // the row's last lane
            float ms = ss / (float)D;
            if (ms < eps) ms = eps;
            const float rr = sqrtf(ms);
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = St<DT>::rnd((x[u] / rr) * gn);
        }
        const int64_t row = (bg * n + jj) * D + t0;
        if (act) store8<DT>(kc + row, x);
        if (kb) {
#pragma unroll
            for (int u = 0; u < 8; ++u) kb[r * (D + 1) + t0 + u] = x[u];
        }
        if (kr) {
            float cs[8], sn[8], y[8];
            load8<0>(cosT + jj * D + t0, cs);
            load8<0>(sinT + jj * D + t0, sn);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float part = __shfl_xor(x[u], TPH / 2, 64);
                const float rot = lo ? -part : part;
                y[u] = St<DT>::rnd(St<DT>::rnd(x[u] * St<DT>::rnd(cs[u])) + St<DT>::rnd(rot * St<DT>::rnd(sn[u])));
            }
            if (act) store8<DT>(kr + row, y);
        }
        if (vt) {
            float vv[8];
            load8<DT>(v + b * vsb + jj * vsn + g * vsh + t0, vv);
#pragma unroll
            for (int u = 0; u < 8; ++u) vs[t0 + u][r] = vv[u];
        }
    }
    if (!vt) return;
    __syncthreads();
    // vt[bg][t][tile*64 + 8c' .. +7]: 8 consecutive keys of one row per thread
    T *vrow = vt + bg * D * n;
    const int64_t k0 = tile * 64;
    const bool vec = ((reinterpret_cast<uintptr_t>(vt) & 15) == 0) && (n % 8 == 0);   // uniform
#pragma unroll 1
    for (int c = tid; c < D * 8; c += 256) {
        const int t = c / 8, j8 = 8 * (c % 8);
        float o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = vs[t][j8 + u];
        const int64_t jo = k0 + j8;
        if (vec && jo + 8 <= n) {
            store8<DT>(vrow + (int64_t)t * n + jo, o);
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (jo + u < n) St<DT>::st(vrow, (int64_t)t * n + jo + u, o[u]);
        }
    }
}

template <int DT, int D>
__global__ __launch_bounds__(256) void prep_keys_kernel(
    const typename St<DT>::T *__restrict__ k, int64_t ksb, int64_t ksn, int64_t ksh,
    const typename St<DT>::T *__restrict__ v, int64_t vsb, int64_t vsn, int64_t vsh,
    const float *__restrict__ kgain, float eps, const float *__restrict__ cosT,
    const float *__restrict__ sinT, int64_t n, int64_t Hkv, int64_t ntile,
    typename St<DT>::T *__restrict__ kc, typename St<DT>::T *__restrict__ kr,
    typename St<DT>::T *__restrict__ vt) {
    prep_tile<DT, D>(k, ksb, ksn, ksh, v, vsb, vsn, vsh, kgain, eps, cosT, sinT, n, Hkv, blockIdx.x % ntile,
                     blockIdx.x / ntile, kc, kr, vt, nullptr);
}

// LDS of one block summary: the block's 64 key rows (reused, once the pooled
// rows are done, for chunks of the projection), slot scores, pooled rows,
// and for LONE the probes.
template <int D, bool LONE> struct SummSmem {
    float kb[64][D + 1];
    float att[8][64];
    float pooled[8][D];
    float prl[LONE ? 8 : 1][D];
};

// summarize_staged's pooling and projection: thread tid has column tid % D of slots
// tid / D, tid / D + 256 / D, ... (NQ of them), one chain each.
template <int D, int NQ, class SM> __device__ __forceinline__ void pool_columns(SM &sm, int m, int tid) {
    const int dd = tid % D, s0 = __builtin_amdgcn_readfirstlane(tid / D);
    if (s0 >= m) return;
    float acc[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) acc[q] = 0.0f;
#pragma unroll 8
    for (int t = 0; t < 64; ++t) {
        const float x = sm.kb[t][dd];
#pragma unroll
        for (int q = 0; q < NQ; ++q) acc[q] = fmaf(sm.att[min(s0 + q * (256 / D), m - 1)][t], x, acc[q]);
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q)
        if (s0 + q * (256 / D) < m) sm.pooled[s0 + q * (256 / D)][dd] = acc[q];
}
template <int DT, int D, int NQ, class SM>
__device__ __forceinline__ void project_columns(SM &sm, const float *__restrict__ pj, int m,
                                                typename St<DT>::T *__restrict__ dst, int tid) {
    const int ee = tid % D, s0 = __builtin_amdgcn_readfirstlane(tid / D);
    if (s0 >= m) return;
    float acc[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) acc[q] = 0.0f;
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += 16) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = pj[(d0 + i) * D + ee];
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
                acc[q] = fmaf(sm.pooled[min(s0 + q * (256 / D), m - 1)][d0 + i], x[i], acc[q]);
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q)
        if (s0 + q * (256 / D) < m) St<DT>::st(dst, (int64_t)(s0 + q * (256 / D)) * D + ee, acc[q]);
}
template <int D, class SM> __device__ __forceinline__ void summarize_columns(SM &sm, int m, int tid) {
    if (m * D <= 256) pool_columns<D, 1>(sm, m, tid);
    else if (m * D <= 512) pool_columns<D, 2>(sm, m, tid);
    else pool_columns<D, 4>(sm, m, tid);
}
template <int DT, int D, class SM>
__device__ __forceinline__ void summarize_project(SM &sm, const float *__restrict__ pj, int m,
                                                  typename St<DT>::T *__restrict__ dst, int tid) {
    if (m * D <= 256) project_columns<DT, D, 1>(sm, pj, m, dst, tid);
    else if (m * D <= 512) project_columns<DT, D, 2>(sm, pj, m, dst, tid);
    else project_columns<DT, D, 4>(sm, pj, m, dst, tid);
}

// Slot summaries of one block whose 64 key rows are staged in sm.kb: slot
// scores, softmax over the 64 keys of each slot, pooling, projection.  Every
// output is one sequential fma chain in the index order of the sums
// (probes . key, att . keys, pooled . proj), so both forms below give the
// same bits.  256 threads; starts after the staging barrier; its callers
// barrier before restaging sm.kb.
//   LONE = false (many workgroups, prefill and page lists): probes come as
//     scalar loads (a wave has one slot), the projection from global memory 16
//     rows at a time; a thread's outputs share a column, so each key element and
//     projection element is read once for all of them.
//   LONE = true (a workgroup or two, the decode loop's page fill): probes and
//     the projection are staged through LDS in coalesced bulk loads (the
//     projection in chunks over sm.kb's space), so the workgroup waits on a
//     few load round trips instead of one per chain step.
template <int DT, int D, bool LONE>
__device__ __forceinline__ void summarize_staged(SummSmem<D, LONE> &sm, const float *__restrict__ pr,
                                                 const float *__restrict__ pj, int m, float att_scale,
                                                 typename St<DT>::T *__restrict__ dst, int tid) {
    constexpr int BK = 64;
    if constexpr (LONE) {
        for (int e = tid; e < m * D; e += 256) sm.prl[e / D][e % D] = pr[e];
        __syncthreads();
    }
    for (int e = tid; e < m * BK; e += 256) {
        int s = e / BK, t = e % BK;
        float acc = 0.0f;
        if constexpr (LONE) {
#pragma unroll 16
            for (int dd = 0; dd < D; ++dd) acc = fmaf(sm.prl[s][dd], sm.kb[t][dd], acc);
        } else {
            const float *row = pr + __builtin_amdgcn_readfirstlane(s) * D;   // 64 keys of one slot to a wave
#pragma unroll 16
            for (int dd = 0; dd < D; ++dd) acc = fmaf(row[dd], sm.kb[t][dd], acc);
        }
        sm.att[s][t] = acc * att_scale;
    }
    __syncthreads();
    {   // softmax over the 64 keys of each slot: one wave per slot
        int w = tid / 64, l = tid % 64;
        for (int s = w; s < m; s += 4) {
            float x = sm.att[s][l];
            float mx = wave_max(x);
            float e = expf(x - mx);
            float sm_ = wave_sum(e);
            sm.att[s][l] = e / sm_;
        }
    }
    __syncthreads();
    if constexpr (LONE) {
        for (int e = tid; e < m * D; e += 256) {
            int s = e / D, dd = e % D;
            float acc = 0.0f;
            for (int t = 0; t < BK; ++t) acc = fmaf(sm.att[s][t], sm.kb[t][dd], acc);
            sm.pooled[s][dd] = acc;
        }
    } else {
        summarize_columns<D>(sm, m, tid);
    }
    __syncthreads();
    if constexpr (!LONE) {
        summarize_project<DT, D>(sm, pj, m, dst, tid);
    } else {
        // up to 4 outputs per thread (m * D <= 1024); pj rows staged CHR at a
        // time into the key tile's space (65 or 64 rows fit; CHR divides D)
        constexpr int CH = (BK * (D + 1)) / D;
        constexpr int CHR = (CH < D) ? CH : D;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float *pjl = &sm.kb[0][0];
        for (int c0 = 0; c0 < D; c0 += CHR) {
            if (c0) __syncthreads();   // the previous chunk is used
#pragma unroll 8
            for (int i = tid; i < CHR * D; i += 256) pjl[i] = pj[(int64_t)c0 * D + i];
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int e = tid + 256 * q;
                if (e < m * D) {
                    const int s = e / D, ee = e % D;
                    float a = acc[q];
#pragma unroll 16
                    for (int dd = 0; dd < CHR; ++dd) a = fmaf(sm.pooled[s][c0 + dd], pjl[dd * D + ee], a);
                    acc[q] = a;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = tid + 256 * q;
            if (e < m * D) St<DT>::st(dst, e, acc[q]);
        }
    }
}

// Stage the rows of one cache page (page_key_chunk order) into kb, all but
// row `skip` (-1: none).
template <int DT, int D>
__device__ __forceinline__ void stage_page(const typename St<DT>::T *__restrict__ src, float (&kb)[64][D + 1],
                                           int skip, int tid) {
    for (int c = tid; c < 8 * D; c += 256) {
        int j, t0;
        page_key_chunk(c, D, j, t0);
        if (j == skip) continue;
#pragma unroll
        for (int u = 0; u < 8; ++u) kb[j][t0 + u] = St<DT>::ld(src, 8 * c + u);
    }
}

// One workgroup (256 threads) per 64-key block.  Block base pointers come
// from the contiguous head-major layout, from a list of pages, or (ptab set)
// from a page table: workgroup c takes sequence c's page that its last append
// filled (seq_lens[c] a positive multiple of 64) and exits otherwise (LONE:
// few workgroups run).
template <int DT, int D, bool LONE>
__global__ __launch_bounds__(256) void summarize_kernel(
    const typename St<DT>::T *__restrict__ kc, int64_t n, int64_t nb, int64_t Hkv,
    const int32_t *__restrict__ pages, const int32_t *__restrict__ ptab, int64_t maxp,
    const int32_t *__restrict__ lens, const float *__restrict__ probes,
    const float *__restrict__ proj, int m, float att_scale, typename St<DT>::T *__restrict__ out) {
    constexpr int BK = 64;
    __shared__ SummSmem<D, LONE> sm;
    auto &kb = sm.kb;
    const int tid = threadIdx.x;
    const int64_t c = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
    const typename St<DT>::T *src;
    typename St<DT>::T *dst;
    int64_t filled = -1;
    if (ptab) {   // uniform per workgroup: the exit comes before any barrier
        const int64_t L = lens[c];
        if (L <= 0 || L % BK != 0 || L / BK > maxp) return;
        filled = ptab[c * maxp + L / BK - 1];
    }
    if (pages || ptab) {   // a cache page: chunks of 8 elements in the page layout (page_key_chunk)
        int64_t p = ptab ? filled : (int64_t)pages[c];
        src = kc + (p * Hkv + g) * BK * D;
        dst = out + (p * Hkv + g) * m * D;
        stage_page<DT, D>(src, kb, -1, tid);
    } else {
        src = kc + ((b * Hkv + g) * n + c * BK) * D;
        dst = out + ((b * Hkv + g) * nb + c) * m * D;
        for (int c8 = tid; c8 < BK * D / 8; c8 += 256) {   // 16-byte loads, 8 elements of one row
            float x[8];
            load8<DT>(src + 8 * c8, x);
            const int r = (8 * c8) / D, t0 = (8 * c8) % D;
#pragma unroll
            for (int u = 0; u < 8; ++u) kb[r][t0 + u] = x[u];
        }
    }
    __syncthreads();
    summarize_staged<DT, D, LONE>(sm, probes + g * m * D, proj + g * D * D, m, att_scale, dst, tid);
}

// prep_keys and the slot summaries of every full block in one launch: the
// workgroup of a 64-key tile keeps its kc rows (as the floats it stores) in
// LDS and runs summarize_staged on them, so that S0 has the bits of
// summarize_kernel over the stored kc, without its launch and its re-read.
template <int DT, int D>
__global__ __launch_bounds__(256) void prep_summ_kernel(
    const typename St<DT>::T *__restrict__ k, int64_t ksb, int64_t ksn, int64_t ksh,
    const typename St<DT>::T *__restrict__ v, int64_t vsb, int64_t vsn, int64_t vsh,
    const float *__restrict__ kgain, float eps, const float *__restrict__ cosT,
    const float *__restrict__ sinT, int64_t n, int64_t Hkv, int64_t ntile,
    typename St<DT>::T *__restrict__ kc, typename St<DT>::T *__restrict__ kr,
    typename St<DT>::T *__restrict__ vt, const float *__restrict__ probes, const float *__restrict__ proj,
    int m, float att_scale, typename St<DT>::T *__restrict__ S0) {
    __shared__ SummSmem<D, false> sm;
    const int64_t tile = blockIdx.x % ntile, bg = blockIdx.x / ntile;
    prep_tile<DT, D>(k, ksb, ksn, ksh, v, vsb, vsn, vsh, kgain, eps, cosT, sinT, n, Hkv, tile, bg, kc, kr, vt,
                     &sm.kb[0][0]);
    const int64_t nb = n / 64;
    if (tile >= nb) return;   // a partial last tile has no summary (workgroup-uniform)
    __syncthreads();          // every kb row is written
    const int64_t g = bg % Hkv;
    summarize_staged<DT, D, false>(sm, probes + g * m * D, proj + g * D * D, m, att_scale,
                                   S0 + (bg * nb + tile) * m * D, threadIdx.x);
}

// Super-summaries: sequential child sum, rounded, divided by the child count,
// rounded (the reference's bf16 sum-then-divide, attention.py:210-214).
template <int DT>
__global__ __launch_bounds__(256) void build_super_kernel(const typename St<DT>::T *__restrict__ S0,
                                                           int64_t BH, int64_t nb, int64_t m,
                                                           int64_t d, int64_t F,
                                                           typename St<DT>::T *__restrict__ S1) {
    int64_t ns = (nb + F - 1) / F;
    int64_t total = BH * ns * m * d;
    int64_t gid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (gid >= total) return;
    int64_t t = gid % d;
    int64_t s = (gid / d) % m;
    int64_t p = (gid / (d * m)) % ns;
    int64_t bh = gid / (d * m * ns);
    int64_t c0 = p * F;
    int64_t cn = (c0 + F <= nb) ? F : nb - c0;
    const typename St<DT>::T *base = S0 + bh * nb * m * d;
    float acc = St<DT>::ld(base, (c0 * m + s) * d + t);
    for (int64_t c = 1; c < cn; ++c) acc = acc + St<DT>::ld(base, ((c0 + c) * m + s) * d + t);
    acc = St<DT>::rnd(acc);
    St<DT>::st(S1, gid, acc / (float)cn);
}

// One appended token row (one sequence, one KV head) spread over TPH = D/8
// lanes of a wave, lane jl holding elements t0 = 8*jl .. t0+7: QKNorm with
// the sum of squares chained across the row's lanes in element order (DPP
// row_shr:1, so the fma order is qknorm_row's), the rotation with the
// partner half from lane jl ^ TPH/2 (rope_row's roundings), the key and its
// rotation stored as one 8-element chunk each at page_key_off(j, t0), the
// value elements at page_val_off(j, t).  Every lane of the wave calls it
// (the chain needs them all); act = false lanes load nothing and store
// nothing.  x returns the lane's 8 key elements.
template <int DT, int D>
__device__ __forceinline__ void append_row8(bool act, const typename St<DT>::T *__restrict__ krow,
                                            const typename St<DT>::T *__restrict__ vrow, const float *kgain,
                                            int64_t g, float eps, const float *cs, const float *sn, int64_t base,
                                            int j, typename St<DT>::T *__restrict__ kcp,
                                            typename St<DT>::T *__restrict__ krp,
                                            typename St<DT>::T *__restrict__ vp, float (&x)[8]) {
    constexpr int TPH = D / 8;
    const int jl = (int)(threadIdx.x % TPH), t0 = 8 * jl;
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = act ? St<DT>::ld(krow, t0 + u) : 0.0f;
    if (kgain) {
        float run = 0.0f;
#pragma unroll
        for (int step = 0; step < TPH; ++step) {
            const float in = __builtin_bit_cast(
                float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, run), 0x111, 0xf, 0xf, false));
            if (jl == step) {
                float a = (jl == 0) ? 0.0f : in;
#pragma unroll
                for (int u = 0; u < 8; ++u) a = fmaf(x[u], x[u], a);
                run = a;
            }
        }
        const float ss = __shfl(run, (int)(threadIdx.x & 63) | (TPH - 1), 64);   // the row's last lane
        float ms = ss / (float)D;
        if (ms < eps) ms = eps;
        const float r = sqrtf(ms);
        const float gn = act ? kgain[g] : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = St<DT>::rnd((x[u] / r) * gn);
    }
    const bool lo = t0 < D / 2;
    float y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const float part = __shfl_xor(x[u], TPH / 2, 64);
        const float rot = lo ? -part : part;
        const float c = act ? St<DT>::rnd(cs[t0 + u]) : 0.0f;
        const float sv = act ? St<DT>::rnd(sn[t0 + u]) : 0.0f;
        y[u] = St<DT>::rnd(St<DT>::rnd(x[u] * c) + St<DT>::rnd(rot * sv));
    }
    if (!act) return;
    const int64_t o = base + page_key_off(j, t0, D);   // 8 consecutive elements, 16-byte aligned
    if constexpr (DT == 1) {
        uint32_t wk[4], wr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            wk[e] = (uint32_t)f2bf(x[2 * e]) | ((uint32_t)f2bf(x[2 * e + 1]) << 16);
            wr[e] = (uint32_t)f2bf(y[2 * e]) | ((uint32_t)f2bf(y[2 * e + 1]) << 16);
        }
        *reinterpret_cast<uint4 *>(kcp + o) = make_uint4(wk[0], wk[1], wk[2], wk[3]);
        *reinterpret_cast<uint4 *>(krp + o) = make_uint4(wr[0], wr[1], wr[2], wr[3]);
    } else {
        float4 *pk = reinterpret_cast<float4 *>(kcp + o), *pq = reinterpret_cast<float4 *>(krp + o);
        pk[0] = make_float4(x[0], x[1], x[2], x[3]);
        pk[1] = make_float4(x[4], x[5], x[6], x[7]);
        pq[0] = make_float4(y[0], y[1], y[2], y[3]);
        pq[1] = make_float4(y[4], y[5], y[6], y[7]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) St<DT>::st(vp, base + page_val_off(j, t0 + u), St<DT>::ld(vrow, t0 + u));
}

// kv_append: rows (s, g) = blockIdx.x * RPP + threadIdx.x / TPH, one token
// each at position seq_lens[s] - 1.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(
    const typename St<DT>::T *__restrict__ knew, const typename St<DT>::T *__restrict__ vnew,
    const float *__restrict__ kgain, float eps, const float *__restrict__ cosT,
    const float *__restrict__ sinT, const int32_t *__restrict__ ptab, int64_t maxp,
    const int32_t *__restrict__ lens, int64_t lmax, int64_t Bd, int64_t Hkv,
    typename St<DT>::T *__restrict__ kcp, typename St<DT>::T *__restrict__ krp,
    typename St<DT>::T *__restrict__ vp) {
    constexpr int BK = 64, TPH = D / 8, RPP = 256 / TPH;
    const int64_t row = (int64_t)blockIdx.x * RPP + threadIdx.x / TPH;
    const int64_t s = row / Hkv, g = row % Hkv;
    const int64_t pos = (row < Bd * Hkv) ? (int64_t)lens[s] - 1 : -1;
    // nothing to append, outside the page table or past the RoPE tables
    const bool act = pos >= 0 && pos / BK < maxp && pos < lmax;
    const int64_t page = act ? (int64_t)ptab[s * maxp + pos / BK] : 0;
    const int64_t pc = act ? pos : 0;
    const int64_t rr = act ? row : 0;
    float x[8];
    append_row8<DT, D>(act, knew + rr * D, vnew + rr * D, kgain, g, eps, cosT + pc * D, sinT + pc * D,
                       (page * Hkv + g) * BK * D, (int)(pc % BK), kcp, krp, vp, x);
}

// The decode loop's append: one workgroup per sequence s.  The token goes to
// position pos = seq_lens[s] (KV head g on lanes g*TPH ..); when it fills its
// page, the page's summaries are computed from the page staged in LDS (the
// new row from the writers' registers through LDS, so no global
// read-after-write inside the launch); then seq_lens[s] = pos + 1 and
// scales[s] = scale_tab[pos + 1].  A position outside the page table or the
// RoPE tables appends nothing and leaves seq_lens[s] as it is.  Only thread
// 0 reads and writes seq_lens[s].
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_append_advance_kernel(
    const typename St<DT>::T *__restrict__ knew, const typename St<DT>::T *__restrict__ vnew,
    const float *__restrict__ kgain, float eps, const float *__restrict__ cosT,
    const float *__restrict__ sinT, int64_t lmax, const int32_t *__restrict__ ptab, int64_t maxp,
    int32_t *__restrict__ lens, int64_t Hkv, typename St<DT>::T *__restrict__ kcp,
    typename St<DT>::T *__restrict__ krp, typename St<DT>::T *__restrict__ vp,
    const float *__restrict__ probes, const float *__restrict__ proj, int m, float att_scale,
    typename St<DT>::T *__restrict__ summ, const float *__restrict__ scale_tab, int64_t n_scale,
    float *__restrict__ scales) {
    constexpr int BK = 64, TPH = D / 8, RPP = 256 / TPH;
    __shared__ SummSmem<D, true> sm;
    __shared__ float newk[RPP][D];
    __shared__ int32_t pos_lds;
    const int tid = threadIdx.x;
    const int64_t s = blockIdx.x;
    if (tid == 0) pos_lds = lens[s];
    __syncthreads();
    const int64_t pos = pos_lds;
    const bool ok = pos >= 0 && pos / BK < maxp && pos < lmax;
    const int64_t pc = ok ? pos : 0;
    const int j = (int)(pc % BK);
    const bool filled = ok && j == BK - 1;
    const int64_t page = ok ? (int64_t)ptab[s * maxp + pos / BK] : 0;
    const int r = tid / TPH, t0 = 8 * (tid % TPH);
    for (int64_t g0 = 0; g0 < Hkv; g0 += RPP) {
        const int64_t g = g0 + r;
        const bool act = ok && g < Hkv;
        const int64_t row = s * Hkv + (act ? g : 0);
        float x[8];
        append_row8<DT, D>(act, knew + row * D, vnew + row * D, kgain, g, eps, cosT + pc * D, sinT + pc * D,
                           (page * Hkv + g) * BK * D, j, kcp, krp, vp, x);
        if (!filled) continue;
#pragma unroll
        for (int u = 0; u < 8; ++u) newk[r][t0 + u] = x[u];
        __syncthreads();   // newk rows come from other waves
        const int64_t gend = (Hkv < g0 + RPP) ? Hkv : g0 + RPP;
        for (int64_t gg = g0; gg < gend; ++gg) {
            const int64_t hp = page * Hkv + gg;
            stage_page<DT, D>(kcp + hp * BK * D, sm.kb, BK - 1, tid);
            for (int t = tid; t < D; t += 256) sm.kb[BK - 1][t] = newk[gg - g0][t];
            __syncthreads();
            summarize_staged<DT, D, true>(sm, probes + gg * m * D, proj + gg * D * D, m, att_scale,
                                          summ + hp * m * D, tid);
            __syncthreads();
        }
    }
    if (tid == 0) {
        const int64_t L = ok ? pos + 1 : pos;
        if (scales) scales[s] = scale_tab[(L < n_scale) ? (L > 0 ? L : 0) : n_scale - 1];
        if (ok) lens[s] = (int32_t)L;
    }
}

// ---------------------------------------------------------- ragged append --
struct RaggedArgs {
    const char *k, *v;              // [T, Hkv, D]; byte strides of token and head
    int64_t kst, ksh, vst, vsh;
    const int32_t *cu;
    int T, Bd, Hkv, maxp, m;
    const float *kgain, *cosT, *sinT, *probes, *proj;
    float eps, att_scale;
    int64_t n_tab, pages;
    const int32_t *ptab, *lens;
    char *kc, *kr, *vp, *summ;      // kc, summ may be nullptr
};

// Tokens of sequence s that are appended: positions first .. last - 1, token i of
// them at place c0 + i of the batch.  Positions outside the page table or past
// the rotation tables, or below 0 (a length below the token count) are not.
struct NewTokens {
    int c0, first, last;
};
__device__ __forceinline__ NewTokens new_tokens(const RaggedArgs &a, int s) {
    NewTokens x;
    const int n = ragged::tokens(a.cu, s, a.T, x.c0);
    const int64_t most = min((int64_t)a.maxp * 64, a.n_tab), L = a.lens[s];
    int64_t first = L - n;
    if (first < 0) {
        x.c0 -= (int)max(first, -(int64_t)n);
        first = 0;
    }
    x.first = (int)min(first, most);
    x.last = (int)max((int64_t)x.first, min(L, most));
    return x;
}

// A page's keys in LDS: 8 elements of a key together, keys beside one another, a
// chunk of room after every 64.  Written by rows, read by columns and by rows, all
// without bank conflicts.
template <int DT, int D> struct KeyTile {
    using T = typename St<DT>::T;
    __align__(16) T x[D / 8 * 65 * 8];
    __device__ __forceinline__ T *at(int j, int t) { return x + ((t / 8) * 65 + j) * 8 + t % 8; }
};

// Slot summaries of the page whose 64 keys are in a tile: summarize_staged's chains
// in the same order, so the same bits, from the keys as stored.  A thread has 4
// columns of one slot's pooled row.
template <int DT, int D, class SM>
__device__ __forceinline__ void summarize_tile(SM &sm, const float *__restrict__ pr, const float *__restrict__ pj,
                                               int m, float att_scale, typename St<DT>::T *__restrict__ dst, int tid) {
    for (int e = tid; e < m * 64; e += 256) {
        const int s = __builtin_amdgcn_readfirstlane(e / 64), t = e % 64;
        float acc = 0.0f;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
            float x[8];
            load8<DT>(sm.keys.at(t, 8 * c), x);
#pragma unroll
            for (int u = 0; u < 8; ++u) acc = fmaf(pr[s * D + 8 * c + u], x[u], acc);
        }
        sm.att[s][t] = acc * att_scale;
    }
    __syncthreads();
    for (int s = tid / 64; s < m; s += 4) {   // softmax over the 64 keys: one wave per slot
        const float x = sm.att[s][tid % 64], e = expf(x - wave_max(x));
        sm.att[s][tid % 64] = e / wave_sum(e);
    }
    __syncthreads();
    for (int e = tid; e < m * (D / 4); e += 256) {
        const int s = e / (D / 4), t0 = 4 * (e % (D / 4));
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int t = 0; t < 64; ++t) {
            const float w = sm.att[s][t];
            const auto *x = sm.keys.at(t, t0);
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[u] = fmaf(w, St<DT>::ld(x, u), acc[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) sm.pooled[s][t0 + u] = acc[u];
    }
    __syncthreads();
    summarize_project<DT, D>(sm, pj, m, dst, tid);
}

template <class T> __device__ __forceinline__ void load_raw(T (&x)[8], const T *p) {
    using V = uint32_t __attribute__((ext_vector_type(2 * sizeof(T))));
    const V v = *reinterpret_cast<const V *>(p);
    __builtin_memcpy(x, &v, sizeof v);
}

// One workgroup per (page that gets tokens, KV head): D/8 lanes a row as in
// prep_tile (the same chain for the norm, so kc has the bits of every other way
// to append it), 256 / (D/8) rows at a time.  kr is rounded once, from the
// normalised key in fp32.  The page's summaries follow when its last token is
// among the new ones (the earlier keys are read back: no other workgroup writes
// this page).
// HBM-bound in the large: k and v read once, kc, kr and v written once.  14000
// tokens, 4 KV heads, d = 128, bf16 with summaries: 37 us, 21 at a copy's rate;
// 59 before each of these:
//   - values, rotated keys and keys go through LDS in turn, and a wave writes 1 KB
//     runs of the page where rows written as they come fill 64 bytes of a line at a
//     time; the summary reads the same keys there;
//   - 22 KB of LDS, so that all 1088 workgroups are there at once (at 40 KB four to
//     a CU, 1024, and the rest follow as a second round: 46 us);
//   - workgroups of one page's heads run on one XCD, whose L2 then has their rows
//     of the cos/sin tables.
template <int DT, int D, bool SUMM>
__global__ __launch_bounds__(256) void kv_append_ragged_kernel(const RaggedArgs a) {
    using T = typename St<DT>::T;
    constexpr int TPH = D / 8, RPP = 256 / TPH, ESZ = DT == 1 ? 2 : 4, VS = 64 + 16 / ESZ;
    // values, rotated keys, keys in turn: 22 KB (bf16, d = 128)
    __shared__ union {
        __align__(16) T vs[D][VS];
        struct {
            KeyTile<DT, D> keys;
            float att[SUMM ? 8 : 1][64], pooled[SUMM ? 8 : 1][D];
        } sm;
    } lds;
    auto &vs = lds.vs;
    auto &sm = lds.sm;
    const int tid = threadIdx.x, g = blockIdx.x / 8 % a.Hkv;
    int slot;
    const int s = ragged::find(blockIdx.x / 8 / a.Hkv * 8 + blockIdx.x % 8, a.Bd, [&](int i) {
        const NewTokens x = new_tokens(a, i);
        return x.last > x.first ? (x.last - 1) / 64 - x.first / 64 + 1 : 0;
    }, slot);
    if (s < 0) return;
    const NewTokens x = new_tokens(a, s);
    const int lp = x.first / 64 + slot, p0 = lp * 64;
    const int ja = max(x.first - p0, 0), jb = min(x.last - p0, 64);   // the page's new tokens
    const int64_t page = a.ptab[(int64_t)s * a.maxp + lp];
    if (page < 0 || page >= a.pages) return;                          // not a page of this cache
    const int64_t base = (page * a.Hkv + g) * 64 * D;
    T *kcp = reinterpret_cast<T *>(a.kc) + base, *krp = reinterpret_cast<T *>(a.kr) + base;
    T *vp = reinterpret_cast<T *>(a.vp) + base;
    const bool fills = SUMM && jb == 64;
    const int jl = tid % TPH, t0 = 8 * jl;
    const bool lo = t0 < D / 2;
    const float gn = a.kgain ? a.kgain[g] : 0.0f;
    // all loads of a kind at once: a row outside the new ones repeats one of those
    T kx[64 / RPP][8], vx[64 / RPP][8];
#pragma unroll
    for (int pass = 0; pass < 64 / RPP; ++pass) {
        const int64_t tok = x.c0 + (p0 + min(max(pass * RPP + tid / TPH, ja), jb - 1) - x.first);
        load_raw(kx[pass], reinterpret_cast<const T *>(a.k + tok * a.kst + g * a.ksh) + t0);
        load_raw(vx[pass], reinterpret_cast<const T *>(a.v + tok * a.vst + g * a.vsh) + t0);
    }
#pragma unroll
    for (int pass = 0; pass < 64 / RPP; ++pass) {
        const int j = pass * RPP + tid / TPH;
        if (j >= ja && j < jb) {
#pragma unroll
            for (int u = 0; u < 8; ++u) vs[t0 + u][j ^ (8 * (jl % 8))] = vx[pass][u];
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = tid; c < 8 * D; c += 256) {
        int t, j0;
        page_val_chunk(c, t, j0);
        const int jp = j0 ^ (8 * (t / 8 % 8));
        if (j0 >= ja && j0 + 8 <= jb) {
            if constexpr (DT == 1) {
                *reinterpret_cast<uint4 *>(vp + 8 * c) = *reinterpret_cast<const uint4 *>(&vs[t][jp]);
            } else {
                reinterpret_cast<float4 *>(vp + 8 * c)[0] = *reinterpret_cast<const float4 *>(&vs[t][jp]);
                reinterpret_cast<float4 *>(vp + 8 * c)[1] = *reinterpret_cast<const float4 *>(&vs[t][jp + 4]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (j0 + u >= ja && j0 + u < jb) vp[8 * c + u] = vs[t][jp + u];
        }
    }
    __syncthreads();   // vs becomes sm
#pragma unroll
    for (int pass = 0; pass < 64 / RPP; ++pass) {
        const int j = pass * RPP + tid / TPH;
        if (pass * RPP >= jb || pass * RPP + RPP <= ja) continue;     // uniform
        const int64_t pos = p0 + min(max(j, ja), jb - 1);
        float cs[8], sn[8], y[8], z[8];
        load8<0>(a.cosT + pos * D + t0, cs);
        load8<0>(a.sinT + pos * D + t0, sn);
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = St<DT>::ld(kx[pass], u);
        if (a.kgain) {
            float run = 0.0f;
#pragma unroll
            for (int step = 0; step < TPH; ++step) {
                const float in = __builtin_bit_cast(
                    float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, run), 0x111, 0xf, 0xf, false));
                if (jl == step) {
                    float c = (jl == 0) ? 0.0f : in;
#pragma unroll
                    for (int u = 0; u < 8; ++u) c = fmaf(y[u], y[u], c);
                    run = c;
                }
            }
            const float ss = __shfl(run, (tid & 63) | (TPH - 1), 64);   // the row's last lane
            float ms = ss / (float)D;
            if (ms < a.eps) ms = a.eps;
            const float rr = sqrtf(ms);
#pragma unroll
            for (int u = 0; u < 8; ++u) y[u] = (y[u] / rr) * gn;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float part = __shfl_xor(y[u], TPH / 2, 64);
            z[u] = y[u] * cs[u] + (lo ? -part : part) * sn[u];
            St<DT>::st(kx[pass], u, y[u]);
        }
        if (j >= ja && j < jb) store8<DT>(sm.keys.at(j, t0), z);
    }
    __syncthreads();
#pragma unroll
    for (int c = tid; c < 8 * D; c += 256) {
        int j, e0;
        page_key_chunk(c, D, j, e0);
        if (j >= ja && j < jb) __builtin_memcpy(krp + 8 * c, sm.keys.at(j, e0), 8 * sizeof(T));
    }
    if (!a.kc) return;
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 64 / RPP; ++pass) {
        const int j = pass * RPP + tid / TPH;
        if (j >= ja && j < jb) __builtin_memcpy(sm.keys.at(j, t0), kx[pass], sizeof kx[pass]);
    }
    __syncthreads();
#pragma unroll
    for (int c = tid; c < 8 * D; c += 256) {
        int j, e0;
        page_key_chunk(c, D, j, e0);
        if (j >= ja && j < jb) __builtin_memcpy(kcp + 8 * c, sm.keys.at(j, e0), 8 * sizeof(T));
        else if (SUMM && fills) __builtin_memcpy(sm.keys.at(j, e0), kcp + 8 * c, 8 * sizeof(T));   // it was there
    }
    if constexpr (SUMM) {
        if (!fills) return;
        __syncthreads();
        summarize_tile<DT, D>(sm, a.probes + (int64_t)g * a.m * D, a.proj + (int64_t)g * D * D, a.m, a.att_scale,
                              reinterpret_cast<T *>(a.summ) + (page * a.Hkv + g) * a.m * D, tid);
    }
}

}  // namespace hba

using namespace hba;

// ------------------------------------------------------------ entry points --
extern "C" int hba_abi_version(void) { return HBA_ABI_VERSION; }

extern "C" const char *hba_status_string(int status) {
    switch (status) {
        case HBA_OK: return "ok";
        case HBA_ERR_INVALID_ARG: return "invalid argument";
        case HBA_ERR_UNSUPPORTED: return "unsupported shape or dtype";
        case HBA_ERR_DEVICE: return "no gfx950 device";
        case HBA_ERR_LAUNCH: return "kernel launch failed";
        case HBA_ERR_SCRATCH: return "request exceeds the fixed scratch of the no-allocation entry point";
        default: return "unknown status";
    }
}

extern "C" int hba_device_check(void) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return HBA_ERR_DEVICE;
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, dev) != hipSuccess) return HBA_ERR_DEVICE;
    const char *a = prop.gcnArchName;
    if (!(a[0] == 'g' && a[1] == 'f' && a[2] == 'x' && a[3] == '9' && a[4] == '5' && a[5] == '0'))
        return HBA_ERR_DEVICE;
    return HBA_OK;
}

extern "C" int hba_prep_keys(int dtype, const void *k, const int64_t k_strides[3], const void *v,
                             const int64_t v_strides[3], const float *k_gain, float eps,
                             const float *cos_tab, const float *sin_tab, int64_t B, int64_t n,
                             int64_t Hkv, int64_t d, void *kc, void *kr, void *vt, void *stream) {
    if (dtype == HBA_DTYPE_F32 && d != 64 && d != 128) {   // fp32, another head dim: the generic kernel
        if (!gen_shape_ok(d, 1)) return HBA_ERR_UNSUPPORTED;
        if (!k || !k_strides || !kc || B <= 0 || n <= 0 || Hkv <= 0) return HBA_ERR_INVALID_ARG;
        if ((kr && (!cos_tab || !sin_tab)) || (vt && (!v || !v_strides))) return HBA_ERR_INVALID_ARG;
        return gen_prep_keys((const float *)k, k_strides, (const float *)v, v_strides ? v_strides : k_strides,
                             k_gain, eps, cos_tab, sin_tab, B, n, Hkv, d, (float *)kc, (float *)kr, (float *)vt,
                             (hipStream_t)stream);
    }
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!k || !k_strides || !kc || B <= 0 || n <= 0 || Hkv <= 0) return HBA_ERR_INVALID_ARG;
    if (kr && (!cos_tab || !sin_tab)) return HBA_ERR_INVALID_ARG;
    if (vt && (!v || !v_strides)) return HBA_ERR_INVALID_ARG;
    if (kr && (!abi::aligned16(cos_tab) || !abi::aligned16(sin_tab))) return HBA_ERR_UNSUPPORTED;
    if (!abi::rows_aligned(dtype, k, k_strides) || (vt && !abi::rows_aligned(dtype, v, v_strides)) ||
        !abi::aligned16(kc) || (kr && !abi::aligned16(kr)))
        return HBA_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const int64_t ntile = (n + 63) / 64;
    if (B * Hkv * ntile > 0x7fffffff) return HBA_ERR_UNSUPPORTED;
    dim3 grid((unsigned)(B * Hkv * ntile));
    const int64_t *vs = v_strides ? v_strides : k_strides;
#define HBA_PREP(DT, D)                                                                            \
    hipLaunchKernelGGL((prep_keys_kernel<DT, D>), grid, dim3(256), 0, s,                           \
                       (const St<DT>::T *)k, k_strides[0], k_strides[1], k_strides[2],             \
                       (const St<DT>::T *)v, vs[0], vs[1], vs[2], k_gain, eps, cos_tab, sin_tab, n, \
                       Hkv, ntile, (St<DT>::T *)kc, (St<DT>::T *)kr, (St<DT>::T *)vt)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PREP);
#undef HBA_PREP
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_prep_keys_summarize(int dtype, const void *k, const int64_t k_strides[3], const void *v,
                                       const int64_t v_strides[3], const float *k_gain, float eps,
                                       const float *cos_tab, const float *sin_tab, int64_t B, int64_t n,
                                       int64_t Hkv, int64_t d, void *kc, void *kr, void *vt, const float *probes,
                                       const float *proj, int64_t m, void *S0, void *stream) {
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!k || !k_strides || !kc || !probes || !proj || !S0 || B <= 0 || n <= 0 || Hkv <= 0)
        return HBA_ERR_INVALID_ARG;
    if (kr && (!cos_tab || !sin_tab)) return HBA_ERR_INVALID_ARG;
    if (vt && (!v || !v_strides)) return HBA_ERR_INVALID_ARG;
    if (m < 1 || m > 8) return HBA_ERR_UNSUPPORTED;
    if (kr && (!abi::aligned16(cos_tab) || !abi::aligned16(sin_tab))) return HBA_ERR_UNSUPPORTED;
    if (!abi::rows_aligned(dtype, k, k_strides) || (vt && !abi::rows_aligned(dtype, v, v_strides)) ||
        !abi::aligned16(kc) || (kr && !abi::aligned16(kr)))
        return HBA_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const int64_t ntile = (n + 63) / 64;
    if (B * Hkv * ntile > 0x7fffffff) return HBA_ERR_UNSUPPORTED;
    dim3 grid((unsigned)(B * Hkv * ntile));
    const int64_t *vs = v_strides ? v_strides : k_strides;
    const float att_scale = (float)(1.0 / __builtin_sqrt((double)d));
#define HBA_PREP_SUMM(DT, D)                                                                       \
    hipLaunchKernelGGL((prep_summ_kernel<DT, D>), grid, dim3(256), 0, s,                           \
                       (const St<DT>::T *)k, k_strides[0], k_strides[1], k_strides[2],             \
                       (const St<DT>::T *)v, vs[0], vs[1], vs[2], k_gain, eps, cos_tab, sin_tab, n, \
                       Hkv, ntile, (St<DT>::T *)kc, (St<DT>::T *)kr, (St<DT>::T *)vt, probes, proj, \
                       (int)m, att_scale, (St<DT>::T *)S0)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PREP_SUMM);
#undef HBA_PREP_SUMM
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

static int summarize_common(int dtype, const void *kc, int64_t B, int64_t Hkv, int64_t n, int64_t d,
                            int64_t Bk, const int32_t *pages, const int32_t *ptab, int64_t maxp,
                            const int32_t *lens, int64_t nblocks, const float *probes,
                            const float *proj, int64_t m, void *out, void *stream) {
    if (dtype == HBA_DTYPE_F32 && !pages && !ptab && !tuned_shape(d, Bk)) {   // fp32 prefill, other geometry
        if (!kc || !probes || !proj || !out || B <= 0 || Hkv <= 0) return HBA_ERR_INVALID_ARG;
        if (!gen_shape_ok(d, Bk) || m < 1 || m > 8) return HBA_ERR_UNSUPPORTED;
        if (nblocks <= 0) return HBA_OK;
        if (nblocks > 0x7fffffff || Hkv > 65535 || B > 65535) return HBA_ERR_UNSUPPORTED;
        return gen_summarize((const float *)kc, B, Hkv, n, d, Bk, nblocks, probes, proj, m, (float *)out,
                             (hipStream_t)stream);
    }
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!kc || !probes || !proj || !out || B <= 0 || Hkv <= 0) return HBA_ERR_INVALID_ARG;
    if (Bk != 64) return HBA_ERR_UNSUPPORTED;
    if (m < 1 || m > 8) return HBA_ERR_UNSUPPORTED;
    if (nblocks <= 0) return HBA_OK;
    if (nblocks > 0x7fffffff || Hkv > 65535 || B > 65535) return HBA_ERR_UNSUPPORTED;
    if (!abi::aligned16(kc)) return HBA_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    dim3 grid((unsigned)nblocks, (unsigned)Hkv, (unsigned)B);
    float att_scale = (float)(1.0 / __builtin_sqrt((double)d));
#define HBA_SUMM(DT, D)                                                                            \
    do {                                                                                           \
        if (ptab)                                                                                  \
            hipLaunchKernelGGL((summarize_kernel<DT, D, true>), grid, dim3(256), 0, s,             \
                               (const St<DT>::T *)kc, n, nblocks, Hkv, pages, ptab, maxp, lens,    \
                               probes, proj, (int)m, att_scale, (St<DT>::T *)out);                 \
        else                                                                                       \
            hipLaunchKernelGGL((summarize_kernel<DT, D, false>), grid, dim3(256), 0, s,            \
                               (const St<DT>::T *)kc, n, nblocks, Hkv, pages, ptab, maxp, lens,    \
                               probes, proj, (int)m, att_scale, (St<DT>::T *)out);                 \
    } while (0)
    HBA_DISPATCH_DT_D(dtype, d, HBA_SUMM);
#undef HBA_SUMM
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_summarize(int dtype, const void *kc, int64_t B, int64_t Hkv, int64_t n, int64_t d,
                             int64_t Bk, const float *probes, const float *proj, int64_t m, void *S0,
                             void *stream) {
    if (Bk <= 0 || n <= 0) return HBA_ERR_INVALID_ARG;
    return summarize_common(dtype, kc, B, Hkv, n, d, Bk, nullptr, nullptr, 0, nullptr, n / Bk, probes,
                            proj, m, S0, stream);
}

extern "C" int hba_summarize_pages(int dtype, const void *kc_pages, const int32_t *pages,
                                   int64_t npages, int64_t Hkv, int64_t d, int64_t Bk,
                                   const float *probes, const float *proj, int64_t m,
                                   void *summ_pages, void *stream) {
    if (!pages || npages < 0) return HBA_ERR_INVALID_ARG;
    return summarize_common(dtype, kc_pages, 1, Hkv, Bk, d, Bk, pages, nullptr, 0, nullptr, npages,
                            probes, proj, m, summ_pages, stream);
}

extern "C" int hba_summarize_filled(int dtype, const void *kc_pages, const int32_t *page_table,
                                    int64_t max_pages, const int32_t *seq_lens, int64_t Bd,
                                    int64_t Hkv, int64_t d, int64_t Bk, const float *probes,
                                    const float *proj, int64_t m, void *summ_pages, void *stream) {
    if (!page_table || !seq_lens || max_pages <= 0 || Bd < 0) return HBA_ERR_INVALID_ARG;
    return summarize_common(dtype, kc_pages, 1, Hkv, Bk, d, Bk, nullptr, page_table, max_pages,
                            seq_lens, Bd, probes, proj, m, summ_pages, stream);
}

extern "C" int hba_build_super(int dtype, const void *S0, int64_t B, int64_t Hkv, int64_t nb,
                               int64_t m, int64_t d, int64_t fanout, void *S1, void *stream) {
    if (dtype != HBA_DTYPE_F32 && dtype != HBA_DTYPE_BF16) return HBA_ERR_UNSUPPORTED;
    if (!S0 || !S1 || B <= 0 || Hkv <= 0 || nb <= 0 || m <= 0 || d <= 0 || fanout <= 0)
        return HBA_ERR_INVALID_ARG;
    int64_t ns = (nb + fanout - 1) / fanout;
    int64_t total = B * Hkv * ns * m * d;
    hipStream_t s = (hipStream_t)stream;
    dim3 grid((unsigned)((total + 255) / 256));
    if (dtype == HBA_DTYPE_F32)
        hipLaunchKernelGGL(build_super_kernel<0>, grid, dim3(256), 0, s, (const float *)S0, B * Hkv,
                           nb, m, d, fanout, (float *)S1);
    else
        hipLaunchKernelGGL(build_super_kernel<1>, grid, dim3(256), 0, s, (const bf16_t *)S0, B * Hkv,
                           nb, m, d, fanout, (bf16_t *)S1);
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_kv_append_advance(int dtype, const void *k_new, const void *v_new,
                                     const float *k_gain, float eps, const float *cos_tab,
                                     const float *sin_tab, int64_t n_tab, const int32_t *page_table,
                                     int64_t max_pages, int32_t *seq_lens, int64_t Bd, int64_t Hkv,
                                     int64_t d, int64_t Bk, void *kc_pages, void *kr_pages,
                                     void *v_pages, const float *probes, const float *proj, int64_t m,
                                     void *summ_pages, const float *scale_tab, int64_t n_scale,
                                     float *scales, void *stream) {
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!k_new || !v_new || !cos_tab || !sin_tab || !page_table || !seq_lens || !kc_pages ||
        !kr_pages || !v_pages || !probes || !proj || !summ_pages || Bd <= 0 || Hkv <= 0 ||
        max_pages <= 0 || n_tab <= 0 || (scales && (!scale_tab || n_scale <= 0)))
        return HBA_ERR_INVALID_ARG;
    if (Bk != 64 || m < 1 || m > 8) return HBA_ERR_UNSUPPORTED;
    if (Bd > 0x7fffffff || Hkv > 65535) return HBA_ERR_UNSUPPORTED;
    if (!abi::aligned16(k_new) || !abi::aligned16(v_new) || !abi::aligned16(kc_pages) ||
        !abi::aligned16(kr_pages) || !abi::aligned16(v_pages))
        return HBA_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const float att_scale = (float)(1.0 / __builtin_sqrt((double)d));
#define HBA_APPA(DT, D)                                                                            \
    hipLaunchKernelGGL((kv_append_advance_kernel<DT, D>), dim3((unsigned)Bd), dim3(256), 0, s,      \
                       (const St<DT>::T *)k_new, (const St<DT>::T *)v_new, k_gain, eps, cos_tab,    \
                       sin_tab, n_tab, page_table, max_pages, seq_lens, Hkv,                       \
                       (St<DT>::T *)kc_pages, (St<DT>::T *)kr_pages, (St<DT>::T *)v_pages, probes, \
                       proj, (int)m, att_scale, (St<DT>::T *)summ_pages, scale_tab, n_scale, scales)
    HBA_DISPATCH_DT_D(dtype, d, HBA_APPA);
#undef HBA_APPA
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_kv_append(int dtype, const void *k_new, const void *v_new, const float *k_gain,
                             float eps, const float *cos_tab, const float *sin_tab, int64_t n_tab,
                             const int32_t *page_table, int64_t max_pages, const int32_t *seq_lens,
                             int64_t Bd, int64_t Hkv, int64_t d, int64_t Bk, void *kc_pages,
                             void *kr_pages, void *v_pages, void *stream) {
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!k_new || !v_new || !cos_tab || !sin_tab || !page_table || !seq_lens || !kc_pages ||
        !kr_pages || !v_pages || Bd <= 0 || Hkv <= 0 || max_pages <= 0 || n_tab <= 0)
        return HBA_ERR_INVALID_ARG;
    if (Bk != 64) return HBA_ERR_UNSUPPORTED;
    if (!abi::aligned16(k_new) || !abi::aligned16(v_new) || !abi::aligned16(kc_pages) ||
        !abi::aligned16(kr_pages) || !abi::aligned16(v_pages))
        return HBA_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const int64_t rpp = 256 / (d / 8);   // token rows per workgroup
    if ((Bd * Hkv + rpp - 1) / rpp > 0x7fffffff) return HBA_ERR_UNSUPPORTED;
    dim3 grid((unsigned)((Bd * Hkv + rpp - 1) / rpp));
#define HBA_APP(DT, D)                                                                             \
    hipLaunchKernelGGL((kv_append_kernel<DT, D>), grid, dim3(256), 0, s, (const St<DT>::T *)k_new,   \
                       (const St<DT>::T *)v_new, k_gain, eps, cos_tab, sin_tab, page_table,        \
                       max_pages, seq_lens, n_tab, Bd, Hkv, (St<DT>::T *)kc_pages,                  \
                       (St<DT>::T *)kr_pages, (St<DT>::T *)v_pages)
    HBA_DISPATCH_DT_D(dtype, d, HBA_APP);
#undef HBA_APP
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}

extern "C" int hba_kv_append_ragged(int dtype, const void *k, const int64_t k_strides[2], const void *v,
                                    const int64_t v_strides[2], const int32_t *cu, int64_t T, const float *k_gain,
                                    float eps, const float *cos_tab, const float *sin_tab, int64_t n_tab,
                                    const int32_t *page_table, int64_t max_pages, const int32_t *seq_lens, int64_t Bd,
                                    int64_t Hkv, int64_t d, int64_t Bk, int64_t num_pages, void *kc_pages,
                                    void *kr_pages, void *v_pages, const float *probes, const float *proj, int64_t m,
                                    void *summ_pages, void *stream) {
    int st = abi::check_dtype_dim(dtype, d);
    if (st) return st;
    if (!k || !k_strides || !v || !v_strides || !cu || !cos_tab || !sin_tab || !page_table || !seq_lens || !kr_pages ||
        !v_pages || T < 0 || Bd <= 0 || Hkv <= 0 || max_pages <= 0 || n_tab <= 0 || num_pages <= 0)
        return HBA_ERR_INVALID_ARG;
    if (summ_pages && (!kc_pages || !probes || !proj)) return HBA_ERR_INVALID_ARG;
    if (Bk != 64 || (summ_pages && (m < 1 || m > 8))) return HBA_ERR_UNSUPPORTED;
    if (T > (1 << 30) || Bd > (1 << 24) || Hkv > 65535 || max_pages > (1 << 24)) return HBA_ERR_UNSUPPORTED;
    const int64_t e = abi::elem_size(dtype), al = 16 / e;
    if (!abi::aligned16(k) || !abi::aligned16(v) || k_strides[0] % al || k_strides[1] % al || v_strides[0] % al ||
        v_strides[1] % al || !abi::aligned16(cos_tab) || !abi::aligned16(sin_tab) || !abi::aligned16(kc_pages) ||
        !abi::aligned16(kr_pages) || !abi::aligned16(v_pages))
        return HBA_ERR_UNSUPPORTED;
    if (T == 0) return HBA_OK;
    RaggedArgs a = {};
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
    a.m = (int)m;
    a.kgain = k_gain;
    a.cosT = cos_tab;
    a.sinT = sin_tab;
    a.probes = probes;
    a.proj = proj;
    a.eps = eps;
    a.att_scale = (float)(1.0 / __builtin_sqrt((double)d));
    a.n_tab = n_tab;
    a.pages = num_pages;
    a.ptab = page_table;
    a.lens = seq_lens;
    a.kc = (char *)kc_pages;
    a.kr = (char *)kr_pages;
    a.vp = (char *)v_pages;
    a.summ = (char *)summ_pages;
    // c tokens touch at most c and at most c / 64 + 2 pages
    const int64_t slots = T < T / 64 + 2 * Bd ? T : T / 64 + 2 * Bd;
    if (!abi::launchable((slots + 7) / 8 * 8 * Hkv, 256)) return HBA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)((slots + 7) / 8 * 8 * Hkv));
#define HBA_APPR(DT, D)                                                                                       \
    do {                                                                                                      \
        if (summ_pages)                                                                                       \
            hipLaunchKernelGGL((kv_append_ragged_kernel<DT, D, true>), grid, dim3(256), 0, (hipStream_t)stream, a);  \
        else                                                                                                  \
            hipLaunchKernelGGL((kv_append_ragged_kernel<DT, D, false>), grid, dim3(256), 0, (hipStream_t)stream, a); \
    } while (0)
    HBA_DISPATCH_DT_D(dtype, d, HBA_APPR);
#undef HBA_APPR
    HBA_LAUNCH_CHECK();
    return HBA_OK;
}
