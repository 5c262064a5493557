// Entry points of attention over the paged cache in fp32 or bf16 (the kernels: hba_paged.h).
#include "hba_paged.h"

using namespace hba;

extern "C" int hba_paged_attn_workspace_bytes(int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                                              int64_t S, int64_t shared_pages, int one_each, int64_t max_len,
                                              size_t *bytes) {
    if (!bytes) return HBA_ERR_INVALID_ARG;
    if (int st = paged::check(T, Bd, Hq, Hkv, d, W, S, shared_pages, one_each, max_len, 1 << 24)) return st;
    const paged::Plan p = paged::plan(T, Bd, Hq, Hkv, W, S, shared_pages, one_each != 0, max_len, d, 0);
    *bytes = paged::workspace(p, T, Bd, Hq, Hkv, d, false);
    return HBA_OK;
}

extern "C" int hba_paged_attn(int dtype, const void *q, const int64_t q_strides[2], const float *q_gain, float eps,
                              const float *cos_tab, const float *sin_tab, int64_t n_tab, const void *kr_pages,
                              const void *v_pages, int64_t num_pages, const int32_t *page_table, int64_t max_pages,
                              const int32_t *seq_lens, const float *scales, const int32_t *cu, int64_t T, int64_t Bd,
                              int64_t Hq, int64_t Hkv, int64_t d, int64_t Bk, int64_t W, int64_t S,
                              int64_t shared_pages, int64_t max_len, void *workspace, size_t ws_bytes, void *out,
                              void *stream) {
    paged::Args a;
    paged::Plan p;
    if (int st = paged::setup(a, p, dtype, q, q_strides, q_gain, eps, cos_tab, sin_tab, n_tab, kr_pages, v_pages, num_pages,
                              page_table, max_pages, seq_lens, scales, cu, T, Bd, Hq, Hkv, d, Bk, W, S, shared_pages,
                              max_len, workspace, ws_bytes, out, 0))
        return st;
    int st = HBA_OK;
#define HBA_PAGED(DT, D) st = paged::launch<DT, D, 0, 1>(a, p, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PAGED);
#undef HBA_PAGED
    return st;
}
