// Entry points of attention over the paged cache in 4 or 8 bits (the kernels: hba_paged.h).
#include "hba_paged.h"

using namespace hba;

extern "C" int hba_paged_attn_mx_workspace_bytes(int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                                                 int64_t S, int64_t shared_pages, int one_each, int64_t max_len,
                                                 size_t *bytes) {
    if (!bytes) return HBA_ERR_INVALID_ARG;
    if (int st = paged::check(T, Bd, Hq, Hkv, d, W, S, shared_pages, one_each, max_len, 1 << 24)) return st;
    *bytes = 0;
    for (int bits = 4; bits <= 8; bits += 4) {
        const paged::Plan p = paged::plan(T, Bd, Hq, Hkv, W, S, shared_pages, one_each != 0, max_len, d, bits);
        const size_t n = paged::workspace(p, T, Bd, Hq, Hkv, d, true);
        *bytes = n > *bytes ? n : *bytes;
    }
    return HBA_OK;
}

extern "C" int hba_paged_attn_mx(int dtype, const void *q, const int64_t q_strides[2], const float *q_gain, float eps,
                                 const float *cos_tab, const float *sin_tab, int64_t n_tab, int64_t bits,
                                 const void *k_pages, const void *v_pages, int64_t num_pages, const int32_t *page_table,
                                 int64_t max_pages, const int32_t *seq_lens, const float *scales, const int32_t *cu,
                                 int64_t T, int64_t Bd, int64_t Hq, int64_t Hkv, int64_t d, int64_t Bk, int64_t W,
                                 int64_t S, int64_t shared_pages, int64_t max_len, void *workspace, size_t ws_bytes,
                                 void *out, void *stream) {
    if (bits != 4 && bits != 8) return HBA_ERR_UNSUPPORTED;
    paged::Args a;
    paged::Plan p;
    if (int st = paged::setup(a, p, dtype, q, q_strides, q_gain, eps, cos_tab, sin_tab, n_tab, k_pages, v_pages, num_pages,
                              page_table, max_pages, seq_lens, scales, cu, T, Bd, Hq, Hkv, d, Bk, W, S, shared_pages,
                              max_len, workspace, ws_bytes, out, (int)bits))
        return st;
    int st = HBA_OK;
#define HBA_PAGED_MX(DT, D)                                                             \
    if (bits == 4)                                                                      \
        st = a.G <= 8 ? paged::launch<DT, D, 4, 2>(a, p, (hipStream_t)stream)           \
                      : paged::launch<DT, D, 4, 1>(a, p, (hipStream_t)stream);          \
    else                                                                                \
        st = a.G <= 8 ? paged::launch<DT, D, 8, 2>(a, p, (hipStream_t)stream)           \
                      : paged::launch<DT, D, 8, 1>(a, p, (hipStream_t)stream)
    HBA_DISPATCH_DT_D(dtype, d, HBA_PAGED_MX);
#undef HBA_PAGED_MX
    return st;
}
