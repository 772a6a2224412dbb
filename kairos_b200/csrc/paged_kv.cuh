// A layer of a paged key-value cache as the kernels see it.
#pragma once
#include "rotary.cuh"

namespace kairos {

struct KvView {
    void *k, *v;
    float *ks, *vs;
    int pages, heads, page_shift, dim;   // page_size = 1 << page_shift
};

inline int kv_view(const kairos_kv_layer* kv, KvView* out) {
    if (!kv) return KAIROS_ERR_ARG;
    int shift = 0;
    while (shift < 8 && (1 << shift) != kv->page_size) ++shift;
    if (kv->pages <= 0 || kv->kv_heads <= 0 || kv->kv_heads > 65535 || shift < 4 || (1 << shift) != kv->page_size ||
        (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)) {
        set_last_error("paged cache: pages and kv_heads > 0 (kv_heads < 65536), page_size 16, 32, 64, 128 or 256, head_dim 64, 128 or 256");
        return KAIROS_ERR_SHAPE;
    }
    if (!kv->k || !kv->v || ((uintptr_t)kv->k & 15) || ((uintptr_t)kv->v & 15)) return KAIROS_ERR_ALIGN;
    const bool scaled = kv->dtype == KAIROS_DTYPE_I8 || kv->dtype == KAIROS_DTYPE_E4M3;
    if (!scaled && kv->dtype != KAIROS_DTYPE_F16 && kv->dtype != KAIROS_DTYPE_BF16) return KAIROS_ERR_ARG;
    if (scaled && (!kv->k_scale || !kv->v_scale || ((uintptr_t)kv->k_scale & 15) || ((uintptr_t)kv->v_scale & 15)))
        return KAIROS_ERR_ALIGN;
    *out = KvView{kv->k, kv->v, kv->k_scale, kv->v_scale, kv->pages, kv->kv_heads, shift, kv->head_dim};
    return KAIROS_OK;
}

// Row of the pool that holds kv head `head` of flat slot `slot` = page * page_size + offset.
__device__ __forceinline__ size_t pool_row(const KvView& kv, long long slot, int head) {
    const long long page = slot >> kv.page_shift;
    return (((size_t)page * kv.heads + head) << kv.page_shift) + (size_t)(slot & ((1 << kv.page_shift) - 1));
}

}  // namespace kairos
