// Attention of one new token per sequence over a paged key-value cache (kairos_paged_attention).
#include "paged_kv.cuh"

namespace kairos {

template <typename C> __device__ __forceinline__ float cache_f32(C v) { return to_f32(v); }
template <> __device__ __forceinline__ float cache_f32<signed char>(signed char v) { return (float)v; }
template <> __device__ __forceinline__ float cache_f32<__nv_fp8_e4m3>(__nv_fp8_e4m3 v) { return (float)v; }

struct AttnShape {
    long long qb, qh, table_stride;
    int table_width, H, group;
    float scale;
};

// One warp per (sequence, query head): every lane holds D / 32 channels; the softmax's running maximum and sum are
// updated key by key, in fp32.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(32) paged_attention_kernel(const T* Q, const KvView kv, const int* __restrict__ table,
                                                             const int* __restrict__ lens, T* O, float* LSE,
                                                             const AttnShape p, int* status) {
    constexpr int E = D / 32;
    chain_release();
    chain_wait();
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
    int len = lens[b];
    const int most = p.table_width << kv.page_shift;
    if (len > most) {
        *status = KAIROS_ERR_ARG;
        len = most;
    }
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) q[e] = to_f32(Q[b * p.qb + h * p.qh + lane + 32 * e]);
    const C* kp = static_cast<const C*>(kv.k);
    const C* vp = static_cast<const C*>(kv.v);
    for (int j = 0; j < len; ++j) {
        const int page = table[b * p.table_stride + (j >> kv.page_shift)];
        if ((unsigned)page >= (unsigned)kv.pages) {
            *status = KAIROS_ERR_ARG;
            continue;
        }
        const size_t r = pool_row(kv, ((long long)page << kv.page_shift) + (j & ((1 << kv.page_shift) - 1)), h / p.group);
        float s = 0.f;
        for (int e = 0; e < E; ++e) s = __fmaf_rn(q[e], cache_f32(kp[r * D + lane + 32 * e]), s);
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= p.scale;
        float vs = 1.f;
        if (kv.ks) {
            s *= kv.ks[r];
            vs = kv.vs[r];
        }
        const float top = fmaxf(m, s), safe = top == -INFINITY ? 0.f : top;
        const float keep = expf(m - safe), weight = expf(s - safe);
        l = __fmaf_rn(l, keep, weight);
        for (int e = 0; e < E; ++e) o[e] = __fmaf_rn(weight * vs, cache_f32(vp[r * D + lane + 32 * e]), o[e] * keep);
        m = top;
    }
    const float inv = len > 0 ? 1.f / l : 0.f;
    for (int e = 0; e < E; ++e) put(O + ((size_t)b * p.H + h) * D + lane + 32 * e, o[e] * inv);
    if (LSE && lane == 0) LSE[(size_t)b * p.H + h] = len > 0 ? m + logf(l) : -INFINITY;
}

template <typename T, typename C>
static int pick_attention(const void* Q, const KvView& kv, const void* table, const void* lens, void* O, void* LSE,
                          const AttnShape& p, int B, int* status, cudaStream_t st) {
    auto kernel = kv.dim == 64 ? paged_attention_kernel<T, C, 64>
                               : kv.dim == 128 ? paged_attention_kernel<T, C, 128> : paged_attention_kernel<T, C, 256>;
    const cudaError_t e = launch_chained(kernel, dim3(p.H, B), dim3(32), 0, st, static_cast<const T*>(Q), kv,
                                         static_cast<const int*>(table), static_cast<const int*>(lens), static_cast<T*>(O),
                                         static_cast<float*>(LSE), p, status);
    if (e != cudaSuccess) return note_cuda_error(e);
    return launch_status();
}

int* device_status_word();   // api.cu

}  // namespace kairos

extern "C" size_t kairos_paged_attention_workspace_bytes(const kairos_kv_layer* layer, int B, int H, int table_width) {
    return 0;
}

extern "C" int kairos_paged_attention(const void* Q, const long long* q_strides, const kairos_kv_layer* layer,
                                      const void* page_table, long long table_stride, int table_width, const void* lens,
                                      void* O, void* LSE, int B, int H, float scale, int dtype, void* workspace,
                                      size_t workspace_bytes, kairos_stream_t stream) {
    using namespace kairos;
    KvView kv;
    const int rc = kv_view(layer, &kv);
    if (rc != KAIROS_OK) return rc;
    if (B < 0 || B > 65535 || H <= 0 || H % kv.heads != 0 || table_width < 0 || table_stride < 0 || !q_strides ||
        ((long long)table_width << kv.page_shift) > 0x7fffffffLL)
        return KAIROS_ERR_SHAPE;
    const bool coded = layer->dtype == KAIROS_DTYPE_I8 || layer->dtype == KAIROS_DTYPE_E4M3;
    if ((dtype != KAIROS_DTYPE_F16 && dtype != KAIROS_DTYPE_BF16) || (!coded && layer->dtype != dtype)) {
        set_last_error("paged_attention: queries are fp16 or bf16, and a 16-bit cache has their type");
        return KAIROS_ERR_ARG;
    }
    if (q_strides[0] % 8 != 0 || q_strides[1] % 8 != 0) return KAIROS_ERR_ALIGN;
    if (B == 0) return KAIROS_OK;
    if (!Q || !O || !lens || (!page_table && table_width > 0) || ((uintptr_t)Q & 15) || ((uintptr_t)O & 15) ||
        ((uintptr_t)page_table & 3) || ((uintptr_t)lens & 3) || ((uintptr_t)LSE & 3))
        return KAIROS_ERR_ALIGN;
    int* status = device_status_word();
    if (!status) return KAIROS_ERR_CUDA;
    AttnShape p = {q_strides[0], q_strides[1], table_stride, table_width, H, H / kv.heads, scale};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == KAIROS_DTYPE_F16) {
        if (layer->dtype == KAIROS_DTYPE_I8) return pick_attention<__half, signed char>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
        if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_attention<__half, __nv_fp8_e4m3>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
        return pick_attention<__half, __half>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
    }
    if (layer->dtype == KAIROS_DTYPE_I8) return pick_attention<__nv_bfloat16, signed char>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
    if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_attention<__nv_bfloat16, __nv_fp8_e4m3>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
    return pick_attention<__nv_bfloat16, __nv_bfloat16>(Q, kv, page_table, lens, O, LSE, p, B, status, st);
}
