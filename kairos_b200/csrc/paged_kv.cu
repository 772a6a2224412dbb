// Writing a paged key-value cache (rotary positions, quantization and the scatter in one pass over the fused QKV
// activation) and reading it back.  Both are HBM-bound: an activation is read once and a cache row written once.
// Measured on B200: 4099 tokens of 32 + 8 + 8 heads of 128 into int8 rows and back 24.7 us for the two kernels (118 MB: 18.0
// at the copy rate; the write alone 18.0 for 14.1), 16384 tokens of 14 + 2 + 2 heads into e4m3 rows and back 35.0 us (25.7; 28.8
// for 21.8); a step of 64 tokens 2.2 us; 50021 tokens of 8 heads read back from int8 52.4 us = 5.9 TB/s (0.90 of the copy
// rate).  With no angles to apply and no codes to check the e4m3 write would take 23.9 us: instructions and loads share the
// time where a block has its rows in two batches.
#include <cfloat>
#include <type_traits>

#include "paged_kv.cuh"

namespace kairos {

// Largest magnitude of a row held by `lanes` consecutive threads (a power of two, aligned), 16 values each; NaN if the row
// has an infinity or a NaN.  Magnitudes are compared as bit patterns, in whose order infinities and NaN are the largest.
__device__ __forceinline__ float row_amax(const float (&a)[8], const float (&b)[8], int lanes) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
    for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return __uint_as_float(m < 0x7f800000u ? m : 0x7fffffffu);
}

// Codes of eight values: the nearest of x / scale, as IEEE division rounds it.  With inv the rounded 1 / scale, x times
// inv (1 - 2^-22) and x times inv (1 + 2^-22) enclose the quotient, whatever their own roundings (3 * 2^-24 in all), so where
// both become the same code it is the quotient's.  A chunk with a value next to a border between two codes, or with a
// scale whose inverse is not a normal number, is divided.
constexpr float kBelow = 1.f - 2.384185791015625e-07f, kAbove = 1.f + 2.384185791015625e-07f;
struct CodesI8 {
    static constexpr float kTop = 127.f;
    static __device__ __forceinline__ uint2 encode(const float (&x)[8], float scale, float inv) {
        const float magic = 12582912.f;             // 1.5 * 2^23: adding it rounds to a whole number in the low byte
        const float below = inv * kBelow, above = inv * kAbove;
        uint32_t q[8], differ = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q[i] = __float_as_uint(__fmaf_rn(x[i], below, magic));
            differ |= q[i] ^ __float_as_uint(__fmaf_rn(x[i], above, magic));
        }
        if (differ || scale < FLT_MIN) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = (uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale))));
        }
        uint2 out;
        out.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        out.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
        return out;
    }
    static __device__ __forceinline__ void decode(const uint2& v, float (&f)[8]) {
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)));
    }
};
struct CodesE4M3 {
    static constexpr float kTop = 448.f;
    static __device__ __forceinline__ uint2 encode(const float (&x)[8], float scale, float inv) {
        const float below = inv * kBelow, above = inv * kAbove;
        uint32_t p[4], differ = 0;
        auto code2 = [](float a, float b) { return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = code2(x[2 * i] * below, x[2 * i + 1] * below);
            differ |= p[i] ^ code2(x[2 * i] * above, x[2 * i + 1] * above);
        }
        if (differ || scale < FLT_MIN) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = code2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale));
        }
        return make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
    }
    static __device__ __forceinline__ void decode(const uint2& v, float (&f)[8]) {
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
};

struct WriteShape {
    long long row_stride;
    int T, H, rot, layout, tokens_per_block;
    unsigned by_q, by_kv, by_pairs;             // div_magic of H, 2 kv heads and rot / 2
    float magnitude;
};

// Codes = void: the cache holds the activation's own type.  One block takes `tokens_per_block` tokens; the D / 16 cells of
// a row go to neighbouring threads of one warp, so the row's maximum is a few shuffles.  A thread requests its first cells
// before the block computes the tokens' angles, once for all heads, into shared memory beside their slots (each read where
// its rows are stored: 2% slower).
template <typename T, typename Codes, int D>
__global__ void __launch_bounds__(256, 4) rope_paged_kv_kernel(const T* __restrict__ QKV, const long long* __restrict__ positions,
                                                            const long long* __restrict__ slots,
                                                            const unsigned long long* __restrict__ steps, const KvView kv,
                                                            T* __restrict__ Q, const WriteShape p, int* status) {
    constexpr int kLanes = D / 16, kU = kCells<T>;
    __shared__ __align__(16) float cs[kTablePairs], sn[kTablePairs];
    __shared__ long long to_slot[kBlockTokens];
    chain_release();
    chain_wait();
    const int t0 = blockIdx.x * p.tokens_per_block;
    const int here = min(p.tokens_per_block, p.T - t0);
    // rows of the block: the q heads of its tokens, then their k and v heads, so that most warps have one kind
    const int pairs = p.rot >> 1, q_rows = here * p.H, rows = q_rows + 2 * here * kv.heads;
    auto split = [&](int r, int* t, int* head) {
        const bool q = r < q_rows;
        const int k = q ? r : r - q_rows, per = q ? p.H : 2 * kv.heads;
        *t = div_small(k, q ? p.by_q : p.by_kv);
        *head = k - *t * per + (q ? 0 : p.H);
    };
    const long long capacity = (long long)kv.pages << kv.page_shift;
    const int at = threadIdx.x / kLanes, j = threadIdx.x % kLanes, step = blockDim.x / kLanes;
    const Cell cell = cell_of(j, p.rot, p.layout);
    for (int base = 0; base < rows; base += kU * step) {
        RawCell<T> raw[kU];
        int ts[kU], heads[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            split(min(base + u * step + at, rows - 1), &ts[u], &heads[u]);  // whole warps stay together
            raw[u].load(QKV + (size_t)(t0 + ts[u]) * p.row_stride + heads[u] * D, cell);
        }
        if (base == 0) {
            if (threadIdx.x < here) to_slot[threadIdx.x] = __ldcg(slots + t0 + threadIdx.x);
            for (int i = threadIdx.x; i < here * pairs; i += blockDim.x) {
                const int t = div_small(i, p.by_pairs), pair = i - t * pairs;
                float c, s;
                turn_of(__ldcg(positions + t0 + t), __ldg(steps + pair), p.magnitude, &c, &s);
                const int to = t * pairs + table_place(pair, pairs);
                cs[to] = c;
                sn[to] = s;
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int t = ts[u], head = heads[u];
            float a[8], b[8];
            RawCell<T>::widen(raw[u].w[0], a);
            RawCell<T>::widen(raw[u].w[1], b);
            if (cell.pair >= 0 && head < p.H + kv.heads) turn_cell(a, b, cs + t * pairs, sn + t * pairs, cell.pair, pairs, p.layout);
            float amax = 0.f;
            if constexpr (!std::is_void<Codes>::value) {
                if (__any_sync(0xffffffffu, head >= p.H)) amax = row_amax(a, b, kLanes);
            }
            if (base + u * step + at >= rows) continue;
            if (head < p.H) {
                T* q = Q + ((size_t)(t0 + t) * p.H + head) * D;
                store8(q + cell.first, a);
                store8(q + cell.second, b);
                continue;
            }
            const long long slot = to_slot[t];
            if (slot < 0) continue;                        // padding
            if (slot >= capacity) {
                *status = KAIROS_ERR_ARG;
                continue;
            }
            const bool is_v = head >= p.H + kv.heads;
            const size_t to = pool_row(kv, slot, head - p.H - (is_v ? kv.heads : 0));
            if constexpr (std::is_void<Codes>::value) {
                T* y = static_cast<T*>(is_v ? kv.v : kv.k) + to * D;
                store8(y + cell.first, a);
                store8(y + cell.second, b);
            } else {
                const float scale = __fdiv_rn(amax, Codes::kTop);
                uint2 qa = make_uint2(0, 0), qb = qa;
                if (scale > 0.f) {                         // false for a row of zeros and for NaN: codes 0
                    const float inv = __frcp_rn(scale);
                    qa = Codes::encode(a, scale, inv);
                    qb = Codes::encode(b, scale, inv);
                }
                uint8_t* y = static_cast<uint8_t*>(is_v ? kv.v : kv.k) + to * D;
                *reinterpret_cast<uint2*>(y + cell.first) = qa;
                *reinterpret_cast<uint2*>(y + cell.second) = qb;
                if (j == 0) (is_v ? kv.vs : kv.ks)[to] = scale;
            }
        }
    }
}

// One thread brings the same eight channels of a K row and of its V row, of two rows half the grid apart, so that four
// independent rows are under way.
template <typename C, typename Codes, typename T>
__global__ void __launch_bounds__(256) paged_kv_read_kernel(const KvView kv, const long long* __restrict__ slots,
                                                            T* __restrict__ K, T* __restrict__ V, int total, int half,
                                                            unsigned by_heads, int* status) {
    constexpr bool kCoded = !std::is_void<Codes>::value;
    chain_release();
    chain_wait();
    const int chunk_shift = kv.dim == 64 ? 3 : kv.dim == 128 ? 4 : 5;
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= half) return;
    const int c = 8 * (i & ((1 << chunk_shift) - 1));
    const long long capacity = (long long)kv.pages << kv.page_shift;
    uint4 kw[2], vw[2];
    float ks[2] = {}, vs[2] = {};
    bool there[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int row = (i + u * half) >> chunk_shift;
        const bool mine = i + u * half < total;
        const int token = by_heads ? (int)__umulhi((unsigned)row, by_heads) : row;
        const long long slot = mine ? __ldcg(slots + token) : -1;
        there[u] = slot >= 0 && slot < capacity;
        if (slot >= capacity) *status = KAIROS_ERR_ARG;
        kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
        if (there[u]) {
            const size_t r = pool_row(kv, slot, row - token * kv.heads);
            if constexpr (kCoded) {
                const uint2 x = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(kv.k) + r * kv.dim + c));
                const uint2 y = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(kv.v) + r * kv.dim + c));
                kw[u].x = x.x, kw[u].y = x.y, vw[u].x = y.x, vw[u].y = y.y;
                ks[u] = __ldcg(kv.ks + r), vs[u] = __ldcg(kv.vs + r);
            } else {
                kw[u] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const C*>(kv.k) + r * kv.dim + c));
                vw[u] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const C*>(kv.v) + r * kv.dim + c));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (i + u * half >= total) break;
        const size_t to = (size_t)(i + u * half) * 8;
        auto put8 = [&](const uint4& w, float scale, T* out) {
            float f[8];
            if constexpr (kCoded) {
                Codes::decode(make_uint2(w.x, w.y), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= scale;
            } else {
                const uint4 one[1] = {w};
                RawCell<C>::widen(one, f);
            }
            store8(out + to, f);
        };
        put8(kw[u], ks[u], K);
        put8(vw[u], vs[u], V);
    }
}

template <typename T, typename Codes, int D>
static int run_write(const void* QKV, const void* positions, const void* slots, const void* steps, const KvView& kv, void* Q,
                     WriteShape p, int* status, cudaStream_t st) {
    const RowBlocks form = row_blocks(p.T, p.H + 2 * kv.heads, p.rot, 128 / (D / 16), kCells<T>, 64);
    p.tokens_per_block = form.tokens;
    p.by_q = div_magic(p.H);
    p.by_kv = div_magic(2 * kv.heads);
    p.by_pairs = div_magic(max(1, p.rot / 2));
    const cudaError_t e = launch_chained(
        rope_paged_kv_kernel<T, Codes, D>, dim3((unsigned)((p.T + p.tokens_per_block - 1) / p.tokens_per_block)), dim3(form.threads), 0,
        st, static_cast<const T*>(QKV), static_cast<const long long*>(positions), static_cast<const long long*>(slots),
        static_cast<const unsigned long long*>(steps), kv, static_cast<T*>(Q), p, status);
    if (e != cudaSuccess) return note_cuda_error(e);
    return launch_status();
}

template <typename T, typename Codes>
static int pick_write(const void* QKV, const void* positions, const void* slots, const void* steps, const KvView& kv, void* Q,
                      const WriteShape& p, int* status, cudaStream_t st) {
    if (kv.dim == 64) return run_write<T, Codes, 64>(QKV, positions, slots, steps, kv, Q, p, status, st);
    if (kv.dim == 128) return run_write<T, Codes, 128>(QKV, positions, slots, steps, kv, Q, p, status, st);
    return run_write<T, Codes, 256>(QKV, positions, slots, steps, kv, Q, p, status, st);
}

template <typename C, typename Codes, typename T>
static int run_read(const KvView& kv, const void* slots, void* K, void* V, long long T_, int* status, cudaStream_t st) {
    // whole tokens a launch, so that 32-bit indexes and the division by a multiplication are exact (rows * heads < 2^32)
    const long long per_token = (long long)kv.heads * (kv.dim / 8);
    const long long most = max(1LL, min((1LL << 30) / per_token, (long long)0xffffffffLL / kv.heads / kv.heads));
    for (long long t0 = 0; t0 < T_; t0 += most) {
        const int total = (int)(min(most, T_ - t0) * per_token);
        const int half = ((total / 2 + 255) & ~255) + (total < 512 ? total : 0);
        const cudaError_t e = launch_chained(paged_kv_read_kernel<C, Codes, T>, dim3((min(half, total) + 255) / 256), dim3(256), 0, st,
                                             kv, static_cast<const long long*>(slots) + t0,
                                             static_cast<T*>(K) + t0 * kv.heads * kv.dim, static_cast<T*>(V) + t0 * kv.heads * kv.dim,
                                             total, min(half, total), div_magic(kv.heads), status);
        if (e != cudaSuccess) return note_cuda_error(e);
    }
    return launch_status();
}

template <typename T>
static int pick_read(int dtype, const KvView& kv, const void* slots, void* K, void* V, long long n, int* status,
                     cudaStream_t st) {
    switch (dtype) {
        case KAIROS_DTYPE_F16: return run_read<__half, void, T>(kv, slots, K, V, n, status, st);
        case KAIROS_DTYPE_BF16: return run_read<__nv_bfloat16, void, T>(kv, slots, K, V, n, status, st);
        case KAIROS_DTYPE_I8: return run_read<uint8_t, CodesI8, T>(kv, slots, K, V, n, status, st);
        default: return run_read<uint8_t, CodesE4M3, T>(kv, slots, K, V, n, status, st);
    }
}

int* device_status_word();   // api.cu

}  // namespace kairos

extern "C" int kairos_rope_paged_kv(const void* QKV, long long row_stride, const void* positions, const void* slots,
                                    const kairos_rotary_plan* plan, const kairos_kv_layer* layer, void* Q_out, int T, int H,
                                    int dtype, kairos_stream_t stream) {
    using namespace kairos;
    KvView kv;
    const int rc = kv_view(layer, &kv);
    if (rc != KAIROS_OK) return rc;
    if (T < 0 || H <= 0 || row_stride % 8 != 0 || row_stride < (long long)(H + 2LL * kv.heads) * kv.dim) return KAIROS_ERR_SHAPE;
    if (H + 2LL * kv.heads >= 65536) return KAIROS_ERR_SHAPE;
    if (!rotary_plan_ok(plan, kv.dim) || plan->rot % 16 != 0) {
        set_last_error("rope_paged_kv: the rotated part is a multiple of 16 channels, at most the head");
        return KAIROS_ERR_ARG;
    }
    const bool coded = layer->dtype == KAIROS_DTYPE_I8 || layer->dtype == KAIROS_DTYPE_E4M3;
    if ((dtype != KAIROS_DTYPE_F16 && dtype != KAIROS_DTYPE_BF16) || (!coded && layer->dtype != dtype)) {
        set_last_error("rope_paged_kv: activations are fp16 or bf16, and a 16-bit cache has their type");
        return KAIROS_ERR_ARG;
    }
    if (T == 0) return KAIROS_OK;
    if (!QKV || !Q_out || !positions || !slots || ((uintptr_t)QKV & 15) || ((uintptr_t)Q_out & 15) ||
        ((uintptr_t)positions & 7) || ((uintptr_t)slots & 7))
        return KAIROS_ERR_ALIGN;
    int* status = device_status_word();
    if (!status) return KAIROS_ERR_CUDA;
    WriteShape p = {};
    p.row_stride = row_stride;
    p.T = T; p.H = H; p.rot = plan->rot; p.layout = plan->layout; p.magnitude = plan->magnitude;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const void* s = plan->steps;
    if (dtype == KAIROS_DTYPE_F16) {
        if (layer->dtype == KAIROS_DTYPE_I8) return pick_write<__half, CodesI8>(QKV, positions, slots, s, kv, Q_out, p, status, st);
        if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_write<__half, CodesE4M3>(QKV, positions, slots, s, kv, Q_out, p, status, st);
        return pick_write<__half, void>(QKV, positions, slots, s, kv, Q_out, p, status, st);
    }
    if (layer->dtype == KAIROS_DTYPE_I8) return pick_write<__nv_bfloat16, CodesI8>(QKV, positions, slots, s, kv, Q_out, p, status, st);
    if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_write<__nv_bfloat16, CodesE4M3>(QKV, positions, slots, s, kv, Q_out, p, status, st);
    return pick_write<__nv_bfloat16, void>(QKV, positions, slots, s, kv, Q_out, p, status, st);
}

extern "C" int kairos_paged_kv_read(const kairos_kv_layer* layer, const void* slots, void* K_out, void* V_out, int T, int dtype,
                                    kairos_stream_t stream) {
    using namespace kairos;
    KvView kv;
    const int rc = kv_view(layer, &kv);
    if (rc != KAIROS_OK) return rc;
    if (T < 0) return KAIROS_ERR_SHAPE;
    if (dtype != KAIROS_DTYPE_F16 && dtype != KAIROS_DTYPE_BF16 && dtype != KAIROS_DTYPE_F32) return KAIROS_ERR_ARG;
    if (T == 0) return KAIROS_OK;
    if (!K_out || !V_out || !slots || ((uintptr_t)K_out & 15) || ((uintptr_t)V_out & 15) || ((uintptr_t)slots & 7))
        return KAIROS_ERR_ALIGN;
    int* status = device_status_word();
    if (!status) return KAIROS_ERR_CUDA;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == KAIROS_DTYPE_F16) return pick_read<__half>(layer->dtype, kv, slots, K_out, V_out, T, status, st);
    if (dtype == KAIROS_DTYPE_BF16) return pick_read<__nv_bfloat16>(layer->dtype, kv, slots, K_out, V_out, T, status, st);
    return pick_read<float>(layer->dtype, kv, slots, K_out, V_out, T, status, st);
}
