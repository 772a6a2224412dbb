// Rotary positions of a tensor of heads (kairos_rotary): pair (a, b) -> m (a cos - b sin, b cos + a sin) of the angle
// position * f, in fp32, one rounding at the end.  HBM-bound: every element is read and written once, 16 bytes at a time;
// the angles cost one integer product and two short series per (token, pair) and are shared by all heads of the token.
// Measured on B200: 16381 x 32 heads of 128 in bf16 43.8 us = 6.1 TB/s (0.93 of the copy rate), 4099 x 28 in fp32 20.3 us =
// 5.8 TB/s, eight tokens 2.2 us, as much as an empty launch.
#include "rotary.cuh"

namespace kairos {

struct RotaryShape {
    long long xb, xs, xh, yb, ys, yh, pb, ps;   // element strides of X, Y and the positions
    long long tokens;                            // B * S, below 2^31
    int S, H, D, rot, layout, tokens_per_block;
    unsigned by_heads, by_pairs, by_lanes;       // div_magic of H, rot / 2, D / 16
    float magnitude, sign;
};

// One block turns `tokens_per_block` tokens.  A row's D / 16 cells go to neighbouring threads; a thread requests its first
// cells before the block computes the tokens' angles, once for all heads, into shared memory.
template <typename T>
__global__ void __launch_bounds__(256, 4) rotary_kernel(const T* X, T* Y, const long long* __restrict__ positions,
                                                     const unsigned long long* __restrict__ steps, const RotaryShape p) {
    constexpr int kU = kCells<T>;
    __shared__ __align__(16) float cs[kTablePairs], sn[kTablePairs];
    chain_release();
    chain_wait();
    const long long t0 = (long long)blockIdx.x * p.tokens_per_block;
    const int here = (int)min((long long)p.tokens_per_block, p.tokens - t0);
    const int pairs = p.rot >> 1, lanes = p.D >> 4, rows = here * p.H;
    const int at = div_small((int)threadIdx.x, p.by_lanes), j = (int)threadIdx.x - at * lanes;
    const int step = div_small(blockDim.x, p.by_lanes);        // rows in one go; threads behind the last whole row idle
    const bool idle = at >= step;
    const Cell cell = cell_of(j, p.rot, p.layout);
    auto place = [&](int r, long long sb, long long ss, long long sh) {
        const int t = div_small(r, p.by_heads);
        const long long token = t0 + t, b = p.S == p.tokens ? 0 : (unsigned)token / (unsigned)p.S;
        return b * sb + (token - b * p.S) * ss + (r - t * p.H) * sh;
    };
    for (int base = 0; base < rows; base += kU * step) {
        RawCell<T> raw[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int r = base + u * step + at;
            if (r < rows && !idle) raw[u].load(X + place(r, p.xb, p.xs, p.xh), cell);
        }
        if (base == 0) {
            for (int i = threadIdx.x; i < here * pairs; i += blockDim.x) {
                const int t = div_small(i, p.by_pairs), pair = i - t * pairs;
                const long long token = t0 + t, b = p.S == p.tokens ? 0 : (unsigned)token / (unsigned)p.S;
                float c, s;
                turn_of(__ldcg(positions + b * p.pb + (token - b * p.S) * p.ps), __ldg(steps + pair), p.magnitude, &c, &s);
                const int to = t * pairs + table_place(pair, pairs);
                cs[to] = c;
                sn[to] = s * p.sign;
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int r = base + u * step + at;
            if (r >= rows || idle) continue;
            float a[8], b[8];
            RawCell<T>::widen(raw[u].w[0], a);
            RawCell<T>::widen(raw[u].w[1], b);
            const int t = div_small(r, p.by_heads);
            if (cell.pair >= 0) turn_cell(a, b, cs + t * pairs, sn + t * pairs, cell.pair, pairs, p.layout);
            T* y = Y + place(r, p.yb, p.ys, p.yh);
            store8(y + cell.first, a);
            store8(y + cell.second, b);
        }
    }
}

// Rows that do not move in 16-byte accesses: one thread per pair, or per two elements behind `rot`.
template <typename T>
__global__ void __launch_bounds__(256) rotary_scalar_kernel(const T* X, T* Y, const long long* __restrict__ positions,
                                                            const unsigned long long* __restrict__ steps,
                                                            const RotaryShape p) {
    chain_release();
    chain_wait();
    const int per_row = (p.D + 1) >> 1;
    const long long total = p.tokens * p.H * per_row;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int j = (int)(i % per_row);
        const long long row = i / per_row;
        const int h = (int)(row % p.H);
        const long long t = row / p.H, b = t / p.S, s = t - b * p.S;
        const T* x = X + b * p.xb + s * p.xs + h * p.xh;
        T* y = Y + b * p.yb + s * p.ys + h * p.yh;
        int e0 = 2 * j, e1 = 2 * j + 1;
        const bool turning = j < (p.rot >> 1);
        if (turning && p.layout == 0) {
            e0 = j;
            e1 = j + (p.rot >> 1);
        }
        float a = to_f32(x[e0]), c = e1 < p.D ? to_f32(x[e1]) : 0.f;
        if (turning) {
            float co, si;
            turn_of(__ldcg(positions + b * p.pb + s * p.ps), __ldg(steps + j), p.magnitude, &co, &si);
            turn_pair(a, c, co, si * p.sign);
        }
        put(y + e0, a);
        if (e1 < p.D) put(y + e1, c);
    }
}

template <typename T>
static int run_rotary(const void* X, void* Y, const void* positions, const void* steps, RotaryShape p, cudaStream_t st) {
    const int per16 = 16 / (int)sizeof(T);
    const bool wide = p.H < 65536 && (p.D % 16) == 0 && (p.rot % 16) == 0 && ((uintptr_t)X & 15) == 0 && ((uintptr_t)Y & 15) == 0 &&
                      p.xb % per16 == 0 && p.xs % per16 == 0 && p.xh % per16 == 0 && p.yb % per16 == 0 &&
                      p.ys % per16 == 0 && p.yh % per16 == 0;
    const T* x = static_cast<const T*>(X);
    T* y = static_cast<T*>(Y);
    const long long* pos = static_cast<const long long*>(positions);
    const unsigned long long* st64 = static_cast<const unsigned long long*>(steps);
    cudaError_t e;
    if (wide) {
        const RowBlocks form = row_blocks(p.tokens, p.H, p.rot, 128 / (p.D / 16), kCells<T>, sizeof(T) == 4 ? 32 : 64);
        p.tokens_per_block = form.tokens;
        p.by_heads = div_magic(p.H);
        p.by_pairs = div_magic(max(1, p.rot / 2));
        p.by_lanes = div_magic(p.D / 16);
        const long long blocks = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
        e = launch_chained(rotary_kernel<T>, dim3((unsigned)blocks), dim3(form.threads), 0, st, x, y, pos, st64, p);
    } else {
        const long long total = p.tokens * p.H * ((p.D + 1) / 2);
        const long long blocks = min((total + 255) / 256, (long long)1 << 20);
        e = launch_chained(rotary_scalar_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, x, y, pos, st64, p);
    }
    if (e != cudaSuccess) return note_cuda_error(e);
    return launch_status();
}

}  // namespace kairos

extern "C" int kairos_rotary(const void* X, long long x_b, long long x_s, long long x_h, void* Y, long long y_b, long long y_s,
                             long long y_h, const void* positions, long long pos_b, long long pos_s,
                             const kairos_rotary_plan* plan, int dtype, int transpose, int B, int S, int H, int D,
                             kairos_stream_t stream) {
    using namespace kairos;
    if (B < 0 || S < 0 || H < 0 || D <= 0 || D > 512) return KAIROS_ERR_SHAPE;
    if ((long long)B * S > 0x7fffffffLL) return KAIROS_ERR_SHAPE;      // one block per token at the least
    if (!rotary_plan_ok(plan, D)) return KAIROS_ERR_ARG;
    if (B == 0 || S == 0 || H == 0) return KAIROS_OK;
    if (!X || !Y || !positions || ((uintptr_t)positions & 7)) return KAIROS_ERR_ALIGN;
    RotaryShape p = {};
    p.xb = x_b; p.xs = x_s; p.xh = x_h;
    p.yb = y_b; p.ys = y_s; p.yh = y_h;
    p.pb = pos_b; p.ps = pos_s;
    p.tokens = (long long)B * S;
    p.S = S; p.H = H; p.D = D; p.rot = plan->rot; p.layout = plan->layout;
    p.magnitude = plan->magnitude;
    p.sign = transpose ? -1.f : 1.f;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case KAIROS_DTYPE_F16: return run_rotary<__half>(X, Y, positions, plan->steps, p, st);
        case KAIROS_DTYPE_BF16: return run_rotary<__nv_bfloat16>(X, Y, positions, plan->steps, p, st);
        case KAIROS_DTYPE_F32: return run_rotary<float>(X, Y, positions, plan->steps, p, st);
        default: return KAIROS_ERR_ARG;
    }
}
