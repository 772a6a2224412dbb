// Rotary positions of a tensor of heads (kairos_rotary).  HBM-bound: every element is read and written once; the
// angles cost one integer product and one sincospif per (token, pair) and are shared by all heads of the token.
#include "rotary.cuh"

namespace kairos {

struct RotaryShape {
    long long xb, xs, xh, yb, ys, yh, pb, ps;   // element strides of X, Y and the positions
    long long tokens;                            // B * S
    int S, H, D, rot, layout, tokens_per_block;
    float magnitude, sign;
};

// One block turns `tokens_per_block` tokens: their angles go to shared memory once, then every thread moves cells.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const T* X, T* Y, const long long* __restrict__ positions,
                                                     const unsigned long long* __restrict__ steps, const RotaryShape p) {
    __shared__ __align__(16) float cs[kTablePairs], sn[kTablePairs];
    chain_release();
    chain_wait();
    const long long t0 = (long long)blockIdx.x * p.tokens_per_block;
    const int here = (int)min((long long)p.tokens_per_block, p.tokens - t0);
    const int pairs = p.rot >> 1;
    for (int i = threadIdx.x; i < here * pairs; i += 256) {
        const int t = i / pairs, pair = i - t * pairs;
        const long long b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
        float c, sv;
        turn_of(__ldcg(positions + b * p.pb + s * p.ps), __ldg(steps + pair), p.magnitude, &c, &sv);
        cs[i] = c;
        sn[i] = sv * p.sign;
    }
    __syncthreads();
    const int per_row = p.D >> 4;
    const int per_token = p.H * per_row;
    for (int i = threadIdx.x; i < here * per_token; i += 256) {
        const int t = i / per_token, k = i - t * per_token;
        const int h = k / per_row, j = k - h * per_row;
        const long long b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
        const T* x = X + b * p.xb + s * p.xs + h * p.xh;
        T* y = Y + b * p.yb + s * p.ys + h * p.yh;
        const Cell cell = cell_of(j, p.rot, p.layout);
        float a[8], c[8];
        load8(x + cell.first, a);
        load8(x + cell.second, c);
        if (cell.pair >= 0) turn_cell(a, c, cs + t * pairs, sn + t * pairs, cell.pair, p.layout);
        store8(y + cell.first, a);
        store8(y + cell.second, c);
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
    const bool wide = (p.D % 16) == 0 && (p.rot % 16) == 0 && ((uintptr_t)X & 15) == 0 && ((uintptr_t)Y & 15) == 0 &&
                      p.xb % per16 == 0 && p.xs % per16 == 0 && p.xh % per16 == 0 && p.yb % per16 == 0 &&
                      p.ys % per16 == 0 && p.yh % per16 == 0;
    const T* x = static_cast<const T*>(X);
    T* y = static_cast<T*>(Y);
    const long long* pos = static_cast<const long long*>(positions);
    const unsigned long long* st64 = static_cast<const unsigned long long*>(steps);
    cudaError_t e;
    if (wide) {
        // a block has at least 256 cells where the heads of one token are few, and its angles fit its table
        const int cells = p.H * (p.D / 16);
        int tb = cells >= 256 ? 1 : (256 + cells - 1) / cells;
        if (p.rot) tb = min(tb, kTablePairs / (p.rot / 2));
        p.tokens_per_block = max(1, tb);
        const long long blocks = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
        e = launch_chained(rotary_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, x, y, pos, st64, p);
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
