// Attention of one new token per sequence over a paged key-value cache (kairos_paged_attention).
//
// Mathematics.  Per query head, with s_j = scale * q.k_j in units of log2 e:  o = sum_j 2^(s_j - m) v_j / l,
// l = sum_j 2^(s_j - m), m = max_j s_j, in ONE pass over the cache: m, l and o are kept for the keys seen so far and
// multiplied by 2^(m_old - m_new) where the maximum moves.  Parts of a sequence are joined by the same rule.
//
// Bound.  With up to 16 query heads per kv head every cached byte is read once and meets 2 * group flops (group = query heads
// per kv head): below 16 flops a byte, so HBM sets the pace and everything here serves to keep loads in flight.  Each further
// 16 heads are blocks of their own that ask for the pages again (64 sequences up to 4000 positions, 4 kv heads of 128: 16 heads a
// kv head 56 us, 32 75, 48 101 over fp16 rows, 48, 78 and 105 over int8 ones).
//   * a warp owns a ring of stages of 16 positions (8 KB of K and V rows of 128 fp16 channels), filled by 16-byte
//     cp.async with a swizzle of its own; no block-wide barrier until a pair ends, and the next pair is requested first;
//   * the heads that share a kv head are the eight columns of warp-level tensor instructions (m16n8k16): scores^T = K q^T
//     (16 positions a step) and o^T = V^T w^T (16 channels), so a key is read from shared memory once for all of them and
//     no row of a product is empty.  tcgen05 would take 128 positions by eight heads from shared or tensor memory, where
//     codes would have to be written back once widened, and return them through tensor memory; the tensor pipe is 9%
//     busy as it is (19% for codes), so there is nothing to gain from it;
//   * the work goes to blocks by one of three rules (make_plan): a block or a cluster of blocks per pair, many waves of
//     such blocks, or an even cut on the device, whatever the lengths are.  A pair that lies across blocks of the cut
//     leaves one partial result per block in the workspace and a second kernel joins them in the order of the blocks (no
//     atomics: same bits every run).
// Measured on B200, six to twelve calls in a graph: one sequence of 131071 bf16 positions, 8 kv heads: 84.9 us = 6.33 TB/s (0.97
// of the copy rate); 128 sequences of 2048 fp16 positions 161 us = 6.7 TB/s, in int8 92.5 us = 6.0 TB/s; 128 of 1 to 8192 in int8
// 177 us = 6.3 TB/s (back to back for a second, under the power cap, 203); 2 x 1024 positions 6.6 us; 64 positions 3.5 us (2.2 us
// is an empty launch).  For codes the instruction stream comes next: 383 warp instructions per 16 positions, 176 of them widening
// codes, take 60% of the issue slots.  Rows of 64 int8 channels, half the bytes for more than half the instructions, reach
// 5.4 TB/s (128 sequences of 8192: 210 us).
//
// Precision.  Scores, references, sums and outputs are fp32.  What has fewer bits, since tensor instructions take 16-bit
// operands, and why that is enough beside an output of 11 (fp16) or 8 bits (bf16):
//   * the weights of the second product (over codes: weight times V scale) are TWO 16-bit numbers, value and remainder; one alone
//     would add an error as large as the output's own rounding.  Over bf16 rows they are off by 2^-16 of each weight; over fp16 rows
//     2^-22 of each, but no less than 2^-37 of the head's largest; over codes the same with 2^-33 of the largest product;
//   * bf16 queries over codes become fp16 times a power of two per head: exact to 2^-38 of the head's largest value.
// Exponentials are ex2.approx (2 U); an argument below -126 gives 0: weights of less than 2^-110 of the reference (fp16 rows:
// 2^-138).  The reference need not be the maximum: it moves (and o and l are rescaled) only when a score passes it by 2^slack, so
// most stages need neither a reduction over lanes nor a rescaling.
#include <cfloat>
#include <type_traits>

#include "paged_kv.cuh"

namespace kairos {

int* device_status_word();   // api.cu

constexpr int kWarps = 4;
constexpr int kSub = 16;                    // positions of a stage
constexpr int kTile = kSub * kWarps;        // positions per scheduling tile
// Weights are kept times 2^lift and pass the reference by 2^slack at the most.  Over fp16 rows they are fp16 numbers themselves
// and stay below 2^15; the smallest step is 2^-36 of a weight at the reference (a slack of 2^8 and steps of 2^-30 measure the
// same within 0.2%).  Over bf16 rows and codes nothing but fp32 bounds them, and they are kept small instead, so that sums of
// values up to bf16's largest stay finite.
template <bool kHalfRows>
struct Span {
    static constexpr float kLift = kHalfRows ? 12.f : -16.f, kSlack = kHalfRows ? 3.f : 8.f;
    static constexpr float kMost = kHalfRows ? 32768.f : 1.f / 256.f;      // 2^(lift + slack)
};
// Reference of a head before its first score: any score passes it.  References are finite, so that differences of two are
// never NaN; a head that has seen no score has a sum of 0.
constexpr float kUnset = -FLT_MAX;
// Coded caches: what enters the second product is weight * V scale, and each head keeps a power of two of its own under it: the
// largest product so far lies between 2^8 and 2^9 when the power is set and below 2^15 until the next time, so fp16's smallest
// step is 2^-32 of it.  A row's scale alone sets nothing: one that is 2^60 times the others', with a weight of 2^-90, takes
// no bits from them.  (2^12 in place of 2^8 moves the power more often: 64 sequences up to 4000 positions in int8, 16 heads a
// kv head, 51.2 us from 48.2.)
constexpr int kLargest = 8;
constexpr float kOver = 32768.f;
// Inverse of a power of two.
__device__ __forceinline__ float inverse_pow2(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnShape {
    long long qb, qh, table_stride;
    int B, H, group, blocks_per_kv;         // head blocks (of 8 or 16 query heads) per kv head
    int table_width, workers, lanes;        // the even cut: workers in `lanes` equal parts, each with its own pairs
    int cluster;                            // blocks of a cluster that share one pair; 0: the even cut over all workers
    float scale_log2;
};

// ---- the cut of the work --------------------------------------------------------------------------------
__device__ __forceinline__ int seq_len(const int* lens, int b, int most) { return max(0, min(__ldcg(lens + b), most)); }

struct Cut {
    unsigned total, run;                    // units of a lane, units per worker
    int b, pair, unit;                      // where the worker begins: sequence, pair (kv head, head block) and unit of it
    int len;                                // of that sequence
};

// The work of a pair in units: a tile of positions each, and kEnding more for ending it (joining the warps, starting the
// next pair); none for an empty sequence.
constexpr int kEnding = 2;                  // 1: 64 sequences of 1 to 4000 positions 90.1 us for 85.7; 3: 86.0
__device__ __forceinline__ unsigned units_of(int len) { return len > 0 ? (unsigned)(len + kTile - 1) / kTile + kEnding : 0; }

// Units that a block may take over what an even cut gives it before cutting pays: a join costs about as long as a block
// needs for so many.
constexpr unsigned kSpare = 6;

// Block-wide (128 threads).  Scans the sequences' units and finds where worker blockIdx.x begins; returns false where it
// has no work.  Pair p belongs to lane p % lanes and worker w is number w / lanes of lane w % lanes; a lane's pairs lie end
// to end, sequence after sequence, and its workers take equal runs.  With a lane per pair of a sequence, neighbouring
// workers read the same pages' heads at the same time.  If every pair is short -- no more than kSpare units over the even
// run -- and there are no more pairs than workers, a worker takes one whole pair (run = 0).
__device__ __forceinline__ bool locate(const int* lens, const AttnShape& p, int pairs, int most, Cut* out) {
    __shared__ unsigned warp_sum[kWarps], warp_top[kWarps];
    __shared__ Cut found;
    const int tid = threadIdx.x, per = (p.B + 127) >> 7;
    const int first = tid * per, last = min(p.B, first + per);
    unsigned mine = 0, top = 0;
    int own_len = 0;                        // the only length of this thread where there are no more sequences than threads
    for (int b = first; b < last; ++b) {
        own_len = seq_len(lens, b, most);
        const unsigned n = units_of(own_len);
        mine += n;
        top = max(top, n);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    unsigned upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
        if ((tid & 31) >= o) upto += v;
    }
    if ((tid & 31) == 31) warp_sum[tid >> 5] = upto, warp_top[tid >> 5] = top;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < (tid >> 5)) upto += warp_sum[w];
        total += warp_sum[w];
        top = max(top, warp_top[w]);
    }
    const unsigned deep = pairs / p.lanes, team = p.workers / p.lanes, rank = blockIdx.x / p.lanes;
    const int lane = blockIdx.x - rank * p.lanes;
    total *= deep;
    const unsigned run = (total + team - 1) / team;
    const bool whole = top <= run + kSpare && (long long)p.B * pairs <= p.workers;
    if (whole) {
        const int b = blockIdx.x / pairs;
        if (b >= p.B) return false;
        *out = Cut{total, 0, b, (int)(blockIdx.x - b * pairs), 0, seq_len(lens, b, most)};
        return out->len > 0;
    }
    const unsigned x = rank * run;
    if (x >= total) return false;           // the same for every thread
    unsigned before = upto - mine;
    if (x >= before * deep && x < upto * deep) {
        for (int b = first; b < last; ++b) {
            const int len = per == 1 ? own_len : seq_len(lens, b, most);
            const unsigned n = units_of(len);
            if (x < (before + n) * deep) {
                const unsigned rest = x - before * deep;
                found = Cut{total, run, b, (int)(rest / n) * p.lanes + lane, (int)(rest % n), len};
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    *out = found;
    return true;
}

// Partial results in the workspace: slot 2 w of worker w is the pair that its run begins in, slot 2 w + 1 the one that it
// ends in.  Behind them a record per worker: the pair that begins in its run and lies across the run's end, if there is one.
struct Crossing {
    int b, pair;
    unsigned slot, last;                    // this worker's part, the worker of the last part; last == the worker: none
};
template <int R, int D>
struct Partials {
    static constexpr size_t kFloats = (size_t)R * (D + 2);
    static __device__ __forceinline__ float* o(float* ws, unsigned slot) { return ws + slot * kFloats; }
    static __device__ __forceinline__ float* ml(float* ws, unsigned slot) { return ws + slot * kFloats + R * D; }
    static __device__ __forceinline__ Crossing* crossing(float* ws, int workers, unsigned worker) {
        return reinterpret_cast<Crossing*>(ws + 2 * (size_t)workers * kFloats) + worker;
    }
};
static_assert(sizeof(Crossing) == 16, "one 16-byte access");

// ---- instructions -------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void lds(uint32_t (&v)[4], uint32_t a) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void lds(uint32_t (&v)[2], uint32_t a) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(__half, float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(__nv_bfloat16, float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 operations in one instruction: what the loop does to the scores of heads 2 t and 2 t + 1 of a position (rows of 64
// int8 channels, 64 sequences up to 4000 positions: 37.6 us, 38.3 with an instruction each).
__device__ __forceinline__ uint64_t bits2(const float2& a) { return (uint64_t)__float_as_uint(a.y) << 32 | __float_as_uint(a.x); }
__device__ __forceinline__ float2 from_bits2(uint64_t a) { return make_float2(__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32))); }
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
    return from_bits2(r);
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
    return from_bits2(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
// What a row's sum is divided by.  Where no position was left (every page outside the pool) the row is an empty one: zeros, and
// a logarithm of -inf; NaN among the inputs stays NaN.
__device__ __forceinline__ float inverse_sum(float sum) { return sum == 0.f ? 0.f : __fdiv_rn(1.f, sum); }
// A thread-block cluster: barrier halves, and the shared memory of block `rank` at the address that `a` has in this one.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_map(uint32_t a, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
// Transposes an 8 x 8 matrix of 16-bit values held as ldmatrix delivers it.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two fp32 as a pair of 16-bit values, and the pair of what the rounding left.
__device__ __forceinline__ void split(__half, float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void split(__nv_bfloat16, float x, float y, uint32_t* hi, uint32_t* lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - __uint_as_float(b << 16), y - __uint_as_float(b & 0xffff0000u));
    *hi = b;
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void put4(__half* to, const float4& v, float f) {
    __half2 h[2] = {__floats2half2_rn(v.x * f, v.y * f), __floats2half2_rn(v.z * f, v.w * f)};
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(h);
}
__device__ __forceinline__ void put4(__nv_bfloat16* to, const float4& v, float f) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v.x * f, v.y * f), __floats2bfloat162_rn(v.z * f, v.w * f)};
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(h);
}

// Codes as fp16 pairs, exactly.  bytes 0, 1 -> first, 2, 3 -> second.
struct WidenI8 {      // 1024 + (code + 128) has the shifted code in its low byte
    static __device__ __forceinline__ void run(uint32_t w, uint32_t* first, uint32_t* second) {
        w ^= 0x80808080u;
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));    // 1152
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        *first = *reinterpret_cast<const uint32_t*>(&x);
        *second = *reinterpret_cast<const uint32_t*>(&y);
    }
};
struct WidenE4M3 {
    static __device__ __forceinline__ void run(uint32_t w, uint32_t* first, uint32_t* second) {
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(*first), "=r"(*second) : "r"(w));
    }
};

// ---- shared memory: where chunk c (16 bytes) of row r lies ----------------------------------------------------
// Rows of 128 bytes and more: the chunk index is xored with the row's low three bits, so eight rows of one chunk (an
// ldmatrix) and two chunks of four even rows (the V reads of coded caches) fall on different banks.  64-byte rows share a
// line in pairs.
template <int ROWB>
__device__ __forceinline__ uint32_t place(int r, int c) {
    if constexpr (ROWB >= 128) return r * ROWB + ((c ^ (r & 7)) << 4);
    else return r * ROWB + ((c ^ ((r >> 1) & 3)) << 4);
}

// A warp's ring of stages of 16 positions; stages and blocks on an SM by what registers and measurements allow.
// int8, 128 channels, 128 sequences up to 8192, six calls in a graph: 2 stages x 4 blocks an SM 176.6 us, 3 x 4 177.8, 4 x 3 181,
// 2 x 5 188 (within 0.2 each); of 2048 positions each 92.5, 94.4, 104 and 106; 64 up to 4000 55.3, 57.1, 58.8 and 61.  fp16, one
// of 131071: 3 x 2 84.9 us, 2 x 3 85.9, 4 x 1 102.  64 sequences up to 4000: 256 channels int8 2 x 2 96 us, 3 x 2 100, 4 x 1
// 134; 64 channels fp16 3 x 4 48.1, 4 x 3 49.2, 3 x 5 59; int8 2 x 4 37.2, 3 or 4 x 4 38.1, 2 x 5 38.0, 2 x 6 42.  Stages of 32
// positions cost 5 to 50% more in all of them.
template <int D, bool kCoded, int kHalves>
struct Ring {
    static constexpr int kRowBytes = kCoded ? D : 2 * D;
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kRows = kSub * kRowBytes;
    static constexpr int kStage = (2 * kRows + (kCoded ? 2 * kSub * 4 : 0) + kRowBytes - 1) / kRowBytes * kRowBytes;
    static constexpr int kStages = kCoded ? 2 : 3;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kBytes = kWarps * kRing + kRowBytes;                  // the rings begin at a multiple of a row
    static constexpr int kFit = kBytes > 112 * 1024 ? 1 : kBytes > 74 * 1024 || D == 256 ? 2 : kBytes > 55 * 1024 ? 3 : 4;
    static constexpr int kWide = D == 64 ? 4 : 3;                              // of 16 heads: twice the accumulators
    static constexpr int kBlocksPerSm = kHalves == 2 && kFit > kWide ? kWide : kFit;
    // A warp's output rows, when a pair ends, go to a free stage while the next pair is requested; where they need more than
    // a stage they take the ring and the next pair waits.
    static constexpr int kOut = 8 * kHalves * D * 4;
    static constexpr bool kWaits = kOut > kStage;
    static_assert(kOut <= kRing, "a warp's output rows fit its ring");
    static_assert(kStage % kRowBytes == 0, "stages begin at a multiple of a row: chunk addresses are xored into them");
    static constexpr int kSwizzle = kRowBytes >= 128 ? 7 : 0;                  // bits of a row that move its chunks (64 bytes: see place)
    static constexpr int kLastOut = kWaits ? 0 : kRing - kStage;               // where the rows go when nothing follows
};

// One worker's part of one pair.
struct Segment {
    int b, pair, tile, tiles, take, len;
};

// QT: type of q and o; Widen: void for a cache of type QT, else how codes become fp16; kBlockHeads: query heads of a block,
// 4, 8 or 16.  With 4, columns 4..7 of the products are the same heads again: their scores and weights come out the same
// without exchange, and in the second product the first four columns carry the weights and the others their remainders, so
// it is one instruction where 8 heads need two.
template <typename QT, typename Widen, int D, int kBlockHeads>
__global__ void __launch_bounds__(128, (Ring<D, !std::is_void<Widen>::value, (kBlockHeads + 7) / 8>::kBlocksPerSm))
    paged_attention_kernel(const QT* __restrict__ Q, const KvView kv, const int* __restrict__ table, const int* __restrict__ lens,
                           QT* __restrict__ O, float* __restrict__ LSE, float* __restrict__ ws, const AttnShape p, int* status) {
    constexpr bool kCoded = !std::is_void<Widen>::value, kTwin = kBlockHeads == 4;
    constexpr int kHalves = (kBlockHeads + 7) / 8;
    using MT = typename std::conditional<kCoded, __half, QT>::type;
    using R = Ring<D, kCoded, kHalves>;
    constexpr int kHeads = 8 * kHalves;
    using W = Span<!kCoded && std::is_same<QT, __half>::value>;
    constexpr float kLift = W::kLift, kSlack = W::kSlack, kMost = W::kMost;
    extern __shared__ __align__(128) uint8_t dynamic[];
    uint8_t* const smem = dynamic + ((0u - smem_u32(dynamic)) & (R::kRowBytes - 1));
    __shared__ float jm[kWarps][kHeads], jl[kWarps][kHeads];
    __shared__ uint32_t jslot[kWarps];
    __shared__ float2 jpart[kHeads];
    chain_wait();
    chain_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pairs = kv.heads * p.blocks_per_kv, most = p.table_width << kv.page_shift;
    Cut cut = {};
    unsigned left = 0;                          // units still to take: a run of the even cut, or (run == 0) one whole pair
    Segment seg = {};
    bool more = false;
    const int stride = p.cluster ? p.cluster * kTile : kTile;      // from one of this block's tiles to the next
    int first_pages[R::kStages - 1];
    if (p.cluster) {                            // a pair per cluster, its tiles dealt to the cluster's blocks in turn
        const int place = blockIdx.x / p.cluster, rank = blockIdx.x - place * p.cluster;
        seg.b = place / pairs;
        seg.pair = place - seg.b * pairs;
        seg.tile = rank;
        // the first tiles' places do not depend on the length, so their pages are looked up together with it
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i) {
            const int key = rank * kTile + warp * kSub + i * stride;
            first_pages[i] = key < most ? __ldcg(table + (size_t)seg.b * p.table_stride + (key >> kv.page_shift)) : 0;
        }
        seg.len = seq_len(lens, seg.b, most);
        seg.tiles = seg.take = (seg.len + kTile - 1) / kTile;
        more = seg.len > 0;                     // the same for the whole cluster; a block without tiles joins with nothing
    } else if (locate(lens, p, pairs, most, &cut)) {
        left = cut.run ? min(cut.run, cut.total - blockIdx.x / p.lanes * cut.run) : units_of(cut.len);
        seg = {cut.b, cut.pair, cut.unit, 0, 0, cut.len};
    }
    bool first_segment = true;
    // Takes what this worker's run holds of the pair at seg.tile; false where that is only the unit behind its last tile.
    auto take = [&]() {
        seg.tiles = (seg.len + kTile - 1) / kTile;
        const int units = min((int)left, seg.tiles + kEnding - seg.tile);
        left -= units;
        seg.take = min(units, seg.tiles - seg.tile);
        return seg.take > 0;
    };
    // The next pair with something to take; false at the end of the run.
    auto next = [&]() {
        do {
            if (left == 0) return false;
            if ((seg.pair += p.lanes) >= pairs) {
                seg.pair = blockIdx.x % p.lanes;
                do seg.len = seq_len(lens, ++seg.b, most); while (seg.len == 0);
            }
            seg.tile = 0;
            first_segment = false;
        } while (!take());
        return true;
    };
    if (left > 0) more = take() || next();
    const unsigned run_end = min((blockIdx.x / p.lanes + 1) * cut.run, cut.total);
    auto record = [&](const Crossing& c) {
        *reinterpret_cast<uint4*>(Partials<kHeads, D>::crossing(ws, p.workers, blockIdx.x)) =
            make_uint4((unsigned)c.b, (unsigned)c.pair, c.slot, c.last);
    };
    if (!p.cluster && threadIdx.x == 0) record({0, 0, 0, blockIdx.x});

    uint8_t* ring = smem + warp * R::kRing;
    const uint32_t ring_u = smem_u32(ring);
    const int page_mask = (1 << kv.page_shift) - 1;
    int cur = 0, prev = R::kRing - R::kStage;   // byte offsets in the ring: the next stage to read, and the one before it
    unsigned bad = 0;                           // one bit per slot: its page lies outside the pool
    int k0, k1, head;                           // this warp's positions: k0 .. k0 + 15, then `stride` further, below k1
    // Where this lane reads and writes in a stage; a chunk or row further is an xor of chunk bits or a constant.
    const uint32_t k_lane = place<R::kRowBytes>(lane & 15, lane >> 4);
    const uint32_t v_lane = R::kRows + (kCoded ? place<R::kRowBytes>(2 * t, g * (D / 8) >> 4) + (g * (D / 8) & 15)
                                               : place<R::kRowBytes>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1));
    const uint32_t cp_lane = place<R::kRowBytes>(lane / R::kChunks, lane % R::kChunks);
    constexpr int kCpRows = 32 / R::kChunks;    // rows that a warp copies at once
    const int* pages;
    // this lane's first 16 bytes of the segment's head in page 0, of its scales (lanes 0..3: K, 4..7: V); a page further
    const uint8_t *seg_k, *seg_v;
    const float* seg_scale = nullptr;
    const unsigned page_rows = (unsigned)kv.heads << kv.page_shift;
    const size_t page_bytes = (size_t)page_rows * R::kRowBytes;
    int ahead = 0;                              // page of the next stage to request
    uint32_t qb[D / 16][2 * kHalves];
    float2 unit[kHalves];                       // score = product * unit (* scale of the key), heads 2 t and 2 t + 1 (+ 8)

    auto look = [&](int key) { return key < k1 ? __ldcg(pages + (key >> kv.page_shift)) : 0; };
    auto request = [&](int key, int slot, int from) {      // the 16 positions from `key` on, which lie in page `from`, into a slot
        if (key < k1) {
            const int real = k1 - key;
            const uint32_t dst = ring_u + slot;
            const bool ok = (unsigned)from < (unsigned)kv.pages;
            if (!ok) {
                bad |= 1u << (slot / R::kStage);
                *status = KAIROS_ERR_ARG;
            }
            const unsigned page = ok ? (unsigned)from : 0u, in_page = (unsigned)(key & page_mask);
            const size_t off = (size_t)page * page_bytes + in_page * R::kRowBytes;
            const uint8_t* ks = seg_k + off;
            const uint8_t* vs = seg_v + off;
            if (ok && real >= kSub) {
#pragma unroll
                for (int n = 0; n < R::kChunks / 2; ++n) {
                    const uint32_t to = ((dst + cp_lane) ^ ((n * kCpRows & R::kSwizzle) << 4)) + n * kCpRows * R::kRowBytes;
                    cp16(to, ks + 512 * n);
                    cp16(to + R::kRows, vs + 512 * n);
                }
            } else {                            // rows behind the end, or of no page, are zeros: 0 * weight stays 0
#pragma unroll
                for (int n = 0; n < R::kChunks / 2; ++n) {
                    const uint32_t to = ((dst + cp_lane) ^ ((n * kCpRows & R::kSwizzle) << 4)) + n * kCpRows * R::kRowBytes;
                    const bool there = ok && n * kCpRows + lane / R::kChunks < real;
                    cp16(to, ks + 512 * n, there);
                    cp16(to + R::kRows, vs + 512 * n, there);
                }
            }
            if constexpr (kCoded) {             // lanes 0..3: scales of K, 4..7: of V
                if (lane < 8)
                    cp16(dst + 2 * R::kRows + (lane >> 2) * (kSub * 4) + (lane & 3) * 16, seg_scale + ((size_t)page * page_rows + in_page), ok);
            }
        }
        cp_commit();
    };
    // Puts a segment's first stages and its queries under way.
    auto start = [&](const Segment& sg) {
        head = sg.pair / p.blocks_per_kv;
        const int block = sg.pair - head * p.blocks_per_kv;
        const int rows = min(kHeads, p.group - block * kHeads);            // of 4 heads a block: the whole group
        k0 = sg.tile * kTile + warp * kSub;
        k1 = p.cluster ? sg.len : min((sg.tile + sg.take) * kTile, sg.len);
        pages = table + (size_t)sg.b * p.table_stride;
        const unsigned head_row = (unsigned)head << kv.page_shift;
        seg_k = static_cast<const uint8_t*>(kv.k) + (size_t)head_row * R::kRowBytes + lane * 16;
        seg_v = static_cast<const uint8_t*>(kv.v) + (size_t)head_row * R::kRowBytes + lane * 16;
        if constexpr (kCoded) seg_scale = (lane < 4 ? kv.ks : kv.vs) + head_row + (lane & 3) * 4;
        int slot = cur;
        if (!p.cluster) first_pages[0] = look(k0);
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i) {
            if (i + 1 == R::kStages - 1) ahead = look(k0 + (i + 1) * stride);
            else if (!p.cluster) first_pages[i + 1] = look(k0 + (i + 1) * stride);
            request(k0 + i * stride, slot, first_pages[i]);
            slot = slot == R::kRing - R::kStage ? 0 : slot + R::kStage;
        }
        // q as the second operand: head g (and g + 8).  For a coded cache the channels of a step are permuted as the code
        // words lie: a thread's four channels are 4 t .. 4 t + 3.
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {
            unit[r] = both(p.scale_log2);
            const int row = kTwin ? g & 3 : g + 8 * r;
            const bool real = row < rows;
            const QT* q = Q + (size_t)sg.b * p.qb + (size_t)(head * p.group + block * kHeads + (real ? row : 0)) * p.qh;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                uint32_t lo, hi;
                if constexpr (kCoded) {
                    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(q + 16 * s + 4 * t));
                    lo = w.x, hi = w.y;
                } else {
                    lo = __ldcg(reinterpret_cast<const unsigned*>(q + 16 * s + 2 * t));
                    hi = __ldcg(reinterpret_cast<const unsigned*>(q + 16 * s + 2 * t + 8));
                }
                qb[s][2 * r] = real ? lo : 0u;
                qb[s][2 * r + 1] = real ? hi : 0u;
            }
        }
    };
    // bf16 heads become fp16 by a power of two of their own: exact to 2^-38 of the head's largest value.
    auto settle = [&]() {
        if constexpr (kCoded && std::is_same<QT, __nv_bfloat16>::value) {
#pragma unroll
            for (int r = 0; r < kHalves; ++r) {
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w = qb[s][2 * r + e];
                        top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e2 = top > 0.f && top <= FLT_MAX ? max(-110, min(126, (int)(__float_as_uint(top) >> 23) - 127)) : 13;
                const float up = __uint_as_float((uint32_t)(127 + 13 - e2) << 23);
                const float back = p.scale_log2 * __uint_as_float((uint32_t)(127 - 13 + e2) << 23);
                unit[r] = make_float2(__shfl_sync(0xffffffffu, back, 8 * t), __shfl_sync(0xffffffffu, back, 8 * t + 4));
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t& w = qb[s][2 * r + e];
                        const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
                        w = *reinterpret_cast<const uint32_t*>(&h);
                    }
            }
        }
    };

    if (more) start(seg);
    // sequences without positions have no tile: their rows are written here, while the first stages are on their way
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        const int n = __ldcg(lens + b);
        if (n > most && threadIdx.x == 0) *status = KAIROS_ERR_ARG;
        if (min(n, most) > 0) continue;
        for (int i = threadIdx.x; i < p.H * D / 8; i += 128)
            reinterpret_cast<uint4*>(O + (size_t)b * p.H * D)[i] = make_uint4(0, 0, 0, 0);
        if (LSE)
            for (int i = threadIdx.x; i < p.H; i += 128) LSE[(size_t)b * p.H + i] = -INFINITY;
    }
    while (more) {
        settle();
        // o[j][r]: channels 16 j + g and + 8 (coded: g * D / 8 + 2 j and + 1) of heads 2 t, 2 t + 1 (+ 8 r)
        float o[D / 16][kHalves][4] = {};
        // l and o are sums of weights 2^(s + back); heads 2 t and 2 t + 1.  Coded: the power of two that products are kept times,
        // at first 2^126
        float2 back[kHalves], l[kHalves], shift[kHalves];
#pragma unroll
        for (int r = 0; r < kHalves; ++r) back[r] = both(-kUnset), l[r] = both(0.f), shift[r] = both(8.507059173023462e37f);

#pragma unroll 1
        for (int pos = k0; pos < k1; pos += stride) {
            cp_wait<R::kStages - 2>();
            __syncwarp();                       // every lane's copies have landed; the stage before has been read
            request(pos + (R::kStages - 1) * stride, prev, ahead);
            ahead = look(pos + R::kStages * stride);
            const uint32_t ku = ring_u + cur + k_lane, vu = ring_u + cur + v_lane;
            const float* scales = reinterpret_cast<const float*>(ring + cur + 2 * R::kRows);
            const int real = k1 - pos;
            const bool full = real >= kSub && bad == 0;         // the same in all lanes
            bool gone = false;                                  // the page lies outside the pool
            if (!full) {
                const int slot = cur / R::kStage;
                gone = (bad >> slot) & 1u;
                bad &= ~(1u << slot);
            }
            prev = cur;
            cur = cur == R::kRing - R::kStage ? 0 : cur + R::kStage;

            // scores^T: positions g and g + 8, heads 2 t and 2 t + 1: [0], [1] and [2], [3]
            float s[kHalves][4] = {};
#pragma unroll
            for (int c = 0; c < D / 16; c += kCoded ? 2 : 1) {
                uint32_t w[4];                  // uncoded: one step of 16 channels; coded: two
                ldsm4(ku ^ ((kCoded ? c : 2 * c) << 4), w);
                if constexpr (!kCoded) {
#pragma unroll
                    for (int r = 0; r < kHalves; ++r) mma(MT(), s[r], w[0], w[1], w[2], w[3], qb[c][2 * r], qb[c][2 * r + 1]);
                } else {
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        uint32_t a[4];
                        Widen::run(w[2 * d], &a[0], &a[2]);
                        Widen::run(w[2 * d + 1], &a[1], &a[3]);
#pragma unroll
                        for (int r = 0; r < kHalves; ++r)
                            mma(MT(), s[r], a[0], a[1], a[2], a[3], qb[c + d][2 * r], qb[c + d][2 * r + 1]);
                    }
                }
            }
            // positions g, g + 8 (k): the scale of V; where there is no position, 0 and a score of -inf.  Scores are in units of
            // log2 e, rounded to fp32 before the reference is taken off: a score of any size less itself is 0, where the exact
            // product less its rounding can be any number once scores pass 2^27.
            float2 x[kHalves][2];
            float vs[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if constexpr (kCoded) vs[k] = scales[kSub + 8 * k + g];
#pragma unroll
                for (int r = 0; r < kHalves; ++r) {
                    x[r][k] = make_float2(s[r][2 * k], s[r][2 * k + 1]);
                    if constexpr (kCoded) x[r][k] = mul2(x[r][k], both(scales[8 * k + g]));
                    x[r][k] = mul2(x[r][k], unit[r]);
                }
            }
            if (!full) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (8 * k + g >= real || gone) {
                        vs[k] = 0.f;            // scales behind the end may be anything, NaN too
#pragma unroll
                        for (int r = 0; r < kHalves; ++r) x[r][k] = both(-INFINITY);
                    }
            }
            float2 w[kHalves][2], wv[kHalves][2];           // weights, and what enters the second product
            auto weights = [&]() {
#pragma unroll
                for (int r = 0; r < kHalves; ++r)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 y = add2(x[r][k], back[r]);
                        w[r][k] = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                        wv[r][k] = kCoded ? mul2(w[r][k], both(vs[k])) : w[r][k];
                    }
            };
            auto shifted = [&](int r, int k) { return kCoded ? mul2(wv[r][k], shift[r]) : wv[r][k]; };
            weights();
            bool move = false;
#pragma unroll
            for (int r = 0; r < kHalves; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    move |= w[r][k].x > kMost || w[r][k].y > kMost;
                    if constexpr (kCoded) {
                        const float2 v = shifted(r, k);
                        move |= fabsf(v.x) > kOver || fabsf(v.y) > kOver;
                    }
                }
            if (__any_sync(0xffffffffu, move)) {
                float keep[kHalves][2];
                auto top_of = [](float a, float b) {        // over the positions of the stage
                    float top = fmaxf(a, b);
#pragma unroll
                    for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
                    return top;
                };
                // a new reference for a head that needs one; what the sums before are multiplied by
                auto refer = [](float top, float& back) {
                    if (!(top + back > kLift + kSlack)) return 1.f;
                    float to = top - kLift;
                    if (top - to > kLift + kSlack) to = top;            // where fp32 no longer resolves kLift
                    const float keep = exp2_fast(-back - to);
                    back = -to;
                    return keep;
                };
#pragma unroll
                for (int r = 0; r < kHalves; ++r) {
                    keep[r][0] = refer(top_of(x[r][0].x, x[r][1].x), back[r].x);
                    keep[r][1] = refer(top_of(x[r][0].y, x[r][1].y), back[r].y);
                    l[r] = mul2(l[r], make_float2(keep[r][0], keep[r][1]));
                }
                weights();
                if constexpr (kCoded) {
                    auto raise = [](float top, float& keep, float& shift) {
                        // never above the largest product so far, as the new reference leaves it
                        const float was = inverse_pow2(shift);
                        top = fmaxf(top, was * (float)(1 << kLargest) * keep);
                        const int exponent = max(-118, min(126, (int)(__float_as_uint(top) >> 23) - 127));
                        shift = __uint_as_float((uint32_t)(127 + kLargest - exponent) << 23);
                        keep = keep * shift * was;
                    };
#pragma unroll
                    for (int r = 0; r < kHalves; ++r) {
                        raise(top_of(fabsf(wv[r][0].x), fabsf(wv[r][1].x)), keep[r][0], shift[r].x);
                        raise(top_of(fabsf(wv[r][0].y), fabsf(wv[r][1].y)), keep[r][1], shift[r].y);
                    }
                }
#pragma unroll
                for (int r = 0; r < kHalves; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) o[j][r][e] *= keep[r][e], o[j][r][e + 2] *= keep[r][e];
            }
            // the second operand of o^T += V^T w^T: positions 2 t, 2 t + 1 (and 8 further) of head g
            uint32_t wb[kHalves][2], rest[kHalves][2];
#pragma unroll
            for (int r = 0; r < kHalves; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    l[r] = add2(l[r], w[r][k]);
                    const float2 v = shifted(r, k);
                    uint32_t hi, lo;
                    split(MT(), v.x, v.y, &hi, &lo);
                    if constexpr (kTwin) {
                        wb[r][k] = transpose8(t < 2 ? hi : lo);
                    } else {
                        wb[r][k] = transpose8(hi);
                        rest[r][k] = transpose8(lo);
                    }
                }
            auto weigh = [&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int r = 0; r < kHalves; ++r) {
                    mma(MT(), o[j][r], a0, a1, a2, a3, wb[r][0], wb[r][1]);
                    if constexpr (!kTwin) mma(MT(), o[j][r], a0, a1, a2, a3, rest[r][0], rest[r][1]);
                }
            };
            if constexpr (!kCoded) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    uint32_t w[4];
                    ldsm4t(vu ^ (2 * j << 4), w);
                    weigh(j, w[0], w[1], w[2], w[3]);
                }
            } else {
                // a thread's bytes of a row are the D / 8 channels from g * D / 8 on
                constexpr int kWords = D / 32 < 4 ? D / 32 : 4;        // words per access: 2 (8 bytes) or 4 (16 bytes)
#pragma unroll
                for (int c = 0; c < D / 8 / (4 * kWords); ++c) {
                    uint32_t v[4][kWords];
#pragma unroll
                    for (int k = 0; k < 4; ++k)            // positions 2 t, 2 t + 1, and 8 further
                        lds(v[k], (vu ^ ((c ^ (k & 1 & R::kSwizzle)) << 4)) + ((k & 1) + 8 * (k >> 1)) * R::kRowBytes);
#pragma unroll
                    for (int w = 0; w < kWords; ++w)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            uint32_t a0, a1, a2, a3;
                            Widen::run(__byte_perm(v[0][w], v[1][w], d ? 0x7362 : 0x5140), &a0, &a1);
                            Widen::run(__byte_perm(v[2][w], v[3][w], d ? 0x7362 : 0x5140), &a2, &a3);
                            weigh((c * kWords + w) * 2 + d, a0, a1, a2, a3);
                        }
                }
            }
        }

        // ---- the next segment's first stages are requested before this one's parts are joined ----------------
        const Segment done = seg;
        const bool first = first_segment;
        __syncwarp();                           // every lane has read the last stage
        more = next();
        // the one slot that start() leaves alone
        const uint32_t free_slot = more && !R::kWaits ? prev : R::kLastOut;
        if (more && !R::kWaits) start(seg);

        // ---- the four warps' parts become one: each leaves its rows in a slot of its ring.  Column c of row r lies at
        // c ^ 8 (r / 2 % 4): the lanes of a store fall on different banks
        auto at = [](int r, int c) { return r * D + (c ^ (((r >> 1) & 3) << 3)); };
        float* mine = reinterpret_cast<float*>(ring + free_slot);
        if (lane == 0) jslot[warp] = warp * R::kRing + free_slot;
#pragma unroll
        for (int r = 0; r < kHalves; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * r + 2 * t + e;
                float sum = e ? l[r].y : l[r].x;
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                if (g == 0) jm[warp][row] = e ? -back[r].y : -back[r].x, jl[warp][row] = sum;
                if constexpr (kCoded) {
                    const float down = inverse_pow2(e ? shift[r].y : shift[r].x);
#pragma unroll
                    for (int j = 0; j < D / 16; j += 2)
                        *reinterpret_cast<float4*>(mine + at(row, g * (D / 8) + 2 * j)) =
                            make_float4(o[j][r][e] * down, o[j][r][e + 2] * down, o[j + 1][r][e] * down, o[j + 1][r][e + 2] * down);
                } else {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        mine[at(row, 16 * j + g)] = o[j][r][e];
                        mine[at(row, 16 * j + 8 + g)] = o[j][r][e + 2];
                    }
                }
            }
        __syncthreads();
        const int dhead = done.pair / p.blocks_per_kv, dblock = done.pair - dhead * p.blocks_per_kv;
        const int q0 = dhead * p.group + dblock * kHeads, rows = min(kHeads, p.group - dblock * kHeads);
        const bool whole = done.take == done.tiles;
        const unsigned part = 2 * blockIdx.x + (first ? 0 : 1);
        if (!p.cluster && !whole && done.tile == 0 && threadIdx.x == 0)      // begins here and lies across the run's end
            record({done.b, done.pair, part, (run_end - done.take + done.tiles - 1) / cut.run * p.lanes + blockIdx.x % p.lanes});
        for (int i = threadIdx.x; i < rows * (D / 4); i += 128) {
            const int row = i / (D / 4), c = 4 * (i - row * (D / 4));
            float top = kUnset;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, jm[w][row]);
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2_fast(jm[w][row] - top);
                const float* from = reinterpret_cast<const float*>(smem + jslot[w]);
                float4 v = *reinterpret_cast<const float4*>(from + at(row, c));
                if constexpr (kTwin) {          // what the remainders gave
                    const float4 u = *reinterpret_cast<const float4*>(from + at(row + 4, c));
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                }
                sum = __fmaf_rn(f, jl[w][row], sum);
                acc.x = __fmaf_rn(f, v.x, acc.x);
                acc.y = __fmaf_rn(f, v.y, acc.y);
                acc.z = __fmaf_rn(f, v.z, acc.z);
                acc.w = __fmaf_rn(f, v.w, acc.w);
            }
            if (p.cluster > 1) {                // over warp 0's rows: nobody else reads this place
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(smem + R::kLastOut) + at(row, c)) = acc;
                if (c == 0) jpart[row] = make_float2(top, sum);
            } else if (whole) {
                const float inv = inverse_sum(sum);
                const size_t to = (size_t)done.b * p.H + q0 + row;
                put4(O + to * D + c, acc, inv);
                if (LSE && c == 0) LSE[to] = (top + log2f(sum)) * kLn2;
            } else {
                *reinterpret_cast<float4*>(Partials<kHeads, D>::o(ws, part) + row * D + c) = acc;
                if (c == 0) *reinterpret_cast<float2*>(Partials<kHeads, D>::ml(ws, part) + 2 * row) = make_float2(top, sum);
            }
        }
        if (p.cluster > 1) {
            // ---- the cluster's parts become one, read from its blocks' shared memory; each block forms its share of the
            // output, and none leaves before all have read
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            for (int i = threadIdx.x + 128 * (blockIdx.x % p.cluster); i < rows * (D / 4); i += 128 * p.cluster) {
                const int row = i / (D / 4), c = 4 * (i - row * (D / 4));
                float top = kUnset, sum = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                const uint32_t from_o = smem_u32(smem) + R::kLastOut + at(row, c) * 4, from_ml = smem_u32(&jpart[row]);
                for (int k = 0; k < p.cluster; ++k) top = fmaxf(top, ld_cluster2(cluster_map(from_ml, k)).x);
                for (int k = 0; k < p.cluster; ++k) {
                    const float2 ml = ld_cluster2(cluster_map(from_ml, k));
                    const float4 v = ld_cluster4(cluster_map(from_o, k));
                    const float f = exp2_fast(ml.x - top);
                    sum = __fmaf_rn(f, ml.y, sum);
                    acc.x = __fmaf_rn(f, v.x, acc.x);
                    acc.y = __fmaf_rn(f, v.y, acc.y);
                    acc.z = __fmaf_rn(f, v.z, acc.z);
                    acc.w = __fmaf_rn(f, v.w, acc.w);
                }
                const size_t to = (size_t)done.b * p.H + q0 + row;
                put4(O + to * D + c, acc, inverse_sum(sum));
                if (LSE && c == 0) LSE[to] = (top + log2f(sum)) * kLn2;
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
        }
        if (more) {
            __syncthreads();                    // the slots belong to the rings again
            if (R::kWaits) start(seg);
        }
    }
}

// Block (w, y): the pair, if any, that begins in worker w's run and lies across its end; a slice of 32 items (a head's four
// channels) of its partial results of workers w, w + lanes, ... .  The four warps share the parts, and the order in which
// parts are added depends on nothing but their number.
template <typename QT, int D, int kHeads>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(QT* __restrict__ O, float* __restrict__ LSE,
                                                                   float* __restrict__ ws, const AttnShape p) {
    using P = Partials<kHeads, D>;
    constexpr int kPer = 32 / kHeads, kAhead = 8;       // chunks of four channels in a slice; parts whose loads go together
    __shared__ float4 part_o[kWarps][32];
    __shared__ float2 part_ml[kWarps][32];
    chain_wait();
    chain_release();
    const uint4 record = __ldcg(reinterpret_cast<const uint4*>(P::crossing(ws, p.workers, blockIdx.x)));
    const unsigned last = record.w;
    if (last == blockIdx.x) return;
    const int b = (int)record.x, pair = (int)record.y, head = pair / p.blocks_per_kv, block = pair - head * p.blocks_per_kv;
    const int rows = min(kHeads, p.group - block * kHeads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane / kPer, c = 4 * (blockIdx.y * kPer + lane % kPer);
    float top = kUnset, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2 ml, const float4 v) {
        const float next = fmaxf(top, ml.x), keep = exp2_fast(top - next), f = exp2_fast(ml.x - next);
        top = next;
        sum = __fmaf_rn(sum, keep, f * ml.y);
        acc.x = __fmaf_rn(acc.x, keep, f * v.x);
        acc.y = __fmaf_rn(acc.y, keep, f * v.y);
        acc.z = __fmaf_rn(acc.z, keep, f * v.z);
        acc.w = __fmaf_rn(acc.w, keep, f * v.w);
    };
    if (row < rows) {
        const unsigned step = kWarps * p.lanes;
        for (unsigned w = blockIdx.x + warp * p.lanes; w <= last; w += kAhead * step) {
            float2 ml[kAhead];
            float4 v[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const unsigned u = w + a * step;
                if (u <= last) {
                    const unsigned slot = u == blockIdx.x ? record.z : 2 * u;
                    ml[a] = __ldcg(reinterpret_cast<const float2*>(P::ml(ws, slot) + 2 * row));
                    v[a] = __ldcg(reinterpret_cast<const float4*>(P::o(ws, slot) + row * D + c));
                }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (w + a * step <= last) add(ml[a], v[a]);
        }
    }
    part_o[warp][lane] = acc;
    part_ml[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp != 0 || row >= rows) return;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) add(part_ml[w][lane], part_o[w][lane]);
    const size_t at = (size_t)b * p.H + head * p.group + block * kHeads + row;
    put4(O + at * D + c, acc, inverse_sum(sum));
    if (LSE && c == 0) LSE[at] = (top + log2f(sum)) * kLn2;
}

// ---- host ---------------------------------------------------------------------------------------------------
static int sm_count() {
    static std::atomic<int> counts[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = counts[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        counts[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

struct Plan {
    int heads_per_block, blocks_per_kv, workers, lanes, cluster;
    size_t bytes;
};

static int make_plan(const KvView& kv, bool coded, int B, int H, int table_width, Plan* out) {
    const int sms = sm_count();
    if (sms <= 0) return note_cuda_error(cudaGetLastError());
    const int group = H / kv.heads;
    out->heads_per_block = group > 8 ? 16 : group > 4 ? 8 : 4;
    out->blocks_per_kv = (group + out->heads_per_block - 1) / out->heads_per_block;
    const bool wide = out->heads_per_block == 16;
#define KAIROS_PER_SM(D)                                                                       \
    (wide ? (coded ? Ring<D, true, 2>::kBlocksPerSm : Ring<D, false, 2>::kBlocksPerSm)         \
          : (coded ? Ring<D, true, 1>::kBlocksPerSm : Ring<D, false, 1>::kBlocksPerSm))
    const int per_sm = kv.dim == 64 ? KAIROS_PER_SM(64) : kv.dim == 128 ? KAIROS_PER_SM(128) : KAIROS_PER_SM(256);
#undef KAIROS_PER_SM
    const long long tiles = (((long long)table_width << kv.page_shift) + kTile - 1) / kTile;
    const long long pairs = (long long)B * kv.heads * out->blocks_per_kv;
    if ((tiles + kEnding) * pairs > 0x7fffffffLL) return KAIROS_ERR_SHAPE;
    const int full = sms * per_sm;
    // Where the table bounds every pair to a few tiles a block, clusters of one to eight blocks take one pair each and
    // meet in shared memory: one launch, no scan of the lengths, no workspace.  Otherwise the device cuts the work by the
    // lengths, which costs 2 to 4 us more but keeps every block busy whatever they are.  Up to four tiles go to one block, more
    // are shared by two tiles a block: 256 positions take 5.0 us in one block and 5.1 in four, 512 take 6.6 in one or two and
    // 5.6 in four.  A single block takes twenty at the most: in fp16, 32 sequences of 1280 positions take 28.3 us in blocks of
    // their own and 32.4 cut (20.7 and 22.7 with lengths from 1 to 1280, but one of 1280 and 31 of 160 14.7 and 11.1; of 1536:
    // 33.2 and 37.3, 23.9 and 25.0, 19.0 and 11.5).  In clusters sixteen (twelve where pairs are few): 16 of 2048 in clusters of
    // two 24.6 and 28.9 (19.0 and 19.6 with lengths from 128 on), but 16 of 256 to 4096 32.5 and 30.1 (43.4 and 48.0 where all
    // have 4096), one of 8192 in clusters of eight 15.5 and 12.6.
    int cluster = 1;
    while (cluster < 8 && pairs * cluster * 2 <= full && tiles > 4 && tiles > 2 * cluster) cluster *= 2;
    out->cluster = pairs * cluster <= full && (tiles + cluster - 1) / cluster <= (cluster == 1 ? 20 : pairs < 32 ? 12 : 16) ? cluster : 0;
    // With many more pairs than blocks fit, blocks of their own in several waves are balanced by their number and end a
    // pair without holding the next one up: 128 sequences of 1000 positions in int8 50.3 us and 58.4 cut, 128 of 2048 92.8
    // and 97.7 (fp16 84.8 and 85.4, 160.9 and 162.2), with 16 heads a kv head 64 of 1 to 1000 in int8 (512 pairs for 444
    // blocks) 29.6 and 38.7.  From some forty tiles on the last wave's tail costs more (64 sequences of 1 to 4000, fp16: 91.5
    // and 86.1), and just over one wave (320 pairs for 296 blocks of 16 tiles: 36.9 and 34.6) does too.
    if (cluster == 1 && 20 * pairs >= (tiles <= 16 ? 23 : 30) * (long long)full && tiles <= 40) out->cluster = 1;
    // The even cut: a lane per pair of a sequence where that leaves at most 3% of the blocks out, else one lane.
    const long long deep = (long long)kv.heads * out->blocks_per_kv;
    out->lanes = deep <= full && full / deep * deep * 100 >= 97LL * full ? (int)deep : 1;
    out->workers = (int)(out->cluster ? pairs * out->cluster
                                      : max(1LL, min((long long)full / out->lanes, (tiles + kEnding) * pairs / out->lanes)) * out->lanes);
    out->bytes = out->cluster ? 0 : (size_t)2 * out->workers * max(8, out->heads_per_block) * (kv.dim + 2) * 4 + (size_t)out->workers * sizeof(Crossing);
    return KAIROS_OK;
}

template <typename QT, typename Widen, int D, int kBlockHeads>
static int run_attention(const void* Q, const KvView& kv, const void* table, const void* lens, void* O, void* LSE, void* ws,
                         const AttnShape& p, const Plan& plan, int* status, cudaStream_t st) {
    constexpr int kHalves = (kBlockHeads + 7) / 8;
    using R = Ring<D, !std::is_void<Widen>::value, kHalves>;
    static PerDeviceFlag flag;
    auto kernel = paged_attention_kernel<QT, Widen, D, kBlockHeads>;
    const int rc = ensure_dynamic_smem(flag, kernel, R::kBytes);
    if (rc != KAIROS_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.workers);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = R::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    if (plan.cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = plan.cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (chained_launch_enabled()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = attr;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<const QT*>(Q), kv, static_cast<const int*>(table),
                                       static_cast<const int*>(lens), static_cast<QT*>(O), static_cast<float*>(LSE),
                                       static_cast<float*>(ws), p, status);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (!plan.cluster && plan.workers > plan.lanes) {
        constexpr int kSlices = D / 4 / (32 / (8 * kHalves));
        e = launch_chained(paged_attention_join_kernel<QT, D, 8 * kHalves>, dim3(plan.workers - plan.lanes, kSlices), dim3(128), 0, st,
                           static_cast<QT*>(O), static_cast<float*>(LSE), static_cast<float*>(ws), p);
        if (e != cudaSuccess) return note_cuda_error(e);
    }
    return launch_status();
}

template <typename QT, typename Widen>
static int pick_attention(const void* Q, const KvView& kv, const void* table, const void* lens, void* O, void* LSE, void* ws,
                          const AttnShape& p, const Plan& plan, int* status, cudaStream_t st) {
#define KAIROS_ATTN(D)                                                                                                 \
    (plan.heads_per_block == 4 ? run_attention<QT, Widen, D, 4>(Q, kv, table, lens, O, LSE, ws, p, plan, status, st)   \
     : plan.heads_per_block == 8 ? run_attention<QT, Widen, D, 8>(Q, kv, table, lens, O, LSE, ws, p, plan, status, st) \
                                 : run_attention<QT, Widen, D, 16>(Q, kv, table, lens, O, LSE, ws, p, plan, status, st))
    return kv.dim == 64 ? KAIROS_ATTN(64) : kv.dim == 128 ? KAIROS_ATTN(128) : KAIROS_ATTN(256);
#undef KAIROS_ATTN
}

}  // namespace kairos

extern "C" size_t kairos_paged_attention_workspace_bytes(const kairos_kv_layer* layer, int B, int H, int table_width) {
    using namespace kairos;
    KvView kv;
    Plan plan;
    if (kv_view(layer, &kv) != KAIROS_OK || B <= 0 || H <= 0 || H % kv.heads != 0 || table_width < 0) return 0;
    const bool coded = layer->dtype == KAIROS_DTYPE_I8 || layer->dtype == KAIROS_DTYPE_E4M3;
    return make_plan(kv, coded, B, H, table_width, &plan) == KAIROS_OK ? plan.bytes : 0;
}

extern "C" int kairos_paged_attention(const void* Q, long long q_b, long long q_h, const kairos_kv_layer* layer,
                                      const void* page_table, long long table_stride, int table_width, const void* lens,
                                      void* O, void* LSE, int B, int H, float scale, int dtype, void* workspace,
                                      size_t workspace_bytes, kairos_stream_t stream) {
    using namespace kairos;
    KvView kv;
    int rc = kv_view(layer, &kv);
    if (rc != KAIROS_OK) return rc;
    if (B < 0 || B > 65535 || H <= 0 || H % kv.heads != 0 || table_width < 0 || table_stride < 0 ||
        ((long long)table_width << kv.page_shift) > (1LL << 30))    // positions and those looked ahead for fit an int
        return KAIROS_ERR_SHAPE;
    const bool coded = layer->dtype == KAIROS_DTYPE_I8 || layer->dtype == KAIROS_DTYPE_E4M3;
    if ((dtype != KAIROS_DTYPE_F16 && dtype != KAIROS_DTYPE_BF16) || (!coded && layer->dtype != dtype)) {
        set_last_error("paged_attention: queries are fp16 or bf16, and a 16-bit cache has their type");
        return KAIROS_ERR_ARG;
    }
    if (q_b % 8 != 0 || q_h % 8 != 0) return KAIROS_ERR_ALIGN;
    if (B == 0) return KAIROS_OK;
    if (!Q || !O || !lens || (!page_table && table_width > 0) || ((uintptr_t)Q & 15) || ((uintptr_t)O & 15) ||
        ((uintptr_t)page_table & 3) || ((uintptr_t)lens & 3) || ((uintptr_t)LSE & 3))
        return KAIROS_ERR_ALIGN;
    Plan plan;
    if ((rc = make_plan(kv, coded, B, H, table_width, &plan)) != KAIROS_OK) return rc;
    if (workspace_bytes < plan.bytes || (plan.bytes && (!workspace || ((uintptr_t)workspace & 15)))) return KAIROS_ERR_WORKSPACE;
    int* status = device_status_word();
    if (!status) return KAIROS_ERR_CUDA;
    const AttnShape p = {q_b, q_h, table_stride, B, H, H / kv.heads, plan.blocks_per_kv, table_width,
                         plan.workers, plan.lanes, plan.cluster, scale * kLog2e};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == KAIROS_DTYPE_F16) {
        if (layer->dtype == KAIROS_DTYPE_I8) return pick_attention<__half, WidenI8>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
        if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_attention<__half, WidenE4M3>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
        return pick_attention<__half, void>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
    }
    if (layer->dtype == KAIROS_DTYPE_I8) return pick_attention<__nv_bfloat16, WidenI8>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
    if (layer->dtype == KAIROS_DTYPE_E4M3) return pick_attention<__nv_bfloat16, WidenE4M3>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
    return pick_attention<__nv_bfloat16, void>(Q, kv, page_table, lens, O, LSE, workspace, p, plan, status, st);
}
