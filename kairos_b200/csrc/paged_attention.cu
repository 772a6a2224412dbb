// Attention of one new token per sequence over a paged key-value cache (kairos_paged_attention).
//
// Mathematics.  Per query head, with s_j = scale * q.k_j in units of log2 e:  o = sum_j 2^(s_j - m) v_j / l,
// l = sum_j 2^(s_j - m), m = max_j s_j, in ONE pass over the cache: m, l and o are kept for the keys seen so far and
// multiplied by 2^(m_old - m_new) where the maximum moves.  Parts of a sequence are joined by the same rule.
//
// Bound.  Every cached byte is read once and meets 2 * group flops (group = query heads per kv head): below 16 flops
// a byte, so HBM sets the pace and everything here serves to keep loads in flight:
//   * a warp owns a ring of stages of 16 positions (K rows and V rows, 4 KB for 128 channels in fp16 each), filled by
//     16-byte cp.async; no block-wide barrier until a segment ends;
//   * the heads that share a kv head are the rows of warp-level tensor instructions (m16n8k16), so a key is read from
//     shared memory once for all of them.  tcgen05 has no use here: its smallest tile is 64 or 128 rows, 8 to 32 times the
//     heads there are, and the tensor work is a tenth of what mma.sync gives;
//   * the work is cut on the device: all (sequence, kv head) pairs laid end to end in tiles of 64 positions, every block
//     takes an equal run of tiles, whatever the lengths are.  A pair that lies across blocks leaves one partial result per
//     block in the workspace and a second kernel joins them, in the order of the blocks (no atomics: same bits every run).
//
// Precision.  Scores, maxima, sums and outputs are fp32.  The weights enter the second product as TWO 16-bit numbers
// (value and remainder), which costs nothing for up to eight heads: the remainders are the eight rows of the tile that
// would be empty.  Rounding weights to 16 bits alone would add an error as large as the output's own rounding.
#include <type_traits>

#include "paged_kv.cuh"

namespace kairos {

int* device_status_word();   // api.cu

constexpr int kWarps = 4;
constexpr int kSub = 16;                    // positions per warp stage
constexpr int kTile = kSub * kWarps;        // positions per scheduling tile
constexpr float kLift = 14.f;               // weights are kept times 2^14: fp16's smallest step is then 2^-38 of the largest weight
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnShape {
    long long qb, qh, table_stride;
    int B, H, group, blocks_per_kv;         // head blocks (of 8 or 16 query heads) per kv head
    int table_width, workers, min_tiles;
    float scale_log2;
};

// ---- the cut of the work --------------------------------------------------------------------------------
__device__ __forceinline__ int seq_len(const int* lens, int b, int most) { return max(0, min(__ldcg(lens + b), most)); }

struct Cut {
    unsigned total, run;                    // tiles of all pairs, tiles per worker
    int b, pair, tile;                      // where tile `x` lies: sequence, pair (kv head, head block) and tile of it
    int tiles;                              // tiles of that sequence
    unsigned pair_first;                    // flat index of that pair's first tile
};

// Block-wide (128 threads): scan of the sequences' tile counts, then the place of flat tile x (x < total).  `x` is
// computed from the totals by `at`.
template <typename At>
__device__ __forceinline__ bool locate(const int* lens, const AttnShape& p, int pairs, int most, At at, Cut* out) {
    __shared__ unsigned warp_sum[kWarps];
    __shared__ Cut found;
    const int tid = threadIdx.x, per = (p.B + 127) >> 7;
    const int first = tid * per, last = min(p.B, first + per);
    unsigned mine = 0;
    for (int b = first; b < last; ++b) mine += (unsigned)(seq_len(lens, b, most) + kTile - 1) / kTile;
    unsigned upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
        if ((tid & 31) >= o) upto += v;
    }
    if ((tid & 31) == 31) warp_sum[tid >> 5] = upto;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < (tid >> 5)) upto += warp_sum[w];
        total += warp_sum[w];
    }
    total *= pairs;
    const unsigned run = max((unsigned)p.min_tiles, (total + p.workers - 1) / p.workers);
    const unsigned x = at(run);
    if (x >= total) return false;           // the same for every thread
    unsigned before = upto - mine;
    if (x >= before * pairs && x < upto * pairs) {
        for (int b = first; b < last; ++b) {
            const unsigned n = (unsigned)(seq_len(lens, b, most) + kTile - 1) / kTile;
            if (x < (before + n) * pairs) {
                const unsigned rest = x - before * pairs;
                found = Cut{total, run, b, (int)(rest / n), (int)(rest % n), (int)n, before * pairs + rest / n * n};
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    *out = found;
    return true;
}

// Partial results: slot 2 w of worker w is the pair that its run begins in, slot 2 w + 1 the one that it ends in.
template <int R, int D>
struct Partials {
    static constexpr size_t kFloats = (size_t)R * (D + 2);
    static __device__ __forceinline__ float* o(float* ws, unsigned slot) { return ws + slot * kFloats; }
    static __device__ __forceinline__ float* ml(float* ws, unsigned slot) { return ws + slot * kFloats + R * D; }
};

// ---- instructions -------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
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

template <int ROWB, bool kCoded>
struct Ring {
    static constexpr int kRows = kSub * ROWB;
    static constexpr int kStage = 2 * kRows + (kCoded ? 2 * kSub * 4 : 0);
    // stages a warp: 24 KB and more in flight per warp, and two to four blocks of four warps on an SM
    static constexpr int kStages = ROWB >= 256 ? 3 : ROWB == 128 ? 4 : 6;
    static constexpr int kBytes = kWarps * kStages * kStage;
};

// QT: type of q and o; Widen: void for a cache of type QT, else how codes become fp16; kHalves: 1 (up to 8 query heads in
// a block) or 2 (16).
template <typename QT, typename Widen, int D, int kHalves>
struct Attn {
    static constexpr bool kCoded = !std::is_void<Widen>::value;
    using MT = typename std::conditional<kCoded, __half, QT>::type;
    static constexpr int kRowBytes = kCoded ? D : 2 * D;
    static constexpr int kChunks = kRowBytes / 16;
    using R = Ring<kRowBytes, kCoded>;
    static constexpr int kHeads = 8 * kHalves;
    static constexpr int kPadRow = D + 8;      // floats: rows of the joining buffer fall on different banks
    static constexpr int kJoin = kWarps * kHeads * (kPadRow + 2) * 4;
    static constexpr int kSmem = R::kBytes > kJoin ? R::kBytes : kJoin;
    static constexpr int kBlocksPerSm = kSmem > 112 * 1024 ? 1 : kSmem > 74 * 1024 ? 2 : kSmem > 54 * 1024 ? 3 : 4;
};

template <typename QT, typename Widen, int D, int kHalves>
__global__ void __launch_bounds__(128, (Attn<QT, Widen, D, kHalves>::kBlocksPerSm))
    paged_attention_kernel(const QT* __restrict__ Q, const KvView kv, const int* __restrict__ table, const int* __restrict__ lens,
                           QT* __restrict__ O, float* __restrict__ LSE, float* __restrict__ ws, const AttnShape p, int* status) {
    using A = Attn<QT, Widen, D, kHalves>;
    using MT = typename A::MT;
    using R = typename A::R;
    constexpr int kTilesN = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    chain_release();
    chain_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pairs = kv.heads * p.blocks_per_kv, most = p.table_width << kv.page_shift;
    // sequences without positions have no tile: their rows are written here
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        const int n = __ldcg(lens + b);
        if (n > most) *status = KAIROS_ERR_ARG;
        if (min(n, most) > 0) continue;
        for (int i = threadIdx.x; i < p.H * D / 8; i += 128)
            reinterpret_cast<uint4*>(O + (size_t)b * p.H * D)[i] = make_uint4(0, 0, 0, 0);
        if (LSE)
            for (int i = threadIdx.x; i < p.H; i += 128) LSE[(size_t)b * p.H + i] = -INFINITY;
    }
    Cut cut;
    if (!locate(lens, p, pairs, most, [](unsigned run) { return blockIdx.x * run; }, &cut)) return;
    const unsigned begin = blockIdx.x * cut.run, end = min(begin + cut.run, cut.total);
    int b = cut.b, pair = cut.pair, tile = cut.tile, len = seq_len(lens, b, most), tiles = cut.tiles;

    uint8_t* ring = smem + warp * (R::kStages * R::kStage);
    const uint32_t ring_u = smem_u32(ring);
    for (unsigned x = begin; x < end;) {
        const int take = min((int)(end - x), tiles - tile);
        const int head = pair / p.blocks_per_kv, block = pair - head * p.blocks_per_kv;
        const int q0 = head * p.group + block * A::kHeads;                     // first query head of the block
        const int rows = min(A::kHeads, p.group - block * A::kHeads);
        const int k0 = tile * kTile + warp * kSub, k1 = min((tile + take) * kTile, len);   // this warp: k0, k0 + 64, ...
        const int count = k0 < k1 ? (k1 - k0 + kTile - 1) / kTile : 0;
        const int* pages = table + (size_t)b * p.table_stride;
        unsigned bad = 0;                                                      // one bit per stage: page outside the pool

        auto page_of = [&](int i) { return i < count ? __ldcg(pages + ((k0 + i * kTile) >> kv.page_shift)) : 0; };
        auto issue = [&](int i, int page) {
            if (i < count) {
                const int key = k0 + i * kTile, real = min(kSub, k1 - key);
                const int st = i % R::kStages;
                const bool ok = (unsigned)page < (unsigned)kv.pages;
                bad = (bad & ~(1u << st)) | ((ok ? 0u : 1u) << st);
                if (!ok) *status = KAIROS_ERR_ARG;
                const size_t row = ((((size_t)(ok ? page : 0)) * kv.heads + head) << kv.page_shift) + (key & ((1 << kv.page_shift) - 1));
                const uint8_t* ks = static_cast<const uint8_t*>(kv.k) + row * A::kRowBytes;
                const uint8_t* vs = static_cast<const uint8_t*>(kv.v) + row * A::kRowBytes;
                const uint32_t dst = ring_u + st * R::kStage;
#pragma unroll
                for (int n = 0; n < A::kChunks / 2; ++n) {
                    const int c = lane + 32 * n, r = c / A::kChunks;
                    cp16(dst + place<A::kRowBytes>(r, c % A::kChunks), ks + c * 16, ok && r < real);
                }
#pragma unroll
                for (int n = 0; n < A::kChunks / 2; ++n) {
                    const int c = lane + 32 * n, r = c / A::kChunks;
                    cp16(dst + R::kRows + place<A::kRowBytes>(r, c % A::kChunks), vs + c * 16, ok && r < real);
                }
                if constexpr (A::kCoded) {      // lanes 0..3: scales of K, 4..7: of V
                    if (lane < 8) cp16(dst + 2 * R::kRows + lane * 16, (lane < 4 ? kv.ks : kv.vs) + row + (lane & 3) * 4, ok);
                }
            }
            cp_commit();
        };

        int ahead = page_of(0);
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i) {
            const int page = ahead;
            ahead = page_of(i + 1);
            issue(i, page);
        }

        // q as the first operand: rows g (and g + 8) of the block.  For a coded cache the channels of a step are permuted
        // as the code words lie: a thread's four channels are 4 t .. 4 t + 3.
        uint32_t qa[D / 16][2 * kHalves];
        float unit[kHalves];                   // score = product * unit (* scale of the key)
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {
            unit[r] = p.scale_log2;
            const bool real = g + 8 * r < rows;
            const QT* q = Q + (size_t)b * p.qb + (size_t)(q0 + (real ? g + 8 * r : 0)) * p.qh;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                uint32_t lo, hi;
                if constexpr (A::kCoded) {
                    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(q + 16 * s + 4 * t));
                    lo = w.x, hi = w.y;
                } else {
                    lo = __ldcg(reinterpret_cast<const unsigned*>(q + 16 * s + 2 * t));
                    hi = __ldcg(reinterpret_cast<const unsigned*>(q + 16 * s + 2 * t + 8));
                }
                qa[s][r] = real ? lo : 0u;
                qa[s][kHalves + r] = real ? hi : 0u;
            }
            if constexpr (A::kCoded && std::is_same<QT, __nv_bfloat16>::value) {
                // bf16 rows become fp16 by a power of two of their own: exact to 2^-38 of the row's largest value
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w = qa[s][e * kHalves + r];
                        top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e2 = top > 0.f && top <= 3e38f ? max(-110, min(126, (int)(__float_as_uint(top) >> 23) - 127)) : 13;
                const float up = __uint_as_float((uint32_t)(127 + 13 - e2) << 23);
                unit[r] = p.scale_log2 * __uint_as_float((uint32_t)(127 - 13 + e2) << 23);
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t& w = qa[s][e * kHalves + r];
                        const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
                        w = *reinterpret_cast<const uint32_t*>(&h);
                    }
            }
        }

        float o[kTilesN][4] = {};
        float m[kHalves], l[kHalves], vtop = 7.888609052210118e-31f;           // 2^-100
#pragma unroll
        for (int r = 0; r < kHalves; ++r) m[r] = -INFINITY, l[r] = 0.f;

#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            cp_wait<R::kStages - 2>();
            __syncwarp();                       // every lane's copies have landed; the stage before has been read
            {
                const int page = ahead;
                ahead = page_of(i + R::kStages);
                issue(i + R::kStages - 1, page);
            }
            const int st = i % R::kStages;
            const uint32_t ku = ring_u + st * R::kStage, vu = ku + R::kRows;
            const uint8_t* stage = ring + st * R::kStage;
            const int real = (bad >> st) & 1u ? 0 : min(kSub, k1 - (k0 + i * kTile));

            // scores of 16 positions: columns 2 t, 2 t + 1 of two 8-wide tiles
            float s[2][4] = {};
            if constexpr (!A::kCoded) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t w[4];
                    ldsm4(ku + place<A::kRowBytes>((lane & 7) + ((lane >> 4) << 3), 2 * c + ((lane >> 3) & 1)), w);
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        mma(MT(), s[n], qa[c][0], kHalves == 2 ? qa[c][1] : 0u, qa[c][kHalves], kHalves == 2 ? qa[c][3] : 0u,
                            w[2 * n], w[2 * n + 1]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 16; c += 2) {
                    uint32_t w[4];              // two steps of 16 channels x two tiles of 8 positions
                    ldsm4(ku + place<A::kRowBytes>((lane & 7) + (((lane >> 3) & 1) << 3), c + (lane >> 4)), w);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            uint32_t b0, b1;
                            Widen::run(w[2 * h + n], &b0, &b1);
                            mma(MT(), s[n], qa[c + h][0], kHalves == 2 ? qa[c + h][1] : 0u, qa[c + h][kHalves],
                                kHalves == 2 ? qa[c + h][3] : 0u, b0, b1);
                        }
                }
            }
            float vs[2][2];                     // scale of V over the largest scale so far
            float grow = 1.f;
            float ks[2][2];
            if constexpr (A::kCoded) {
                const float* sc = reinterpret_cast<const float*>(stage + 2 * R::kRows);
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float2 k2 = *reinterpret_cast<const float2*>(sc + 8 * n + 2 * t);
                    const float2 v2 = *reinterpret_cast<const float2*>(sc + kSub + 8 * n + 2 * t);
                    ks[n][0] = k2.x, ks[n][1] = k2.y, vs[n][0] = v2.x, vs[n][1] = v2.y;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (8 * n + 2 * t + e >= real) vs[n][e] = 0.f;         // may be anything, NaN too
                        top = fmaxf(top, fabsf(vs[n][e]));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (top > vtop) {               // the same in all lanes
                    grow = __fdividef(vtop, top);
                    vtop = top;
                }
                const float inv = __frcp_rn(vtop);
#pragma unroll
                for (int n = 0; n < 2; ++n) vs[n][0] *= inv, vs[n][1] *= inv;
            }
            uint32_t pa[2][2 * kHalves];        // [tile][half]: weights, [tile][kHalves + half]: their remainders
            float keep[kHalves];
            bool moved = grow != 1.f;
#pragma unroll
            for (int r = 0; r < kHalves; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = s[n][2 * r + e] * unit[r];
                        if constexpr (A::kCoded) v *= ks[n][e];
                        v = 8 * n + 2 * t + e < real ? v : -INFINITY;
                        s[n][2 * r + e] = v;
                        top = fmaxf(top, v);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, m[r]);
                const float safe = top == -INFINITY ? 0.f : top;
                keep[r] = exp2_fast(m[r] - safe);
                moved |= top != m[r];
                m[r] = top;
                float w[2][2];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) w[n][e] = exp2_fast(s[n][2 * r + e] - safe + kLift);
                l[r] = __fmaf_rn(l[r], keep[r], (w[0][0] + w[0][1]) + (w[1][0] + w[1][1]));
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if constexpr (A::kCoded) w[n][0] *= vs[n][0], w[n][1] *= vs[n][1];
                    split(MT(), w[n][0], w[n][1], &pa[n][r], &pa[n][kHalves + r]);
                }
            }
            if (__any_sync(0xffffffffu, moved)) {
                const float f0 = keep[0] * grow, f1 = (kHalves == 2 ? keep[kHalves - 1] : keep[0]) * grow;
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
            }
            // o += weights . V.  kHalves == 1: rows 8..15 are the remainders of rows 0..7; 2: a second product
            auto weigh = [&](float (&acc)[4], uint32_t b0, uint32_t b1) {
                if constexpr (kHalves == 1) {
                    mma(MT(), acc, pa[0][0], pa[0][1], pa[1][0], pa[1][1], b0, b1);
                } else {
                    mma(MT(), acc, pa[0][0], pa[0][1], pa[1][0], pa[1][1], b0, b1);
                    mma(MT(), acc, pa[0][2], pa[0][3], pa[1][2], pa[1][3], b0, b1);
                }
            };
            if constexpr (!A::kCoded) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t w[4];
                    ldsm4t(vu + place<A::kRowBytes>(lane & 15, 2 * c + (lane >> 4)), w);
                    weigh(o[2 * c], w[0], w[1]);
                    weigh(o[2 * c + 1], w[2], w[3]);
                }
            } else {
                // column n of tile j is channel n * D / 8 + j: a thread's bytes of a row are D / 8 neighbours
                constexpr int kWords = D / 32 < 4 ? D / 32 : 4;        // words per access: 2 (8 bytes) or 4 (16 bytes)
#pragma unroll
                for (int c = 0; c < D / 8 / (4 * kWords); ++c) {
                    uint32_t x[4][kWords];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = 2 * t + (k & 1) + ((k >> 1) << 3), byte = g * (D / 8) + c * 16;
                        const uint8_t* from = stage + R::kRows + place<A::kRowBytes>(key, byte >> 4) + (byte & 15);
                        if constexpr (kWords == 4) *reinterpret_cast<uint4*>(x[k]) = *reinterpret_cast<const uint4*>(from);
                        else *reinterpret_cast<uint2*>(x[k]) = *reinterpret_cast<const uint2*>(from);
                    }
#pragma unroll
                    for (int w = 0; w < kWords; ++w) {
                        uint32_t lo[4], hi[4];                          // tiles 4 w .. 4 w + 3: positions 2 t, 2 t + 1 and 8 further
                        Widen::run(__byte_perm(x[0][w], x[1][w], 0x5140), &lo[0], &lo[1]);
                        Widen::run(__byte_perm(x[0][w], x[1][w], 0x7362), &lo[2], &lo[3]);
                        Widen::run(__byte_perm(x[2][w], x[3][w], 0x5140), &hi[0], &hi[1]);
                        Widen::run(__byte_perm(x[2][w], x[3][w], 0x7362), &hi[2], &hi[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) weigh(o[(c * kWords + w) * 4 + e], lo[e], hi[e]);
                    }
                }
            }
        }
        cp_wait<0>();

        // ---- the four warps' parts of the segment become one ------------------------------------------------
        __syncthreads();                        // all rings are read
        float* jo = reinterpret_cast<float*>(smem);                            // [warp][head][kPadRow]
        float* jm = jo + kWarps * A::kHeads * A::kPadRow;                      // [warp][head] maximum, then sum
        float* jl = jm + kWarps * A::kHeads;
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int row = warp * A::kHeads + g + 8 * r;
            if (t == 0) jm[row] = m[r], jl[row] = l[r];
            float* to = jo + row * A::kPadRow;
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) {
                float x = o[j][2 * r], y = o[j][2 * r + 1];
                if constexpr (kHalves == 1) x += o[j][2], y += o[j][3];
                if constexpr (A::kCoded) {
                    to[2 * t * (D / 8) + j] = x * vtop;
                    to[(2 * t + 1) * (D / 8) + j] = y * vtop;
                } else {
                    *reinterpret_cast<float2*>(to + 8 * j + 2 * t) = make_float2(x, y);
                }
            }
        }
        __syncthreads();
        const bool whole = take == tiles;
        const unsigned slot = 2 * blockIdx.x + (x == begin ? 0 : 1);
        for (int i = threadIdx.x; i < rows * (D / 4); i += 128) {
            const int row = i / (D / 4), c = i - row * (D / 4);
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, jm[w * A::kHeads + row]);
            const float safe = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2_fast(jm[w * A::kHeads + row] - safe);
                const float4 v = *reinterpret_cast<const float4*>(jo + (w * A::kHeads + row) * A::kPadRow + 4 * c);
                sum = __fmaf_rn(f, jl[w * A::kHeads + row], sum);
                acc.x = __fmaf_rn(f, v.x, acc.x);
                acc.y = __fmaf_rn(f, v.y, acc.y);
                acc.z = __fmaf_rn(f, v.z, acc.z);
                acc.w = __fmaf_rn(f, v.w, acc.w);
            }
            if (whole) {
                const float inv = __fdiv_rn(1.f, sum);
                const size_t at = (size_t)b * p.H + q0 + row;
                QT* to = O + at * D + 4 * c;
                put(to, acc.x * inv);
                put(to + 1, acc.y * inv);
                put(to + 2, acc.z * inv);
                put(to + 3, acc.w * inv);
                if (LSE && c == 0) LSE[at] = (top + __log2f(sum) - kLift) * kLn2;
            } else {
                *reinterpret_cast<float4*>(Partials<A::kHeads, D>::o(ws, slot) + row * D + 4 * c) = acc;
                if (c == 0) *reinterpret_cast<float2*>(Partials<A::kHeads, D>::ml(ws, slot) + 2 * row) = make_float2(top, sum);
            }
        }
        __syncthreads();                        // the buffer is a ring again

        x += take;
        tile = 0;
        if (x < end && ++pair == pairs) {
            pair = 0;
            do len = seq_len(lens, ++b, most); while (len == 0);
            tiles = (len + kTile - 1) / kTile;
        }
    }
}

// Block w looks at the boundary between the runs of workers w and w + 1.  Where a pair lies across it and no earlier
// boundary, its partial results (workers w, w + 1, ... up to the one that holds its last tile) are joined here; the
// channels are spread over gridDim.y.
template <typename QT, int D, int kHeads>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(const KvView kv, const int* __restrict__ lens, QT* __restrict__ O,
                                                                   float* __restrict__ LSE, float* __restrict__ ws,
                                                                   const AttnShape p) {
    using P = Partials<kHeads, D>;
    chain_release();
    chain_wait();
    const int pairs = kv.heads * p.blocks_per_kv;
    Cut cut;
    if (!locate(lens, p, pairs, p.table_width << kv.page_shift, [](unsigned run) { return (blockIdx.x + 1) * run; }, &cut)) return;
    const unsigned x = (blockIdx.x + 1) * cut.run, first = cut.pair_first;
    if (first >= x || first < x - cut.run) return;      // a pair begins here, or lay across an earlier boundary already
    const unsigned last = (first + cut.tiles - 1) / cut.run;
    const int head = cut.pair / p.blocks_per_kv, block = cut.pair - head * p.blocks_per_kv;
    const int rows = min(kHeads, p.group - block * kHeads);
    const int per = D / 4 / gridDim.y;                  // chunks of four channels of a row in this block
    for (int i = threadIdx.x; i < rows * per; i += 128) {
        const int row = i / per, c = i - row * per + blockIdx.y * per;
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (unsigned w = blockIdx.x; w <= last; ++w) {
            const unsigned slot = 2 * w + (w == blockIdx.x && first > w * cut.run ? 1 : 0);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(P::ml(ws, slot) + 2 * row));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(P::o(ws, slot) + row * D + 4 * c));
            const float next = fmaxf(top, ml.x), safe = next == -INFINITY ? 0.f : next;
            const float keep = exp2_fast(top - safe), f = exp2_fast(ml.x - safe);
            top = next;
            sum = __fmaf_rn(sum, keep, f * ml.y);
            acc.x = __fmaf_rn(acc.x, keep, f * v.x);
            acc.y = __fmaf_rn(acc.y, keep, f * v.y);
            acc.z = __fmaf_rn(acc.z, keep, f * v.z);
            acc.w = __fmaf_rn(acc.w, keep, f * v.w);
        }
        const float inv = __fdiv_rn(1.f, sum);
        const size_t at = (size_t)cut.b * p.H + head * p.group + block * kHeads + row;
        QT* to = O + at * D + 4 * c;
        put(to, acc.x * inv);
        put(to + 1, acc.y * inv);
        put(to + 2, acc.z * inv);
        put(to + 3, acc.w * inv);
        if (LSE && c == 0) LSE[at] = (top + __log2f(sum) - kLift) * kLn2;
    }
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
    int heads_per_block, blocks_per_kv, workers;
    long long most_tiles;      // were every sequence as long as the table allows
    bool joins;
    size_t bytes;
};

// Blocks per SM of the variant that serves (cache type, head dim, head block): what its shared memory leaves room for.
static int blocks_per_sm(const KvView& kv, bool coded, int heads) {
    const bool wide = heads == 16;
#define KAIROS_OCC(D) \
    (coded ? (wide ? Attn<__half, WidenI8, D, 2>::kBlocksPerSm : Attn<__half, WidenI8, D, 1>::kBlocksPerSm) \
           : (wide ? Attn<__half, void, D, 2>::kBlocksPerSm : Attn<__half, void, D, 1>::kBlocksPerSm))
    return kv.dim == 64 ? KAIROS_OCC(64) : kv.dim == 128 ? KAIROS_OCC(128) : KAIROS_OCC(256);
#undef KAIROS_OCC
}

static int make_plan(const KvView& kv, bool coded, int B, int H, int table_width, Plan* out) {
    const int sms = sm_count();
    if (sms <= 0) return note_cuda_error(cudaGetLastError());
    const int group = H / kv.heads;
    out->heads_per_block = group > 8 ? 16 : 8;
    out->blocks_per_kv = (group + out->heads_per_block - 1) / out->heads_per_block;
    const long long per_pair = (((long long)table_width << kv.page_shift) + kTile - 1) / kTile;
    out->most_tiles = per_pair * B * kv.heads * out->blocks_per_kv;
    if (out->most_tiles > 0x7fffffffLL) return KAIROS_ERR_SHAPE;
    const int full = sms * blocks_per_sm(kv, coded, out->heads_per_block);
    out->workers = (int)max(1LL, min((long long)full, out->most_tiles));
    out->joins = per_pair > 1 && out->workers > 1;
    out->bytes = out->joins ? (size_t)2 * out->workers * out->heads_per_block * (kv.dim + 2) * 4 : 0;
    return KAIROS_OK;
}

template <typename QT, typename Widen, int D, int kHalves>
static int run_attention(const void* Q, const KvView& kv, const void* table, const void* lens, void* O, void* LSE, void* ws,
                         const AttnShape& p, const Plan& plan, int* status, cudaStream_t st) {
    using A = Attn<QT, Widen, D, kHalves>;
    static PerDeviceFlag flag;
    auto kernel = paged_attention_kernel<QT, Widen, D, kHalves>;
    const int rc = ensure_dynamic_smem(flag, kernel, A::kSmem);
    if (rc != KAIROS_OK) return rc;
    cudaError_t e = launch_chained(kernel, dim3(plan.workers), dim3(128), A::kSmem, st, static_cast<const QT*>(Q), kv,
                                   static_cast<const int*>(table), static_cast<const int*>(lens), static_cast<QT*>(O),
                                   static_cast<float*>(LSE), static_cast<float*>(ws), p, status);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (plan.joins) {
        // few pairs: few joins of many parts each, so the channels of one are spread over several blocks
        const int slices = (long long)p.B * kv.heads * p.blocks_per_kv < 64 ? 4 : 1;
        e = launch_chained(paged_attention_join_kernel<QT, D, A::kHeads>, dim3(plan.workers - 1, slices), dim3(128), 0, st, kv,
                           static_cast<const int*>(lens), static_cast<QT*>(O), static_cast<float*>(LSE), static_cast<float*>(ws), p);
        if (e != cudaSuccess) return note_cuda_error(e);
    }
    return launch_status();
}

template <typename QT, typename Widen>
static int pick_attention(const void* Q, const KvView& kv, const void* table, const void* lens, void* O, void* LSE, void* ws,
                          const AttnShape& p, const Plan& plan, int* status, cudaStream_t st) {
#define KAIROS_ATTN(D)                                                                                              \
    (plan.heads_per_block == 8 ? run_attention<QT, Widen, D, 1>(Q, kv, table, lens, O, LSE, ws, p, plan, status, st) \
                               : run_attention<QT, Widen, D, 2>(Q, kv, table, lens, O, LSE, ws, p, plan, status, st))
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

extern "C" int kairos_paged_attention(const void* Q, const long long* q_strides, const kairos_kv_layer* layer,
                                      const void* page_table, long long table_stride, int table_width, const void* lens,
                                      void* O, void* LSE, int B, int H, float scale, int dtype, void* workspace,
                                      size_t workspace_bytes, kairos_stream_t stream) {
    using namespace kairos;
    KvView kv;
    int rc = kv_view(layer, &kv);
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
    Plan plan;
    if ((rc = make_plan(kv, coded, B, H, table_width, &plan)) != KAIROS_OK) return rc;
    if (workspace_bytes < plan.bytes || (plan.bytes && (!workspace || ((uintptr_t)workspace & 15)))) return KAIROS_ERR_WORKSPACE;
    int* status = device_status_word();
    if (!status) return KAIROS_ERR_CUDA;
    const AttnShape p = {q_strides[0], q_strides[1], table_stride, B, H, H / kv.heads, plan.blocks_per_kv, table_width,
                         plan.workers, 2, scale * kLog2e};
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
