// Rotary positions: what the stand-alone operator and the cache write share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace kairos {

// Eight consecutive elements of a row from fp32, rounded once, in one or two 16-byte accesses.
__device__ __forceinline__ void store8(__half* p, const float (&f)[8]) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// cos and sin of position * step, step being a binary fraction of a full turn (2^64 = one turn).  The product
// modulo 2^64 is the angle without any rounding but the step's own (2^-65 turns for each position).  Its upper 32 bits split into the nearest
// quarter turn and a signed rest of at most an eighth of a turn, whose sine and cosine are their Taylor series to x^9 and
// x^8: what is left out is below 1.8e-9 and 2.5e-8 at pi / 4, under the half step 3e-8 of fp32.  Dropping the lower
// 32 bits moves the angle by less than 1.5e-9.  A third of the instructions of a general sine and cosine, which has to
// reduce its argument first.
__device__ __forceinline__ void turn_of(long long position, unsigned long long step, float magnitude, float* c, float* s) {
    const unsigned a = (unsigned)(((unsigned long long)position * step) >> 32);
    const unsigned quarter = (a + 0x20000000u) >> 30;
    const float x = __int2float_rn((int)(a - (quarter << 30))) * 1.4629180792671596e-09f;    // 2 pi / 2^32
    const float x2 = x * x;
    float sn = __fmaf_rn(x2, 2.7557319e-06f, -1.9841270e-04f);
    sn = __fmaf_rn(x2, sn, 8.3333333e-03f);
    sn = __fmaf_rn(x2, sn, -1.6666667e-01f);
    sn = __fmaf_rn(x * x2, sn, x);
    float cs = __fmaf_rn(x2, 2.4801587e-05f, -1.3888889e-03f);
    cs = __fmaf_rn(x2, cs, 4.1666667e-02f);
    cs = __fmaf_rn(x2, cs, -0.5f);
    cs = __fmaf_rn(x2, cs, 1.f);
    const float co = quarter & 1u ? sn : cs, si = quarter & 1u ? cs : sn;
    *c = (quarter + 1u) & 2u ? -co * magnitude : co * magnitude;       // quarters 1 and 2
    *s = quarter & 2u ? -si * magnitude : si * magnitude;              // quarters 2 and 3
}

// Both members of a pair; sums and products in fp32.
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
    const float x = a;
    a = __fmaf_rn(x, c, -(b * s));
    b = __fmaf_rn(b, c, x * s);
}

// A row (one head of one token) moves as cells of 16 elements, two chunks of 8, one cell per thread.  In the half
// layout the two chunks of a rotating cell are partners rot / 2 apart; in the interleaved layout and behind `rot` they
// are neighbours.  Cell j of a row: its two element offsets, and the first of its eight pairs (-1: passes unchanged).
struct Cell {
    int first, second, pair;
};
__device__ __forceinline__ Cell cell_of(int j, int rot, int layout) {
    const int turning = rot >> 4;
    Cell c;
    if (layout == 0 && j < turning) {
        c.first = 8 * j;
        c.second = 8 * j + (rot >> 1);
    } else {
        c.first = 16 * j;
        c.second = 16 * j + 8;
    }
    c.pair = j < turning ? 8 * j : -1;
    return c;
}
// Where a token's table of `pairs` angles (a multiple of 8) holds a pair: the first four of every eight, then the other
// fours, so that neighbouring cells read neighbouring 16 bytes without bank conflicts (4099 x 28 fp32 heads 20.3 us against
// 20.9 in order).
__device__ __forceinline__ int table_place(int pair, int pairs) {
    return (pair & 4 ? pairs >> 1 : 0) + (pair >> 3) * 4 + (pair & 3);
}
// Turns the cell's eight pairs from `pair` on by a token's table cs / sn (fp32 cos and sin).
__device__ __forceinline__ void turn_cell(float (&a)[8], float (&b)[8], const float* cs, const float* sn, int pair, int pairs,
                                          int layout) {
    float c[8], s[8];
    const int low = pair >> 1, high = low + (pairs >> 1);
    *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cs + low);
    *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(cs + high);
    *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sn + low);
    *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(sn + high);
    if (layout == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn_pair(a[i], b[i], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            turn_pair(a[2 * i], a[2 * i + 1], c[i], s[i]);
            turn_pair(b[2 * i], b[2 * i + 1], c[4 + i], s[4 + i]);
        }
    }
}

// The 16 elements of a cell as they come from memory: a thread requests several cells before it turns the first.
template <typename T>
struct RawCell {
    static constexpr int kWords = 8 * (int)sizeof(T) / 16;     // 16-byte words of a chunk
    uint4 w[2][kWords];
    __device__ __forceinline__ void load(const T* row, const Cell& c) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            w[0][i] = __ldcg(reinterpret_cast<const uint4*>(row + c.first) + i);
            w[1][i] = __ldcg(reinterpret_cast<const uint4*>(row + c.second) + i);
        }
    }
    static __device__ __forceinline__ void widen(const uint4 (&x)[kWords], float (&f)[8]) {
        const uint32_t* v = reinterpret_cast<const uint32_t*>(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                f[2 * i] = __uint_as_float(v[2 * i]);
                f[2 * i + 1] = __uint_as_float(v[2 * i + 1]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(v + i));
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            } else {
                f[2 * i] = __uint_as_float(v[i] << 16);
                f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            }
        }
    }
};
// Cells that a thread has under way: 64 bytes of loads, which with 1024 threads on an SM keeps 64 KB of loads in flight.
// Twice as many with 512 or 768 threads measured 4 to 20% slower (16381 x 32 heads of 128 in bf16: 51 us against 47), half
// as many with 1536 threads 60%.
template <typename T>
constexpr int kCells = sizeof(T) == 4 ? 1 : 2;

constexpr int kTablePairs = 2048;   // pairs whose cos and sin a block keeps: 16 KB of shared memory
constexpr int kBlockTokens = 64;    // tokens of a block, at most

// i / d for i, d below 2^16 by one multiplication; `magic` = ceil(2^32 / d).
inline unsigned div_magic(int d) { return d == 1 ? 0u : (unsigned)((0x100000000ull + d - 1) / d); }
__device__ __forceinline__ int div_small(int i, unsigned magic) { return magic ? (int)__umulhi((unsigned)i, magic) : i; }

// Tokens and threads of a block.  Where every SM gets four of them or more: 128 threads and about `target` rows (heads of
// tokens) or up to twice as many, so that they fill whole batches (what the threads have under way together; `per_step`
// rows take 128 threads, `deep` of those a batch) best.  64 rows of 16-bit values, 32 of fp32 ones; 256 threads with twice
// the rows measured 5 to 9% slower (a block's barrier and its last stores hold up more loads), 1.5 times the rows the same.
// Else one token, so that a decode step spreads over the SMs, and 256 threads: 64 tokens of 48 heads 2.2 us against 2.7 with
// 128.  The angles of a block's tokens fit its table.
struct RowBlocks {
    int tokens, threads;
};
inline RowBlocks row_blocks(long long tokens, int rows, int rot, int per_step, int deep, int target) {
    if (tokens * rows < 4 * 148 * target) return {1, 256};
    const int batch = per_step * deep;
    const int most = min(kBlockTokens, rot ? kTablePairs / (rot / 2) : kBlockTokens);
    int best = 1;
    long long best_done = 0, best_room = 1;                 // rows of a block over the rows of its batches
    for (int tb = 1; tb <= most && (tb == 1 || tb * rows <= 2 * target); ++tb) {
        const long long done = (long long)tb * rows, room = (done + batch - 1) / batch * batch;
        if (8 * done < 7 * target && tb < most && (tb + 1) * rows <= 2 * target) continue;
        if (done * best_room > best_done * room) best = tb, best_done = done, best_room = room;
    }
    return {best, 128};
}

inline bool rotary_plan_ok(const kairos_rotary_plan* p, int D) {
    return p && p->rot >= 0 && p->rot <= D && (p->rot & 1) == 0 && (p->layout == 0 || p->layout == 1) &&
           (p->rot == 0 || (p->steps && ((uintptr_t)p->steps & 7) == 0));
}

}  // namespace kairos
