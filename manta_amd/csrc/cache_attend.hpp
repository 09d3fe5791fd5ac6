// cache_attend.hpp -- what the attention kernels of the 8-bit cache share:
// matrix operands from codes, the rows of a tile, and the joining of results
// that several workgroups hold.  Device code only.
#pragma once

#include "cache_kernels.hpp"

namespace manta {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight codes as f16: a byte offset by 128 under 0x64 is 1024 + 128 + code,
// exactly, and so is the difference.
__device__ __forceinline__ half8 codes_f16(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const half2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    half2 p[4];
    p[0] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
    p[1] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
    p[2] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
    p[3] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
    return half8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}
// ... and as bf16: an f32 of a code is zero in its lower half.
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t a, uint32_t b) {
    asm("" : "+v"(a), "+v"(b));  // whole registers: the loads' bytes are not kept one a register
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t x = (i < 2 ? a : b) >> (16 * (i & 1));
        const float lo = (float)(int8_t)(x & 0xFF), hi = (float)(int8_t)((x >> 8) & 0xFF);
        r[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    }
    return __builtin_bit_cast(bf16x8, r);
}

// Operands of q k^T in the queries' type.
struct MmaF16 {
    typedef half8 V;
    static __device__ __forceinline__ V codes(uint32_t a, uint32_t b) { return codes_f16(a, b); }
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
struct MmaBf16 {
    typedef bf16x8 V;
    static __device__ __forceinline__ V codes(uint32_t a, uint32_t b) { return codes_bf16(a, b); }
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <class E>
struct MmaOf;
template <>
struct MmaOf<F16> {
    typedef MmaF16 M;
};
template <>
struct MmaOf<Bf16> {
    typedef MmaBf16 M;
};

// Over the lanes that differ in bit 5, and in bits 4 and 5.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ float finite_or_zero(float x) { return x < INFINITY ? x : 0.0f; }

// The rows of a tile (the same for every thread of the workgroup).
struct Tile {
    int row0;    // the sequence's first row in the activation tensors
    int count;   // its rows
    int r0, rows;  // the tile's first row among them, and how many (0: no tile)
    int seq, length;
    int begin, end;  // the keys that any of the rows sees
};
__device__ __forceinline__ int key_end(const AttendArgs& a, int length, int pos) {
    return a.causal ? max(0, min(length, pos + 1)) : length;
}
__device__ __forceinline__ int key_begin(const AttendArgs& a, int pos) {
    return a.window > 0 ? (int)max((int64_t)0, (int64_t)pos - a.window + 1) : 0;
}
__device__ __forceinline__ Tile my_tile(const CacheView& c, const RaggedRows& r, const AttendArgs& a, int64_t slot,
                                        int rows) {
    Tile t{};
    const int i = __builtin_amdgcn_readfirstlane(
        r.n == 1 ? 0 : find_slot(r.n, slot, [&](int j) {
            return tile_base(clamp_row(r.offsets[j], r.tokens), j, a.group, rows);
        }));
    t.row0 = clamp_row(r.offsets[i], r.tokens);
    t.count = clamp_row(r.offsets[i + 1], r.tokens) - t.row0;
    const int64_t r0 = (slot - tile_base(t.row0, i, a.group, rows)) * rows;
    if (t.count <= 0 || r0 < 0 || r0 >= (int64_t)t.count * a.group) return t;
    t.r0 = (int)r0;
    t.rows = (int)min((int64_t)rows, (int64_t)t.count * a.group - r0);
    t.seq = r.seqs ? r.seqs[i] : i;
    if ((unsigned)t.seq < (unsigned)c.seqs) t.length = c.clamp_length(c.lengths[t.seq]);
    else {
        if (threadIdx.x == 0) cache_report(c, kCacheBadSeq, t.seq, 0);
        t.seq = 0;  // length 0: none of its table is read
    }
    const int first = t.length - t.count + t.r0 / a.group;
    const int last = t.length - t.count + (t.r0 + t.rows - 1) / a.group;
    t.end = key_end(a, t.length, last);
    t.begin = key_begin(a, first);
    return t;
}

// Results of a tile's part of the keys, in global memory: [row][pitch + 4],
// the weighted mean of v, then the largest score and the sum of weights.
// Written with agent-scope stores, which the last workgroup's ticket follows.
__device__ __forceinline__ void part_store(float* at, float x) {
    __hip_atomic_store((uint32_t*)at, __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float part_load(const float* at) {
    return __uint_as_float(__hip_atomic_load((const uint32_t*)at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

}  // namespace manta
