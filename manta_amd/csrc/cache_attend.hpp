// cache_attend.hpp -- what the attention kernels of the 8-bit cache share:
// matrix operands from codes, the rows of a tile, and the joining of results
// that several workgroups hold.  Device code only.
#pragma once

#include "cache_kernels.hpp"

namespace manta {

typedef float f32x2 __attribute__((ext_vector_type(2)));
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

// Weights of the second product.  A page's v is code * v_max / 127, so what a
// key adds to a row is weight * v_max: its operand is taken against the largest
// of those that the row sees.  With m the running maximum of the scores and D
// that of score - m + log2 v_max (both of the keys that the row sees),
//
//   p = exp2(score - m + x),  x = log2 v_max - D + lift,
//
// is at most 2^lift (as often as the maxima are kept), and is rounded to f16
// (half a step, 2^-11, as the operand of an f32 sum; codes are exact): zero
// where it is 2^(-25 - lift) of the largest, whatever the scales of the row's
// pages and of those it does not see.  The sum of the weights takes a block's p
// times exp2(-x).  A block's log2 v_max is never taken to be below D - kFar, so
// that this factor stays in f32's range: its p are zero in f16 either way.
constexpr float kFar = 60.0f;
// A product that is rounded before a sum takes it.
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}
// log2 v_max.  (0 and what is not finite: their p are replaced.)
__device__ __forceinline__ float lead_of(float v_max) {
    return __builtin_amdgcn_logf(fminf(fmaxf(v_max, 0x1p-126f), 0x1.fffffep127f));
}
enum BlockKind {
    kBlockUsual = 0,
    kBlockNone = 1,    // no such page: none of its keys is seen
    kBlockPoison = 2,  // v_max is not finite: NaN to the rows that see it
    kBlockEmpty = 3,   // v_max is 0: nothing to add
};
__device__ __forceinline__ BlockKind block_kind(bool bad, float v_max) {
    return bad ? kBlockNone : !(v_max < INFINITY) ? kBlockPoison : v_max < 0x1p-126f ? kBlockEmpty : kBlockUsual;
}
__device__ __forceinline__ float or_zero(float top) { return top == -INFINITY ? 0.0f : top; }
// What sums of p * code are of the row's values, over the sum of the weights: a
// product of two factors, each in f32's range.
struct Unit {
    float a, b;
    // D: less the lift
    __device__ __forceinline__ Unit(float D, float sum) {
        b = __builtin_amdgcn_exp2f(0.5f * D);
        a = b / (127.0f * sum);
    }
    __device__ __forceinline__ f32x4 operator()(f32x4 y) const { return y * a * b; }
};

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
    const Owner o = find_owner(c, r, slot, [&](int offset, int j) { return tile_base(offset, j, a.group, rows); });
    t.row0 = o.from;
    t.count = o.to - o.from;
    t.seq = o.seq;
    const int64_t r0 = (slot - tile_base(t.row0, o.i, a.group, rows)) * rows;
    if (t.count <= 0 || r0 < 0 || r0 >= (int64_t)t.count * a.group) return t;
    t.r0 = (int)r0;
    t.rows = (int)min((int64_t)rows, (int64_t)t.count * a.group - r0);
    if (o.length >= 0) {
        t.length = c.clamp_length(o.length);
    } else {
        if (threadIdx.x == 0) cache_report(c, kCacheBadSeq, t.seq, 0);
        t.seq = 0;  // length 0: none of its table is read
    }
    const int first = t.length - t.count + t.r0 / a.group;
    const int last = t.length - t.count + (t.r0 + t.rows - 1) / a.group;
    t.end = key_end(a, t.length, last);
    t.begin = key_begin(a, first);
    return t;
}

// What the workgroups of a tile leave for the last of them, in global memory.
// Agent scope (sc1): written through, and read past this die's caches; the
// ticket is taken after the stores are done.  Offsets are in bytes, and the
// buffer's size is checked by the access itself.
struct Parts {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ explicit Parts(const AttendArgs& a)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(a.partial, 0, (int)a.partial_bytes, 0x00020000)) {}
    static constexpr int kAgent = 16;
    __device__ __forceinline__ void store(int at, f32x4 x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rsrc, at, 0, kAgent);
    }
    __device__ __forceinline__ void store(int at, f32x2 x) const {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), rsrc, at, 0, kAgent);
    }
    __device__ __forceinline__ f32x4 load4(int at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, kAgent));
    }
    __device__ __forceinline__ f32x2 load2(int at) const {
        return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, kAgent));
    }
};

// The end of a tile's part: true in the last of its `parts` workgroups, which
// sees what all of them stored.  The ticket is zero again.
__device__ __forceinline__ bool last_part(uint32_t* ticket, int parts) {
    __shared__ int last;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(parts - 1);
        if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// Columns k .. k + 3 of a tile's row, and with the first of them its lse.
template <class T>
__device__ __forceinline__ void store_out(const AttendArgs& a, const Tile& t, int kv, int d, int row, int k, f32x4 y,
                                          float big, float sum) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int r = t.r0 + row, token = r / a.group, head = kv * a.group + r % a.group;
    const int pos = t.length - t.count + token;
    const bool none = key_begin(a, pos) >= key_end(a, t.length, pos);
    if (none) y = f32x4{0, 0, 0, 0};
    T* dst = (T*)a.out + (int64_t)(t.row0 + token) * a.o_token + (int64_t)head * a.o_head + k;
    const T4 z = {(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
    if (a.wide && k + 4 <= d) {
        *(T4*)dst = z;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (k + j < d) dst[j] = z[j];
    }
    if (a.lse && k == 0)
        a.lse[(int64_t)(t.row0 + token) * a.heads + head] =
            none ? -INFINITY : (big + __builtin_amdgcn_logf(sum)) * 0.693147180559945f;
}

// In a tile's last workgroup: its parts joined in their order, whichever
// workgroup came last, and stored.  so: 4 * THREADS floats, weight: MOST * RT.
template <class T, int RT, int D, int THREADS, int MOST, class At>
__device__ __forceinline__ void join_parts(const AttendArgs& a, const Tile& t, int kv, int d, const Parts& mem,
                                           At part_at, int parts, float* so, float* weight) {
    constexpr int OP = D + 4;
    __shared__ float top_m[RT], top_l[RT];
    {
        // the parts' weights, by PER threads a row
        constexpr int PER = THREADS / RT, EACH = MOST / PER;
        const int row = min((int)threadIdx.x / PER, t.rows - 1), j = threadIdx.x % PER;
        f32x2 e[EACH];
        float big = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int u = 0; u < EACH; u++)
            if (u * PER < parts) e[u] = mem.load2(part_at(min(j + u * PER, parts - 1)) + row * (OP * 4) + 4 * D);
#pragma unroll
        for (int u = 0; u < EACH; u++)
            if (u * PER < parts) big = fmaxf(big, e[u][0]);
#pragma unroll
        for (int x = 1; x < PER; x <<= 1) big = fmaxf(big, __shfl_xor(big, x));
        const float base = big == -INFINITY ? 0.0f : big;
#pragma unroll
        for (int u = 0; u < EACH; u++) {
            if (j + u * PER < parts) {
                e[u][1] *= __builtin_amdgcn_exp2f(e[u][0] - base);
                sum += e[u][1];
            }
        }
#pragma unroll
        for (int x = 1; x < PER; x <<= 1) sum += __shfl_xor(sum, x);
        // (at most 1: values near the largest number stay finite)
#pragma unroll
        for (int u = 0; u < EACH; u++)
            if (j + u * PER < parts) weight[(j + u * PER) * RT + row] = e[u][1] / sum;
        if (j == 0) {
            top_m[row] = big;
            top_l[row] = sum;
        }
    }
    __syncthreads();
    // 4 columns a thread; where those are few, several threads share one's parts
    const int items = t.rows * (D / 4);
    const int groups = items < THREADS ? min(THREADS / items, parts) : 1;
    const int group = groups > 1 ? (int)threadIdx.x / items : 0;
    const int s1 = parts * (group + 1) / groups;
    for (int i = groups > 1 ? (int)threadIdx.x % items : (int)threadIdx.x; i < items; i += THREADS) {
        const int row = i / (D / 4), k = 4 * (i % (D / 4));
        f32x4 y = {0, 0, 0, 0};
        constexpr int AHEAD = 16;
        if (group < groups) {
            for (int s0 = parts * group / groups; s0 < s1; s0 += AHEAD) {
                f32x4 e[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    if (s0 + u < s1) e[u] = mem.load4(part_at(s0 + u) + row * (OP * 4) + 4 * k);
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    if (s0 + u < s1) y += e[u] * weight[(s0 + u) * RT + row];
            }
        }
        if (groups == 1) store_out<T>(a, t, kv, d, row, k, y, top_m[row], top_l[row]);
        else if (group < groups) *(f32x4*)&so[4 * threadIdx.x] = y;
    }
    if (groups == 1) return;
    __syncthreads();
    if ((int)threadIdx.x < items) {
        const int row = threadIdx.x / (D / 4), k = 4 * (threadIdx.x % (D / 4));
        f32x4 y = {0, 0, 0, 0};
        for (int h = 0; h < groups; h++) y += *(const f32x4*)&so[4 * (h * items + threadIdx.x)];
        store_out<T>(a, t, kv, d, row, k, y, top_m[row], top_l[row]);
    }
}

}  // namespace manta
