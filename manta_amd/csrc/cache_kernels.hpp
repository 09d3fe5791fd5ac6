// cache_kernels.hpp -- host-side launchers of the rotary and cache kernels,
// and the element types they share (internal to libmanta_rocm.so; the public
// surface is include/manta_cache.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cache_layout.hpp"

namespace manta {

// ---- rotary ----
constexpr int kRotaryParts = 4;
struct RotaryPart {
    const void* x;
    void* out;
    int heads;
    int64_t x_token, x_head, out_token, out_head;
};
struct RotaryArgs {
    RotaryPart part[kRotaryParts];
    int parts, heads;      // tensors; heads of all of them
    const double* turns;   // [rot / 2] turns a token
    const int32_t* positions;
    int64_t tokens;
    int head_dim, rot, interleaved;
    float magnitude;
    int inverse;
    int dtype;
    int wide;  // every row starts on 16 bytes and splits into 16-byte pieces
};
hipError_t launch_rotary(const RotaryArgs& a, hipStream_t s);
struct RotaryNorms {
    const float* weight[kRotaryParts];  // [head_dim] each, or nullptr: not normed
    double eps, inv_dim;  // 1 / head_dim
    int past;  // write past the caches (the launcher's)
};
hipError_t launch_rotary_normed(const RotaryArgs& a, const RotaryNorms& n, hipStream_t s);

// ---- cache ----
struct RaggedRows {
    const int32_t* offsets;  // [n + 1]
    const int32_t* seqs;     // [n] or nullptr
    int n;
    int tokens;
};
struct KvRows {  // k and v [tokens, kv_heads, head_dim], in or out
    void* k;
    void* v;
    int64_t k_token, k_head, v_token, v_head;
    int dtype;
    int wide;  // every row starts on 16 bytes
};
hipError_t launch_cache_append(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s);
hipError_t launch_cache_read(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s);

// scratch of the page calls: pairs (from, to) to copy, their count first
struct PageScratch {
    int32_t* count;
    int32_t* from;
    int32_t* to;
    int32_t* remap;  // [pages]
};
hipError_t launch_cache_extend(const CacheView& c, const PageScratch& w, const int32_t* seqs, const int32_t* counts,
                               int n, int32_t* free_list, hipStream_t s);
hipError_t launch_cache_fork(const CacheView& c, const int32_t* parents, const int32_t* children,
                             const int32_t* tokens, int n, hipStream_t s);
hipError_t launch_cache_release(const CacheView& c, const int32_t* seqs, const int32_t* keep, int n, hipStream_t s);
hipError_t launch_cache_reorder(const CacheView& c, const int32_t* seqs, const int32_t* parents, int n, int group,
                                hipStream_t s);
hipError_t launch_cache_compact(const CacheView& c, const PageScratch& w, int32_t* live, hipStream_t s);
// copy pages from[i] -> to[i], i < *count (count in device memory) or n, and
// with remap [pages] replace the pages that the tables name
hipError_t launch_cache_copy(const CacheView& c, const int32_t* from, const int32_t* to, const int32_t* count, int n,
                             const int32_t* remap, hipStream_t s);

struct AttendArgs {
    const void* q;
    void* out;
    float* lse;
    int64_t q_token, q_head, o_token, o_head;
    int dtype;
    int heads, group;
    float scale;  // scale * log2 e / 127: of q . codes * k_max, in units of exp2
    int causal;
    int window;
    int longest;
    int wide;
    float* partial;  // what split tiles leave for their last workgroup
    int64_t partial_bytes;
    uint32_t* tickets;  // ntickets, zero between calls
    int64_t ntickets;
    int cus;
    // the launcher's plan
    int splits;  // workgroups that may share a tile's keys
    int rounds;  // steps over the keys that are worth a workgroup
};
hipError_t launch_attend_many(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                              hipStream_t s);
hipError_t launch_cache_attention(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                                  hipStream_t s);

#ifdef __HIP__
// ---- elements ----
struct F32 {
    typedef float T;
    static constexpr int kWide = 4;  // elements of 16 bytes
    static __device__ __forceinline__ float load(T x) { return x; }
    static __device__ __forceinline__ T store(float x) { return x; }
};
struct F16 {
    typedef _Float16 T;
    static constexpr int kWide = 8;
    static __device__ __forceinline__ float load(T x) { return (float)x; }
    static __device__ __forceinline__ T store(float x) { return (T)x; }
};
struct Bf16 {
    typedef __bf16 T;
    static constexpr int kWide = 8;
    static __device__ __forceinline__ float load(T x) {
        return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, x) << 16);
    }
    static __device__ __forceinline__ T store(float x) { return (T)x; }
};

__device__ __forceinline__ int clamp_row(int x, int tokens) { return x < 0 ? 0 : x > tokens ? tokens : x; }

// The sequence whose slots hold `slot`: the last i < n with base(i) <= slot.
// Every wave of the workgroup finds it, 64 candidates a step.
template <class Base>
__device__ __forceinline__ int find_slot(int n, int64_t slot, Base base) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;  // the answer lies in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const bool below = i < hi && base(i) <= slot;
        // (lane 0's candidate counts as below even where the bases do not ascend)
        const unsigned long long m = __ballot(below) | 1ull;
        const int last = 63 - __clzll(m);
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

struct Owner {  // the sequence that owns a workgroup's slot, as the device arrays have it
    int i, from, to;  // its place in the batch, its rows
    int seq, length;  // (length: -1 where seq is out of range)
};
template <class Base>
__device__ __forceinline__ Owner find_owner(const CacheView& c, const RaggedRows& r, int64_t slot, Base base) {
    Owner o;
    if (r.n <= 64) {
        // every sequence's offsets and length at once, the one wanted picked
        // from the lanes: one wait where a search, its result's offsets and
        // its length are three
        const int lane = threadIdx.x & 63, j = min(lane, r.n - 1);
        const int o0 = clamp_row(r.offsets[j], r.tokens), o1 = clamp_row(r.offsets[j + 1], r.tokens);
        const int seq = r.seqs ? r.seqs[j] : j;
        const int length = (unsigned)seq < (unsigned)c.seqs ? max(c.lengths[seq], 0) : -1;
        const unsigned long long m = __ballot(lane < r.n && base(o0, j) <= slot) | 1ull;
        o.i = 63 - __clzll(m);
        o.from = __builtin_amdgcn_readlane(o0, o.i);
        o.to = __builtin_amdgcn_readlane(o1, o.i);
        o.seq = __builtin_amdgcn_readlane(seq, o.i);
        o.length = __builtin_amdgcn_readlane(length, o.i);
    } else {
        o.i = __builtin_amdgcn_readfirstlane(
            find_slot(r.n, slot, [&](int j) { return base(clamp_row(r.offsets[j], r.tokens), j); }));
        o.from = clamp_row(r.offsets[o.i], r.tokens);
        o.to = clamp_row(r.offsets[o.i + 1], r.tokens);
        o.seq = r.seqs ? r.seqs[o.i] : o.i;
        o.length = (unsigned)o.seq < (unsigned)c.seqs ? max(c.lengths[o.seq], 0) : -1;
    }
    return o;
}

__device__ __forceinline__ void cache_report(const CacheView& c, int kind, int64_t a, int64_t b) {
    atomicMax(c.err, cache_error(kind, a, b));
    // (a plain store: atomics on host memory need what the link may not have)
    __hip_atomic_store(c.err_flag, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
#endif

}  // namespace manta
