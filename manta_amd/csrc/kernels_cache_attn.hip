// kernels_cache_attn.hip -- softmax(scale q k^T) v over the 8-bit cache.
//
// One pass over the keys with a running maximum and sum (f32).  A wave per
// query row and head; a lane per key in the products with k, a lane per
// column in those with v.
#include "cache_kernels.hpp"

namespace manta {

namespace {

// The sequence that owns `row`: the last i with offsets[i] <= row.
__device__ int row_sequence(const RaggedRows& r, int row) {
    int lo = 0, hi = r.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (r.offsets[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <class E>
__global__ __launch_bounds__(64) void attend_kernel(CacheView c, int64_t layer, RaggedRows r, AttendArgs a) {
    typedef typename E::T T;
    __shared__ float qs[kMaxHeadDim];
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    const int i = row_sequence(r, row);
    const int lo = r.offsets[i], hi = r.offsets[i + 1];
    if (row < lo || row >= hi) return;  // no sequence owns the row
    const int seq = r.seqs ? r.seqs[i] : i;
    int length = 0;
    if ((unsigned)seq < (unsigned)c.seqs) length = c.clamp_length(c.lengths[seq]);
    else if (lane == 0) cache_report(c, kCacheBadSeq, seq, 0);
    const int pos = length - (hi - lo) + (row - lo);
    const int end = a.causal ? min(length, pos + 1) : length;
    const int begin = a.window > 0 ? (int)max((int64_t)0, (int64_t)pos - a.window + 1) : 0;
    const int d = c.head_dim, kv = head / a.group;
    const T* q = (const T*)a.q + row * a.q_token + head * a.q_head;
    for (int k = lane; k < d; k += 64) qs[k] = E::load(q[k]);
    __syncthreads();
    const int32_t* table = c.tables + (int64_t)(length ? seq : 0) * c.table_pages;
    const int mask = c.page_tokens - 1;
    float m = -INFINITY, l = 0.0f, o[kMaxHeadDim / 64] = {};
    for (int t0 = begin & ~63; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        float s = -INFINITY, vs = 0.0f;
        int64_t at = 0;  // the head's codes in the token's page
        bool seen = t >= begin && t < end;
        if (seen) {
            const int page = table[t >> c.page_shift];
            if ((unsigned)page >= (unsigned)c.pages) {
                cache_report(c, kCacheBadPage, page, 0);
                seen = false;
            } else {
                const int64_t slab = c.slab(layer, page);
                at = slab * c.page_codes() + (int64_t)kv * c.page_tokens * c.pitch;
                const int8_t* k = c.k_codes + at + (t & mask) * c.pitch;
                float dot = 0.0f;
                for (int j = 0; j < d; j++) dot += qs[j] * (float)k[j];
                s = dot * (c.k_max[slab * c.kv_heads + kv] / 127.0f) * a.scale;
                vs = c.v_max[slab * c.kv_heads + kv] / 127.0f;
            }
        }
        float top = s;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float m2 = fmaxf(m, top);
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - m2);
        const float p = seen ? exp2f(s - m2) : 0.0f;
        const float pv = seen ? p * vs : 0.0f;
        float sum = p;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * keep + sum;
        m = m2;
        for (int k = 0; k < kMaxHeadDim / 64; k++) o[k] *= keep;
        for (int j = 0; j < 64; j++) {
            if (!__shfl((int)seen, j)) continue;
            const float pj = __shfl(pv, j);
            const int64_t aj = __shfl((long long)at, j);
            const int8_t* v = c.v_codes + aj + ((t0 + j) & mask);
            for (int k = 0; k < kMaxHeadDim / 64; k++)
                if (lane + 64 * k < d) o[k] += pj * (float)v[(lane + 64 * k) * c.page_tokens];
        }
    }
    T* out = (T*)a.out + row * a.o_token + head * a.o_head;
    const bool none = begin >= end || (m == -INFINITY && l == 0.0f);
    for (int k = 0; k < kMaxHeadDim / 64; k++)
        if (lane + 64 * k < d) out[lane + 64 * k] = E::store(none ? 0.0f : o[k] / l);
    if (a.lse && lane == 0)
        a.lse[(int64_t)row * a.heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
}

}  // namespace

hipError_t launch_cache_attention(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                                  hipStream_t s) {
    const dim3 grid(r.tokens, a.heads);
    if (a.dtype == MANTA_ROCM_F16) attend_kernel<F16><<<grid, 64, 0, s>>>(c, layer, r, a);
    else attend_kernel<Bf16><<<grid, 64, 0, s>>>(c, layer, r, a);
    return hipGetLastError();
}

}  // namespace manta
