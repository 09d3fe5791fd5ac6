// kernels_cache.hip -- contents and pages of the 8-bit key/value cache.
//
// Append and read move a page's head at a time; the page calls work on the
// book (refs, lengths, tables) in device memory, so a decoding loop never
// waits for the host.  The layout and the mapping of ragged batches are in
// cache_layout.hpp.
#include "cache_kernels.hpp"

#pragma clang fp contract(off)

namespace manta {

namespace {

constexpr int kThreads = 256;

// This workgroup's piece of the ragged batch and its page: false if there is
// none.
__device__ bool my_piece(const CacheView& c, const RaggedRows& r, Piece* p, int* page) {
    const int64_t slot = blockIdx.x;
    const int i = find_slot(
        r.n, slot, [&](int j) { return ragged_base(clamp_row(r.offsets[j], r.tokens), j, c.page_shift); });
    const int a = clamp_row(r.offsets[i], r.tokens), b = clamp_row(r.offsets[i + 1], r.tokens);
    const int seq = r.seqs ? r.seqs[i] : i;
    if ((unsigned)seq >= (unsigned)c.seqs) {
        if (threadIdx.x == 0) cache_report(c, kCacheBadSeq, seq, 0);
        return false;
    }
    const int length = c.clamp_length(c.lengths[seq]);
    if (!ragged_piece(a, b, length, slot - ragged_base(a, i, c.page_shift), c.page_shift, p)) return false;
    *page = c.tables[(int64_t)seq * c.table_pages + p->index];
    if ((unsigned)*page >= (unsigned)c.pages) {
        if (threadIdx.x == 0) cache_report(c, kCacheBadPage, *page, 0);
        return false;
    }
    return true;
}

__device__ __forceinline__ int quantise(float x, float max) {
    const float r = __builtin_rintf(__fdiv_rn(x * 127.0f, max));
    return (int)fminf(127.0f, fmaxf(-127.0f, r));
}
__device__ __forceinline__ int requantise(int code, float old, float max) {
    return (int)__builtin_rintf(__fdiv_rn((float)code * old, max));
}

// One page's head of k (blockIdx.z 0) or v (1).
template <class E>
__global__ __launch_bounds__(kThreads) void append_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    Piece p;
    int page;
    if (!my_piece(c, r, &p, &page)) return;
    const int head = blockIdx.y, is_v = blockIdx.z;
    const int tid = threadIdx.x, d = c.head_dim;
    const T* src = is_v ? (const T*)x.v + head * x.v_head : (const T*)x.k + head * x.k_head;
    const int64_t stride = is_v ? x.v_token : x.k_token;
    const int count = p.to - p.from;

    // the largest magnitude, as ordered bits: NaN above infinity above numbers
    uint32_t top = 0;
    for (int e = tid; e < count * d; e += kThreads) {
        const int t = e / d, col = e % d;
        top = max(top, __float_as_uint(E::load(src[(p.row + t) * stride + col])) & 0x7FFFFFFFu);
    }
    __shared__ uint32_t tops[kThreads / 64];
    for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; w++) top = max(top, tops[w]);

    float* slot = (is_v ? c.v_max : c.k_max) + c.slab(layer, page) * c.kv_heads + head;
    const float old = p.from ? *slot : 0.0f;
    const bool bad = top >= 0x7F800000u || old != old;
    float big = fmaxf(__uint_as_float(top), old);
    const bool zero = bad || big < 0x1p-126f;  // every code 0
    const bool raise = big > old;
    if (zero) big = bad ? __builtin_nanf("") : 0.0f;
    __syncthreads();  // every thread has read *slot
    if (tid == 0) *slot = big;

    const int64_t base = c.slab(layer, page) * c.page_codes() + (int64_t)head * c.page_tokens * c.pitch;
    if (!is_v) {
        int8_t* codes = c.k_codes + base;
        if (p.from && (raise || zero))
            for (int e = tid; e < p.from * c.pitch; e += kThreads)
                codes[e] = zero ? 0 : (int8_t)requantise(codes[e], old, big);
        for (int e = tid; e < count * c.pitch; e += kThreads) {
            const int t = e / c.pitch, col = e % c.pitch;
            int q = 0;
            if (!zero && col < d) q = quantise(E::load(src[(p.row + t) * stride + col]), big);
            codes[(p.from + t) * c.pitch + col] = (int8_t)q;
        }
        return;
    }
    int8_t* codes = c.v_codes + base;
    if (p.from && (raise || zero))
        for (int e = tid; e < p.from * c.pitch; e += kThreads) {
            int8_t* at = codes + (e / p.from) * c.page_tokens + e % p.from;
            *at = zero ? 0 : (int8_t)requantise(*at, old, big);
        }
    for (int e = tid; e < count * c.pitch; e += kThreads) {
        const int t = e / c.pitch, col = e % c.pitch;
        int q = 0;
        if (!zero && col < d) q = quantise(E::load(src[(p.row + t) * stride + col]), big);
        codes[col * c.page_tokens + p.from + t] = (int8_t)q;
    }
}

template <class E>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    Piece p;
    int page;
    if (!my_piece(c, r, &p, &page)) return;
    const int head = blockIdx.y, is_v = blockIdx.z, d = c.head_dim;
    T* dst = is_v ? (T*)x.v + head * x.v_head : (T*)x.k + head * x.k_head;
    const int64_t stride = is_v ? x.v_token : x.k_token;
    const float big = ((is_v ? c.v_max : c.k_max) + c.slab(layer, page) * c.kv_heads)[head];
    const int8_t* codes = (is_v ? c.v_codes : c.k_codes) + c.slab(layer, page) * c.page_codes() +
                          (int64_t)head * c.page_tokens * c.pitch;
    for (int e = threadIdx.x; e < (p.to - p.from) * d; e += kThreads) {
        const int t = e / d, col = e % d;
        const int code = is_v ? codes[col * c.page_tokens + p.from + t] : codes[(p.from + t) * c.pitch + col];
        dst[(p.row + t) * stride + col] = E::store(__fdiv_rn((float)code * big, 127.0f));
    }
}

// ------------------------------------------------------------------ pages

constexpr int kBook = 1024;  // threads of the kernels that walk the book

// Sum over the workgroup's threads below this one; *total: over all of them.
__device__ int block_scan(int x, int* total) {
    __shared__ int sums[kBook / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = x;
    for (int s = 1; s < 64; s <<= 1) {
        const int y = __shfl_up(incl, s);
        if (lane >= s) incl += y;
    }
    __syncthreads();  // an earlier call's sums have been read
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int below = 0, all = 0;
    for (int w = 0; w < kBook / 64; w++) {
        if (w < wave) below += sums[w];
        all += sums[w];
    }
    *total = all;
    return below + incl - x;
}

struct Growth {
    int seq, length, pages, more;  // its pages now, and new ones (a copy not counted)
    int last;                      // the page to copy first, or -1
    bool ok;
};
__device__ Growth growth(const CacheView& c, const int32_t* seqs, const int32_t* counts, int i, bool report) {
    Growth g{0, 0, 0, 0, -1, false};
    g.seq = seqs[i];
    const int add = counts[i];
    if ((unsigned)g.seq >= (unsigned)c.seqs) {
        if (report) cache_report(c, kCacheBadSeq, g.seq, 0);
        return g;
    }
    g.length = c.clamp_length(c.lengths[g.seq]);
    if (add < 0 || (int64_t)g.length + add > (int64_t)c.table_pages << c.page_shift) {
        if (report) cache_report(c, kCacheBadCount, g.seq, add);
        return g;
    }
    const int mask = c.page_tokens - 1;
    g.pages = (int)(((int64_t)g.length + mask) >> c.page_shift);
    g.more = (int)(((int64_t)g.length + add + mask) >> c.page_shift) - g.pages;
    if (add > 0 && (g.length & mask)) {
        const int last = c.tables[(int64_t)g.seq * c.table_pages + g.pages - 1];
        if ((unsigned)last >= (unsigned)c.pages) {
            if (report) cache_report(c, kCacheBadPage, last, 0);
            return g;
        }
        if (c.refs[last] > 1) g.last = last;
    }
    g.ok = true;
    return g;
}

// One workgroup: what every sequence needs, the lowest free pages, and then
// the tables.  An entry that is out of range, or too few pages: nothing changes.
__global__ __launch_bounds__(kBook) void extend_kernel(CacheView c, PageScratch w, const int32_t* seqs,
                                                       const int32_t* counts, int n, int32_t* free_list) {
    const int tid = threadIdx.x;
    __shared__ int wrong;
    if (tid == 0) wrong = 0;
    __syncthreads();
    int64_t need64 = 0;
    for (int i0 = 0; i0 < n; i0 += kBook) {
        int need = 0;
        if (i0 + tid < n) {
            const Growth g = growth(c, seqs, counts, i0 + tid, true);
            if (!g.ok) wrong = 1;
            need = g.more + (g.last >= 0);
        }
        int total;
        block_scan(need, &total);
        need64 += total;
    }
    __syncthreads();
    const bool skip = wrong != 0;
    int found = 0;
    const int need = (int)min(need64, (int64_t)c.pages + 1);
    for (int64_t p0 = 0; p0 < c.pages && found < need && !skip; p0 += kBook) {
        const bool is_free = p0 + tid < c.pages && c.refs[p0 + tid] == 0;
        int total;
        const int at = found + block_scan(is_free, &total);
        if (is_free && at < need) free_list[at] = (int)p0 + tid;
        found += total;
    }
    if (skip || found < need) {
        if (tid == 0) {
            if (!skip) cache_report(c, kCacheFull, need64, found);
            *w.count = 0;
        }
        return;
    }
    __syncthreads();  // free_list is written
    int taken = 0, copies = 0;
    for (int i0 = 0; i0 < n; i0 += kBook) {
        Growth g{0, 0, 0, 0, -1, false};
        if (i0 + tid < n) g = growth(c, seqs, counts, i0 + tid, false);
        const int mine = g.more + (g.last >= 0);
        int total, copied;
        int at = taken + block_scan(mine, &total);
        const int copy = copies + block_scan(g.last >= 0, &copied);
        taken += total;
        copies += copied;
        __syncthreads();  // every growth() of this step has read the book
        // (a list that names a sequence twice could ask for more than was counted)
        if (g.ok && at >= 0 && at + mine <= need && copy < need) {
            int32_t* row = c.tables + (int64_t)g.seq * c.table_pages;
            if (g.last >= 0) {
                const int page = free_list[at++];
                w.from[copy] = g.last;
                w.to[copy] = page;
                row[g.pages - 1] = page;
                c.refs[page] = 1;
            }
            for (int k = 0; k < g.more; k++) {
                const int page = free_list[at++];
                row[g.pages + k] = page;
                c.refs[page] = 1;
            }
        }
    }
    // shared pages lose a reference, and lengths grow, once no growth() can
    // see it: whether a page was shared is asked of the book as it was
    __syncthreads();
    if (tid == 0) *w.count = copies;
    for (int i = tid; i < copies; i += kBook) atomicSub(&c.refs[w.from[i]], 1);
    for (int i = tid; i < n; i += kBook) c.lengths[seqs[i]] += counts[i];
}

__global__ __launch_bounds__(kThreads) void fork_kernel(CacheView c, const int32_t* parents, const int32_t* children,
                                                        const int32_t* tokens) {
    const int i = blockIdx.x, tid = threadIdx.x;
    const int parent = parents[i], child = children[i];
    if ((unsigned)parent >= (unsigned)c.seqs || (unsigned)child >= (unsigned)c.seqs) {
        if (tid == 0) cache_report(c, kCacheBadSeq, (unsigned)parent >= (unsigned)c.seqs ? parent : child, 0);
        return;
    }
    const int held = c.clamp_length(c.lengths[parent]);
    const int keep = tokens ? tokens[i] : held;
    const bool used = c.lengths[child] != 0;
    __syncthreads();  // every thread has read the child's length
    if (used || parent == child) {
        if (tid == 0) cache_report(c, kCacheInUse, child, 0);
        return;
    }
    if (keep < 0 || keep > held) {
        if (tid == 0) cache_report(c, kCacheBadCount, parent, keep);
        return;
    }
    const int pages = (int)(((int64_t)keep + c.page_tokens - 1) >> c.page_shift);
    const int32_t* from = c.tables + (int64_t)parent * c.table_pages;
    int32_t* to = c.tables + (int64_t)child * c.table_pages;
    for (int k = tid; k < pages; k += kThreads) {
        const int page = from[k];
        to[k] = page;
        if ((unsigned)page < (unsigned)c.pages) atomicAdd(&c.refs[page], 1);
        else cache_report(c, kCacheBadPage, page, 0);
    }
    if (tid == 0) c.lengths[child] = keep;
}

__global__ __launch_bounds__(kThreads) void release_kernel(CacheView c, const int32_t* seqs, const int32_t* keeps) {
    const int i = blockIdx.x, tid = threadIdx.x;
    const int seq = seqs[i], keep = keeps ? keeps[i] : 0;
    if ((unsigned)seq >= (unsigned)c.seqs) {
        if (tid == 0) cache_report(c, kCacheBadSeq, seq, 0);
        return;
    }
    const int held = c.clamp_length(c.lengths[seq]);
    __syncthreads();  // every thread has read the length
    if (keep < 0 || keep > held) {
        if (tid == 0) cache_report(c, kCacheBadCount, seq, keep);
        return;
    }
    const int mask = c.page_tokens - 1;
    const int first = (int)(((int64_t)keep + mask) >> c.page_shift);
    const int end = (int)(((int64_t)held + mask) >> c.page_shift);
    int32_t* row = c.tables + (int64_t)seq * c.table_pages;
    for (int k = first + tid; k < end; k += kThreads) {
        const int page = row[k];
        row[k] = -1;
        if ((unsigned)page < (unsigned)c.pages) atomicSub(&c.refs[page], 1);
        else cache_report(c, kCacheBadPage, page, 0);
    }
    if (tid == 0) c.lengths[seq] = keep;
}

// One workgroup: the r-th live page at or past the live count moves to the
// r-th free page below it.
__global__ __launch_bounds__(kBook) void compact_kernel(CacheView c, PageScratch w, int32_t* live_out) {
    const int tid = threadIdx.x;
    int live = 0;
    for (int64_t p0 = 0; p0 < c.pages; p0 += kBook) {
        int total;
        block_scan(p0 + tid < c.pages && c.refs[p0 + tid] != 0, &total);
        live += total;
    }
    int from = 0, to = 0;
    for (int64_t p0 = 0; p0 < c.pages; p0 += kBook) {
        const int64_t p = p0 + tid;
        const bool in = p < c.pages, used = in && c.refs[p] != 0;
        if (in) w.remap[p] = (int)p;
        int total;
        int at = from + block_scan(used && p >= live, &total);
        from += total;
        if (used && p >= live) w.from[at] = (int)p;
        const bool hole = in && !used && p < live;
        at = to + block_scan(hole, &total);
        to += total;
        if (hole) w.to[at] = (int)p;
    }
    __syncthreads();
    for (int i = tid; i < from; i += kBook) {
        const int a = w.from[i], b = w.to[i];
        w.remap[a] = b;
        c.refs[b] = c.refs[a];
        c.refs[a] = 0;
    }
    if (tid == 0) {
        *w.count = from;
        if (live_out) *live_out = live;
    }
}

__global__ __launch_bounds__(kThreads) void remap_kernel(CacheView c, PageScratch w) {
    const int seq = blockIdx.x;
    const int length = c.clamp_length(c.lengths[seq]);
    const int pages = (int)(((int64_t)length + c.page_tokens - 1) >> c.page_shift);
    int32_t* row = c.tables + (int64_t)seq * c.table_pages;
    for (int k = threadIdx.x; k < pages; k += kThreads) {
        const int page = row[k];
        if ((unsigned)page < (unsigned)c.pages) row[k] = w.remap[page];
        else cache_report(c, kCacheBadPage, page, 0);
    }
}

// A workgroup copies one layer's k or v of a page, its largest values too.
__global__ __launch_bounds__(kThreads) void copy_kernel(CacheView c, const int32_t* from, const int32_t* to,
                                                        const int32_t* count, int n) {
    const int64_t pairs = count ? *count : n;
    const int64_t units = pairs * c.layers * 2;
    const int64_t bytes = c.page_codes();
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t pair = u / (2 * c.layers), layer = (u >> 1) % c.layers;
        const int a = from[pair], b = to[pair];
        if ((unsigned)a >= (unsigned)c.pages || (unsigned)b >= (unsigned)c.pages) {
            if (threadIdx.x == 0) cache_report(c, kCacheBadPage, (unsigned)a >= (unsigned)c.pages ? a : b, 0);
            continue;
        }
        int8_t* codes = (u & 1) ? c.v_codes : c.k_codes;
        float* max = (u & 1) ? c.v_max : c.k_max;
        const int64_t sa = c.slab(layer, a), sb = c.slab(layer, b);
        const uint4* src = (const uint4*)(codes + sa * bytes);  // page_codes is a multiple of 512
        uint4* dst = (uint4*)(codes + sb * bytes);
        for (int64_t i = threadIdx.x; i < bytes / 16; i += kThreads) dst[i] = src[i];
        for (int h = threadIdx.x; h < c.kv_heads; h += kThreads) max[sb * c.kv_heads + h] = max[sa * c.kv_heads + h];
    }
}

}  // namespace

hipError_t launch_cache_append(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x,
                               hipStream_t s) {
    const dim3 grid((unsigned)ragged_slots(r.tokens, r.n, c.page_shift), c.kv_heads, 2);
    if (x.dtype == MANTA_ROCM_F32) append_kernel<F32><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else if (x.dtype == MANTA_ROCM_F16) append_kernel<F16><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else append_kernel<Bf16><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    return hipGetLastError();
}

hipError_t launch_cache_read(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s) {
    const dim3 grid((unsigned)ragged_slots(r.tokens, r.n, c.page_shift), c.kv_heads, 2);
    if (x.dtype == MANTA_ROCM_F32) read_kernel<F32><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else if (x.dtype == MANTA_ROCM_F16) read_kernel<F16><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else read_kernel<Bf16><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    return hipGetLastError();
}

hipError_t launch_cache_extend(const CacheView& c, const PageScratch& w, const int32_t* seqs, const int32_t* counts,
                               int n, int32_t* free_list, hipStream_t s) {
    extend_kernel<<<1, kBook, 0, s>>>(c, w, seqs, counts, n, free_list);
    return hipGetLastError();
}

hipError_t launch_cache_fork(const CacheView& c, const int32_t* parents, const int32_t* children,
                             const int32_t* tokens, int n, hipStream_t s) {
    fork_kernel<<<n, kThreads, 0, s>>>(c, parents, children, tokens);
    return hipGetLastError();
}

hipError_t launch_cache_release(const CacheView& c, const int32_t* seqs, const int32_t* keep, int n, hipStream_t s) {
    release_kernel<<<n, kThreads, 0, s>>>(c, seqs, keep);
    return hipGetLastError();
}

hipError_t launch_cache_compact(const CacheView& c, const PageScratch& w, int32_t* live, hipStream_t s) {
    compact_kernel<<<1, kBook, 0, s>>>(c, w, live);
    return hipGetLastError();
}

hipError_t launch_cache_remap(const CacheView& c, const PageScratch& w, hipStream_t s) {
    remap_kernel<<<c.seqs, kThreads, 0, s>>>(c, w);
    return hipGetLastError();
}

hipError_t launch_cache_copy(const CacheView& c, const int32_t* from, const int32_t* to, const int32_t* count, int n,
                             hipStream_t s) {
    const int64_t units = (int64_t)n * c.layers * 2;
    copy_kernel<<<(unsigned)(units < 2048 ? units : 2048), kThreads, 0, s>>>(c, from, to, count, n);
    return hipGetLastError();
}

}  // namespace manta
