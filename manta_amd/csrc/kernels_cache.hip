// kernels_cache.hip -- contents and pages of the 8-bit key/value cache.
//
// Append and read move a page's head at a time; the page calls work on the
// book (refs, lengths, tables) in device memory, so a decoding loop never
// waits for the host.  The layout and the mapping of ragged batches are in
// cache_layout.hpp.
#include "cache_kernels.hpp"
#include "code_common.hpp"
#include "decode_layout.hpp"

#pragma clang fp contract(off)

namespace manta {

namespace {

constexpr int kThreads = 256;

// This workgroup's piece of the ragged batch and its sequence: false if there
// is none.
__device__ __forceinline__ bool my_piece(const CacheView& c, const RaggedRows& r, Piece* p, int* seq) {
    const int64_t slot = blockIdx.x;
    const Owner o = find_owner(c, r, slot, [&](int offset, int j) { return ragged_base(offset, j, c.page_shift); });
    *seq = o.seq;
    if (o.length < 0) {
        if (threadIdx.x == 0) cache_report(c, kCacheBadSeq, o.seq, 0);
        return false;
    }
    return ragged_piece(o.from, o.to, c.clamp_length(o.length), slot - ragged_base(o.from, o.i, c.page_shift),
                        c.page_shift, p);
}
// The piece's page: false where the table names none.
__device__ __forceinline__ bool piece_page(const CacheView& c, const Piece& p, int seq, int* page) {
    *page = c.tables[(int64_t)seq * c.table_pages + p.index];
    if ((unsigned)*page < (unsigned)c.pages) return true;
    if (threadIdx.x == 0) cache_report(c, kCacheBadPage, *page, 0);
    return false;
}

// Whether append leaves the piece alone.  A sequence whose extend was refused
// has not grown: its last tokens are not the rows' place.  A page that several
// tables name is not written (extend gives a sequence that goes on in one its
// own copy).  Both are asked for with the page and looked at before the first
// store, so that nothing waits for them.
struct Keep {
    int refused, refs;
    __device__ __forceinline__ Keep(const CacheView& c, int seq, int page) : refused(c.refused[seq]), refs(c.refs[page]) {}
    __device__ __forceinline__ bool operator()(const CacheView& c, int page) const {
        if (refused) return true;
        if (refs <= 1) return false;
        if (threadIdx.x == 0) cache_report(c, kCacheShared, page, 0);
        return true;
    }
};

__device__ __forceinline__ int quantise(float x, float max) {
    const float r = __builtin_rintf(__fdiv_rn(x * 127.0f, max));
    return (int)fminf(127.0f, fmaxf(-127.0f, r));
}
// Where 127 * max would leave f32, products with codes are taken of numbers
// 2^-8 as large: code * old / max and code * max / 127 are the same, rounding
// for rounding.
__device__ __forceinline__ float headroom(float max) { return max >= 0x1p121f ? 0x1p-8f : 1.0f; }
__device__ __forceinline__ int requantise(int code, float old, float max) {
    const float h = headroom(max);
    const float r = __builtin_rintf(__fdiv_rn((float)code * (old * h), max * h));
    return (int)fminf(127.0f, fmaxf(-127.0f, r));
}

// A page's values.
struct Values {
    float big, up;
    __device__ __forceinline__ explicit Values(float max) : big(max * headroom(max)), up(max >= 0x1p121f ? 0x1p8f : 1.0f) {}
    __device__ __forceinline__ float operator()(int code) const { return __fdiv_rn((float)code * big, 127.0f) * up; }
};

// One page's head of k (blockIdx.z 0) or v (1).
template <class E>
__global__ __launch_bounds__(kThreads) void append_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    Piece p;
    int seq, page;
    if (!my_piece(c, r, &p, &seq) || !piece_page(c, p, seq, &page)) return;
    const Keep keep(c, seq, page);
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
    if (keep(c, page)) return;
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

// Rows that start on 16 bytes and split into 16-byte pieces.  The same
// results, and bytes bound: a new value is read once and held in registers
// (4 NU pieces a thread) while the workgroup finds the largest.  v's codes lie
// token after token: a thread takes four tokens' pieces, so that it has four
// bytes for each of its columns.
template <class E, int NU>
__global__ __launch_bounds__(kThreads) void append_wide_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    constexpr int V = E::kWide;
    struct alignas(16) Piece16 {
        T v[V];
    };
    Piece p;
    int seq, page;
    if (!my_piece(c, r, &p, &seq)) return;
    const int head = blockIdx.y, is_v = blockIdx.z;
    const int tid = threadIdx.x, d = c.head_dim, per = d / V, count = p.to - p.from;
    const T* src = is_v ? (const T*)x.v + head * x.v_head : (const T*)x.k + head * x.k_head;
    const int64_t stride = is_v ? x.v_token : x.k_token;
    // The new values are on their way before the page is asked for.
    // k: piece tid + 256 (4 u + w); v: token 4 g + w of the page, g and the
    // column from tid + 256 u
    const int g0 = p.from >> 2, groups = ((p.to + 3) >> 2) - g0;
    Piece16 y[NU][4];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < NU; u++) {
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int e = is_v ? tid + kThreads * u : tid + kThreads * (4 * u + w);
            const int t = is_v ? 4 * (g0 + e / per) + w - p.from : e / per, at = V * (e % per);
            if (t >= 0 && t < count) y[u][w] = *(const Piece16*)(src + (p.row + t) * stride + at);
            else y[u][w] = Piece16{};
        }
    }
    if (!piece_page(c, p, seq, &page)) return;
    const Keep keep(c, seq, page);
    float* slot = (is_v ? c.v_max : c.k_max) + c.slab(layer, page) * c.kv_heads + head;
    const float old = p.from ? *slot : 0.0f;

    // Words of the codes that tokens before have, four a word (of v the last
    // word may be theirs in part); the first ones fetched ahead.
    const int64_t base = c.slab(layer, page) * c.page_codes() + (int64_t)head * c.page_tokens * c.pitch;
    int8_t* codes = (is_v ? c.v_codes : c.k_codes) + base;
    const int v_words = (p.from + 3) >> 2, words = is_v ? c.pitch * v_words : p.from * c.pitch / 4;
    auto word_at = [&](int e, int* bytes) {
        *bytes = is_v ? min(4, p.from - 4 * (e % v_words)) : 4;
        return (uint32_t*)(is_v ? codes + (e / v_words) * c.page_tokens : codes) + (is_v ? e % v_words : e);
    };
    constexpr int OLD = 2;
    uint32_t was[OLD], *was_at[OLD];
    int was_bytes[OLD];
#pragma unroll
    for (int k = 0; k < OLD; k++) {
        was_bytes[k] = 0;
        if (tid + kThreads * k < words) {
            was_at[k] = word_at(tid + kThreads * k, &was_bytes[k]);
            was[k] = *was_at[k];
        }
    }

#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int j = 0; j < V; j++) top = max(top, __float_as_uint(E::load(y[u][w].v[j])) & 0x7FFFFFFFu);
    __shared__ uint32_t tops[kThreads / 64];
    for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();  // (every thread has read *slot, too)
    for (int w = 0; w < kThreads / 64; w++) top = max(top, tops[w]);
    const bool bad = top >= 0x7F800000u || old != old;
    float big = fmaxf(__uint_as_float(top), old);
    const bool zero = bad || big < 0x1p-126f;  // every code 0
    const bool raise = big > old;
    const bool exact = big >= 0x1p121f;
    if (zero) big = bad ? __builtin_nanf("") : 0.0f;
    if (keep(c, page)) return;
    if (tid == 0) *slot = big;
    const float inv = 1.0f / big;

    if (p.from && (raise || zero)) {
        auto renew = [&](uint32_t word, uint32_t* at, int bytes) {
            const float h = headroom(big);
            float t[4];
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = (float)(int8_t)(word >> (8 * j)) * (old * h);
            word = zero ? 0 : ratio_codes(t, big * h, inv, exact);
            if (bytes == 4) *at = word;
            else
                for (int j = 0; j < bytes; j++) ((uint8_t*)at)[j] = (uint8_t)(word >> (8 * j));
        };
#pragma unroll
        for (int k = 0; k < OLD; k++)
            if (was_bytes[k]) renew(was[k], was_at[k], was_bytes[k]);
        for (int e = tid + kThreads * OLD; e < words; e += kThreads) {
            int bytes;
            uint32_t* at = word_at(e, &bytes);
            renew(*at, at, bytes);
        }
    }
    if (!is_v) {
#pragma unroll
        for (int u = 0; u < NU; u++) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int e = tid + kThreads * (4 * u + w), t = e / per, col = V * (e % per);
                if (t >= count) continue;
                uint32_t* dst = (uint32_t*)(codes + (p.from + t) * c.pitch + col);
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    float f[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) f[k] = E::load(y[u][w].v[j + k]) * 127.0f;
                    dst[j / 4] = zero ? 0 : ratio_codes(f, big, inv, exact);
                }
            }
        }
        const int rest = (c.pitch - d) / 4;
        for (int e = tid; e < count * rest; e += kThreads)
            ((uint32_t*)(codes + (p.from + e / rest) * c.pitch + d))[e % rest] = 0;
        return;
    }
#pragma unroll
    for (int u = 0; u < NU; u++) {
        const int e = tid + kThreads * u, g = e / per, col = V * (e % per), t0 = 4 * (g0 + g);
        if (g >= groups) continue;
        const bool whole = t0 >= p.from && t0 + 4 <= p.to;
#pragma unroll
        for (int j = 0; j < V; j++) {
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = E::load(y[u][k].v[j]) * 127.0f;
            const uint32_t word = zero ? 0 : ratio_codes(f, big, inv, exact);
            int8_t* dst = codes + (col + j) * c.page_tokens + t0;
            if (whole) {
                *(uint32_t*)dst = word;
            } else {
#pragma unroll
                for (int w = 0; w < 4; w++)
                    if (t0 + w >= p.from && t0 + w < p.to) dst[w] = (int8_t)(word >> (8 * w));
            }
        }
    }
    for (int e = tid; e < (c.pitch - d) * count; e += kThreads)
        codes[(d + e / count) * c.page_tokens + p.from + e % count] = 0;
}

template <class E>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    Piece p;
    int seq, page;
    if (!my_piece(c, r, &p, &seq) || !piece_page(c, p, seq, &page)) return;
    const int head = blockIdx.y, is_v = blockIdx.z, d = c.head_dim;
    T* dst = is_v ? (T*)x.v + head * x.v_head : (T*)x.k + head * x.k_head;
    const int64_t stride = is_v ? x.v_token : x.k_token;
    const Values value(((is_v ? c.v_max : c.k_max) + c.slab(layer, page) * c.kv_heads)[head]);
    const int8_t* codes = (is_v ? c.v_codes : c.k_codes) + c.slab(layer, page) * c.page_codes() +
                          (int64_t)head * c.page_tokens * c.pitch;
    for (int e = threadIdx.x; e < (p.to - p.from) * d; e += kThreads) {
        const int t = e / d, col = e % d;
        const int code = is_v ? codes[col * c.page_tokens + p.from + t] : codes[(p.from + t) * c.pitch + col];
        dst[(p.row + t) * stride + col] = E::store(value(code));
    }
}

// The same for rows that start on 16 bytes and split into pieces of 8
// elements; v four tokens at a time.
template <class E>
__global__ __launch_bounds__(kThreads) void read_wide_kernel(CacheView c, int64_t layer, RaggedRows r, KvRows x) {
    typedef typename E::T T;
    struct alignas(16) Piece16 {
        T v[8];
    };
    Piece p;
    int seq, page;
    if (!my_piece(c, r, &p, &seq) || !piece_page(c, p, seq, &page)) return;
    const int head = blockIdx.y, is_v = blockIdx.z, d = c.head_dim, per = d / 8, count = p.to - p.from;
    T* dst = is_v ? (T*)x.v + head * x.v_head : (T*)x.k + head * x.k_head;
    const int64_t stride = is_v ? x.v_token : x.k_token;
    const Values page_value(((is_v ? c.v_max : c.k_max) + c.slab(layer, page) * c.kv_heads)[head]);
    const int8_t* codes = (is_v ? c.v_codes : c.k_codes) + c.slab(layer, page) * c.page_codes() +
                          (int64_t)head * c.page_tokens * c.pitch;
    auto value = [&](uint32_t word, int j) { return E::store(page_value((int8_t)(word >> (8 * j)))); };
    if (!is_v) {
        for (int e = threadIdx.x; e < count * per; e += kThreads) {
            const int t = e / per, col = 8 * (e % per);
            const uint2 w = *(const uint2*)(codes + (p.from + t) * c.pitch + col);
            Piece16 y;
#pragma unroll
            for (int j = 0; j < 8; j++) y.v[j] = value(j < 4 ? w.x : w.y, j & 3);
            *(Piece16*)(dst + (p.row + t) * stride + col) = y;
        }
        return;
    }
    const int g0 = p.from >> 2, groups = ((p.to + 3) >> 2) - g0;
    for (int e = threadIdx.x; e < groups * per; e += kThreads) {
        const int t0 = 4 * (g0 + e / per), col = 8 * (e % per);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = *(const uint32_t*)(codes + (col + j) * c.page_tokens + t0);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t0 + t < p.from || t0 + t >= p.to) continue;
            Piece16 y;
#pragma unroll
            for (int j = 0; j < 8; j++) y.v[j] = value(w[j], t);
            *(Piece16*)(dst + (p.row + (t0 + t - p.from)) * stride + col) = y;
        }
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
    int grown;                     // its length then
    bool ok;
};
__device__ Growth growth(const CacheView& c, const int32_t* seqs, const int32_t* counts, int i, bool report) {
    Growth g{0, 0, 0, 0, -1, 0, false};
    g.seq = seqs[i];
    const int add = counts[i];
    if ((unsigned)g.seq >= (unsigned)c.seqs) {
        if (report) cache_report(c, kCacheBadSeq, g.seq, 0);
        return g;
    }
    const int refused = c.refused[g.seq];  // (looked at last: nothing waits for it)
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
    g.grown = g.length + add;
    g.ok = !refused;
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
    const int first_ref = tid < c.pages ? c.refs[tid] : 1;
    Growth first{0, 0, 0, 0, -1, 0, false};  // of the list's first entries: not asked for twice
    for (int i0 = 0; i0 < n; i0 += kBook) {
        int need = 0;
        if (i0 + tid < n) {
            const Growth g = growth(c, seqs, counts, i0 + tid, true);
            if (i0 == 0) first = g;
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
        const bool is_free = p0 + tid < c.pages && (p0 ? c.refs[p0 + tid] : first_ref) == 0;
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
        for (int i = tid; i < n; i += kBook)
            if ((unsigned)seqs[i] < (unsigned)c.seqs) c.refused[seqs[i]] = 1;
        return;
    }
    __syncthreads();  // free_list is written
    int taken = 0, copies = 0;
    for (int i0 = 0; i0 < n; i0 += kBook) {
        Growth g{0, 0, 0, 0, -1, 0, false};
        if (i0 == 0) g = first;
        else if (i0 + tid < n) g = growth(c, seqs, counts, i0 + tid, false);
        const int mine = g.more + (g.last >= 0);
        int total, copied;
        int at = taken + block_scan(mine, &total);
        const int copy = copies + block_scan(g.last >= 0, &copied);
        taken += total;
        copies += copied;
        __syncthreads();  // every growth() of this step has read the book
        // (a list that names a sequence twice could ask for more than was counted)
        if (g.ok && at >= 0 && at + mine <= need && (g.last < 0 || copy < need)) {
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
            if (n <= kBook) {  // no growth() is to come
                if (g.last >= 0) atomicSub(&c.refs[g.last], 1);
                c.lengths[g.seq] = g.grown;
            }
        }
    }
    if (tid == 0) *w.count = copies;
    if (n <= kBook) return;
    // shared pages lose a reference, and lengths grow, once no growth() can
    // see it: whether a page was shared is asked of the book as it was
    __syncthreads();
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

// Entry i of a group takes over what entry parents[i] of it held.  A workgroup
// takes `columns` columns of a group's tables: it holds the parents' entries
// in LDS before it writes the first, so nothing that is still to be read is
// overwritten, and no two workgroups touch one entry.  Past a sequence's pages
// its table holds -1, so whole rows move without anybody's length, which the
// first workgroup of a group replaces.  References are added and dropped where
// an entry changes (their order does not matter: sums).  Every workgroup
// checks the whole list, so that all of them or none go on: marks of refused
// sequences are only set where every workgroup stops anyway.
constexpr int kSeen = 1 << 17;  // slots whose first naming a workgroup remembers at a time
__global__ __launch_bounds__(kThreads) void reorder_kernel(CacheView c, const int32_t* seqs, const int32_t* parents,
                                                           int n, int group, int columns) {
    extern __shared__ int32_t held[];  // [group][columns]
    __shared__ uint32_t seen[kSeen / 32];
    __shared__ int32_t slot[kMaxReorderGroup], parent[kMaxReorderGroup], length[kMaxReorderGroup];
    const int tid = threadIdx.x;
    const bool first = blockIdx.x == 0 && blockIdx.y == 0;
    int wrong = 0;
    for (int64_t s0 = 0; s0 < c.seqs; s0 += kSeen) {
        const int words = (int)((min((int64_t)kSeen, c.seqs - s0) + 31) / 32);
        for (int k = tid; k < words; k += kThreads) seen[k] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const int seq = seqs[i], p = parents[i];
            if ((unsigned)seq >= (unsigned)c.seqs) {
                if (first && s0 == 0) cache_report(c, kCacheBadSeq, seq, 0);
                wrong = 1;
            } else if (seq >= s0 && seq - s0 < kSeen) {
                const int at = (int)(seq - s0);
                if (atomicOr(&seen[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u) {
                    if (first) cache_report(c, kCacheTwice, seq, 0);
                    wrong = 1;
                }
                if (c.refused[seq]) wrong = 1;
            }
            if (p < -1 || p >= group) {
                if (first && s0 == 0) cache_report(c, kCacheBadParent, i, p);
                wrong = 1;
            }
        }
        __syncthreads();
    }
    if (__syncthreads_or(wrong)) {
        for (int i = tid; i < n && first; i += kThreads)
            if ((unsigned)seqs[i] < (unsigned)c.seqs) c.refused[seqs[i]] = 1;
        return;
    }
    const int base = blockIdx.y * group;
    for (int i = tid; i < group; i += kThreads) {
        slot[i] = seqs[base + i];
        parent[i] = parents[base + i];
    }
    __syncthreads();
    const int shift = __builtin_ctz(columns), col = tid & (columns - 1);
    const int64_t at = (int64_t)blockIdx.x * columns + col;
    const bool in = at < c.table_pages;
    for (int i = tid >> shift; i < group && in; i += kThreads >> shift)
        held[(i << shift) + col] = c.tables[(int64_t)slot[i] * c.table_pages + at];
    if (blockIdx.x == 0)
        for (int i = tid; i < group; i += kThreads) length[i] = c.lengths[slot[i]];
    __syncthreads();
    for (int i = tid >> shift; i < group && in; i += kThreads >> shift) {
        const int p = parent[i], before = held[(i << shift) + col], after = p < 0 ? -1 : held[(p << shift) + col];
        if (before == after) continue;
        c.tables[(int64_t)slot[i] * c.table_pages + at] = after;
        if ((unsigned)before < (unsigned)c.pages) atomicSub(&c.refs[before], 1);
        if ((unsigned)after < (unsigned)c.pages) atomicAdd(&c.refs[after], 1);
    }
    if (blockIdx.x == 0)
        for (int i = tid; i < group; i += kThreads) c.lengths[slot[i]] = parent[i] < 0 ? 0 : length[parent[i]];
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

// A workgroup copies one layer's k or v of a page, its largest values too, 8
// pieces of 16 bytes a thread on their way.  remap, when given: and then
// rewrites tables (compact; the copies do not read them).
__global__ __launch_bounds__(kThreads) void copy_kernel(CacheView c, const int32_t* from, const int32_t* to,
                                                        const int32_t* count, int n, const int32_t* remap) {
    const int64_t pairs = count ? *count : n;
    const int64_t units = pairs * c.layers * 2;
    const int64_t bytes = c.page_codes(), pieces = bytes / 16;
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
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4* src = (const u32x4*)(codes + sa * bytes);  // page_codes is a multiple of 512
        u32x4* dst = (u32x4*)(codes + sb * bytes);
        constexpr int AHEAD = 8;
        int64_t i = threadIdx.x;
        for (; i + (AHEAD - 1) * kThreads < pieces; i += AHEAD * kThreads) {
            u32x4 y[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) y[k] = src[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) dst[i + k * kThreads] = y[k];
        }
        for (; i < pieces; i += kThreads) dst[i] = src[i];
        for (int h = threadIdx.x; h < c.kv_heads; h += kThreads) max[sb * c.kv_heads + h] = max[sa * c.kv_heads + h];
    }
    if (!remap) return;
    for (int seq = blockIdx.x; seq < c.seqs; seq += gridDim.x) {
        const int length = c.clamp_length(c.lengths[seq]);
        const int pages = (int)(((int64_t)length + c.page_tokens - 1) >> c.page_shift);
        int32_t* row = c.tables + (int64_t)seq * c.table_pages;
        for (int k = threadIdx.x; k < pages; k += kThreads) {
            const int page = row[k];
            if ((unsigned)page < (unsigned)c.pages) row[k] = remap[page];
            else cache_report(c, kCacheBadPage, page, 0);
        }
    }
}

}  // namespace

template <class E>
static hipError_t append_of(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s) {
    const dim3 grid((unsigned)ragged_slots(r.tokens, r.n, c.page_shift), c.kv_heads, 2);
    // a few tokens a sequence are soon done and wait less in the plain kernel
    // (64 sequences, 8 heads of 128, with the read back: 1 token each 12.7 us
    // against 16.4, 8 20.6 against 22.3, 16 27.0 against 24.6; prompts of up to
    // 2048: 184 us against 74)
    if (!x.wide || c.head_dim % E::kWide != 0 || r.tokens < (int64_t)12 * r.n) {
        append_kernel<E><<<grid, kThreads, 0, s>>>(c, layer, r, x);
        return hipGetLastError();
    }
    // four-token units of a page's head to a thread
    const int units = (c.page_tokens / 4 * (c.head_dim / E::kWide) + kThreads - 1) / kThreads;
    if (units <= 1) append_wide_kernel<E, 1><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else if (units <= 2) append_wide_kernel<E, 2><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else if (units <= 4) append_wide_kernel<E, 4><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else append_wide_kernel<E, 8><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    return hipGetLastError();
}

hipError_t launch_cache_append(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x,
                               hipStream_t s) {
    if (x.dtype == MANTA_ROCM_F32) return append_of<F32>(c, layer, r, x, s);
    if (x.dtype == MANTA_ROCM_F16) return append_of<F16>(c, layer, r, x, s);
    return append_of<Bf16>(c, layer, r, x, s);
}

template <class E>
static hipError_t read_of(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s) {
    const dim3 grid((unsigned)ragged_slots(r.tokens, r.n, c.page_shift), c.kv_heads, 2);
    if (x.wide && c.head_dim % 8 == 0) read_wide_kernel<E><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    else read_kernel<E><<<grid, kThreads, 0, s>>>(c, layer, r, x);
    return hipGetLastError();
}

hipError_t launch_cache_read(const CacheView& c, int64_t layer, const RaggedRows& r, const KvRows& x, hipStream_t s) {
    if (x.dtype == MANTA_ROCM_F32) return read_of<F32>(c, layer, r, x, s);
    if (x.dtype == MANTA_ROCM_F16) return read_of<F16>(c, layer, r, x, s);
    return read_of<Bf16>(c, layer, r, x, s);
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

hipError_t launch_cache_reorder(const CacheView& c, const int32_t* seqs, const int32_t* parents, int n, int group,
                                hipStream_t s) {
    const int columns = reorder_columns(group);
    const dim3 grid((c.table_pages + columns - 1) / columns, n / group);
    reorder_kernel<<<grid, kThreads, (size_t)group * columns * 4, s>>>(c, seqs, parents, n, group, columns);
    return hipGetLastError();
}

hipError_t launch_cache_compact(const CacheView& c, const PageScratch& w, int32_t* live, hipStream_t s) {
    compact_kernel<<<1, kBook, 0, s>>>(c, w, live);
    return hipGetLastError();
}

hipError_t launch_cache_copy(const CacheView& c, const int32_t* from, const int32_t* to, const int32_t* count, int n,
                             const int32_t* remap, hipStream_t s) {
    int64_t units = (int64_t)n * c.layers * 2;
    if (remap && units < c.seqs) units = c.seqs;
    copy_kernel<<<(unsigned)(units < 2048 ? units : 2048), kThreads, 0, s>>>(c, from, to, count, n, remap);
    return hipGetLastError();
}

}  // namespace manta
