// cache_layout.hpp -- where things lie in the key/value cache, the checks of
// its arguments, and the mapping of a ragged batch's work to workgroups.
// Plain C++ (no HIP), shared by the kernels, the C ABI and the CPU tests.
#pragma once

#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include "manta_cache.h"

#ifdef __HIP__
#define MANTA_HD __host__ __device__ __forceinline__
#else
#define MANTA_HD inline
#endif

namespace manta {

constexpr int kMaxHeadDim = 256;
constexpr int64_t kMaxInt32 = 0x7FFFFFFF;
// A launch has less than 2^32 threads: a workgroup a sequence, or one a slot
// of a ragged batch (tokens / 16 + 2 n of them).
constexpr int64_t kMaxSeqs = 1 << 21;
constexpr int64_t kMaxTokens = 1 << 25;

// What the kernels know of a cache.
struct CacheView {
    int8_t* k_codes;
    int8_t* v_codes;
    float* k_max;
    float* v_max;
    int32_t* refs;     // [pages]
    int32_t* lengths;  // [seqs]
    int32_t* tables;   // [seqs][table_pages]
    int32_t* refused;  // [seqs]: 1 from a refused extend until it is reported
    unsigned long long* err;
    uint32_t* err_flag;  // host memory: 1 where *err may hold something
    int64_t layers, pages;
    int page_tokens, page_shift;
    int kv_heads, head_dim, pitch;
    int seqs, table_pages;

    MANTA_HD int64_t page_codes() const { return (int64_t)kv_heads * page_tokens * pitch; }
    MANTA_HD int64_t slab(int64_t layer, int64_t page) const { return layer * pages + page; }
    // a sequence's tokens, within what its table can name
    MANTA_HD int clamp_length(int len) const {
        const int64_t most = (int64_t)table_pages << page_shift;
        return len < 0 ? 0 : len > most ? (int)most : len;
    }
};

// What a kernel found wrong, in one word (0: nothing).  The largest word is
// kept, so what is reported does not depend on the order of the threads.
enum CacheError {
    kCacheBadSeq = 1,    // a: the sequence
    kCacheBadPage = 2,   // a: the page
    kCacheFull = 3,      // a: pages needed, b: pages free (unsigned)
    kCacheInUse = 4,     // a: the sequence
    kCacheBadCount = 5,  // a: the sequence, b: the count
    kCacheBadOffsets = 6,  // a: the entry of the batch
    kCacheShared = 7,      // a: the page
    kCacheBadParent = 8,   // a: the entry, b: its parent
    kCacheTwice = 9,       // a: the sequence
};
MANTA_HD unsigned long long cache_error(int kind, int64_t a, int64_t b) {
    return ((unsigned long long)kind << 60) | (((unsigned long long)a & 0x3FFFFFFFull) << 30) |
           ((unsigned long long)b & 0x3FFFFFFFull);
}

inline void describe_cache_error(unsigned long long w, char* out, size_t size) {
    const int kind = (int)(w >> 60);
    const long long a = (long long)((w >> 30) & 0x3FFFFFFF), b = (long long)(w & 0x3FFFFFFF);
    // indices are kept in 30 bits, sign included
    const long long as = a & 0x20000000 ? a - 0x40000000 : a, bs = b & 0x20000000 ? b - 0x40000000 : b;
    if (kind == kCacheBadSeq) snprintf(out, size, "cache sequence %lld out of range", as);
    else if (kind == kCacheBadPage) snprintf(out, size, "cache page %lld out of range", as);
    else if (kind == kCacheFull) snprintf(out, size, "cache is out of pages: %lld needed, %lld free", a, b);
    else if (kind == kCacheInUse) snprintf(out, size, "cache sequence %lld is not empty", as);
    else if (kind == kCacheBadOffsets) snprintf(out, size, "cache offsets descend at entry %lld of the batch", as);
    else if (kind == kCacheShared) snprintf(out, size, "cache page %lld is shared: extend copies it before an append", as);
    else if (kind == kCacheBadParent) snprintf(out, size, "cache reorder entry %lld: parent %lld out of range", as, bs);
    else if (kind == kCacheTwice) snprintf(out, size, "cache reorder names sequence %lld twice", as);
    else snprintf(out, size, "cache sequence %lld: count %lld out of range", as, bs);
}

// ---- a ragged batch in page-sized pieces ----
// Rows [a, b) of sequence i lie in at most (b - a) / page + 2 pages, so slots
// [a / page + 2 i, b / page + 2 (i + 1)) are enough for them, and the last
// slot depends on the host's `tokens` and `n` alone.
MANTA_HD int64_t ragged_slots(int64_t tokens, int64_t n, int shift) { return (tokens >> shift) + 2 * n; }
MANTA_HD int64_t ragged_base(int offset, int64_t i, int shift) { return ((int64_t)offset >> shift) + 2 * i; }

// The piece of a sequence that lies in its `local`-th touched page: tokens
// [from, to) of the page `index` of the table, the first of them row `row`.
struct Piece {
    int index, from, to, row;
};
MANTA_HD bool ragged_piece(int a, int b, int length, int64_t local, int shift, Piece* p) {
    const int page = 1 << shift;
    const int count = b - a;
    if (count <= 0 || length <= 0 || local < 0) return false;
    const int start = length - count;  // may be negative: the rows before position 0 are skipped
    const int first = (start > 0 ? start : 0) >> shift;
    const int64_t index = first + local;
    if (index * page >= length) return false;
    const int begin = (int)index * page;
    const int lo = start > begin ? start : begin;
    const int hi = length - begin < page ? length : begin + page;
    p->index = (int)index;
    p->from = lo - begin;
    p->to = hi - begin;
    p->row = a + (lo - start);
    return true;
}

// ---- a ragged batch in tiles of query rows ----
// Row r of sequence i and kv head h is query head h * group + r % group of
// the sequence's token r / group.  A tile is `rows` of them; ceil(count *
// group / rows) tiles fit the slots [tile_base(a, i), tile_base(b, i + 1)).
MANTA_HD int64_t tile_slots(int64_t tokens, int64_t n, int64_t group, int rows) { return tokens * group / rows + n; }
MANTA_HD int64_t tile_base(int offset, int64_t i, int64_t group, int rows) { return offset * group / rows + i; }
// A sequence's tiles: over a batch of ascending offsets at most tile_slots.
MANTA_HD int tile_count(int from, int to, int64_t group, int rows) {
    return to > from ? (int)(((int64_t)(to - from) * group + rows - 1) / rows) : 0;
}
// Whether each tile of a kv head, `tiles` of them, has a ticket of its own.
MANTA_HD bool tiles_fit(int64_t tiles, int64_t kv_heads, int64_t tickets) { return tiles * kv_heads <= tickets; }

// ---- checks (nullptr: nothing wrong) ----

MANTA_HD bool element_type(int dtype) {
    return dtype == MANTA_ROCM_F32 || dtype == MANTA_ROCM_F16 || dtype == MANTA_ROCM_BF16;
}

inline const char* check_cache_shape(const MantaRocmCacheShape& s) {
    if (s.layers <= 0 || s.pages <= 0 || s.kv_heads <= 0 || s.seqs <= 0 || s.table_pages <= 0)
        return "layers, pages, kv_heads, seqs and table_pages must be positive";
    if (s.page_tokens != 16 && s.page_tokens != 32 && s.page_tokens != 64 && s.page_tokens != 128)
        return "page_tokens must be 16, 32, 64 or 128";
    if (s.head_dim <= 0 || s.head_dim > kMaxHeadDim) return "head_dim must be 1 to 256";
    if (s.kv_heads > 65535 || s.layers > 65535) return "at most 65535 kv_heads and layers";
    if (s.pages > (kMaxInt32 >> 2) || s.seqs > kMaxSeqs) return "too many pages or sequences";
    if (s.table_pages > kMaxInt32 / s.page_tokens) return "table_pages * page_tokens exceeds int32 lengths";
    if (s.pages + s.seqs + s.seqs * s.table_pages > (kMaxInt32 >> 1)) return "the book exceeds int32 entries";
    return nullptr;
}

// strides of [tokens, heads, head_dim] elements
inline const char* check_strides(int64_t tokens, int64_t heads, int64_t head_dim, int64_t token, int64_t head) {
    if (token < 0 || head < 0) return "strides must not be negative";
    if (heads > 1 && head < head_dim) return "head stride is below head_dim";
    if (tokens > 1 && token < head_dim) return "token stride is below head_dim";
    return nullptr;
}

// ... that are written: rows may not run into each other
inline const char* check_out_strides(int64_t tokens, int64_t heads, int64_t head_dim, int64_t token, int64_t head) {
    if (const char* bad = check_strides(tokens, heads, head_dim, token, head)) return bad;
    if (tokens <= 1 || heads <= 1) return nullptr;
    typedef __int128 wide;
    if ((wide)token >= (wide)head * (heads - 1) + head_dim) return nullptr;  // heads within a token
    if ((wide)head >= (wide)token * (tokens - 1) + head_dim) return nullptr;  // tokens within a head
    // rows a of the one axis and b of the other apart start near each other
    const bool few_heads = heads <= tokens;
    const int64_t n = few_heads ? heads : tokens, most = few_heads ? tokens : heads;
    const wide step = few_heads ? head : token, other = few_heads ? token : head;
    for (int64_t a = 1; a < n; a++) {
        const wide at = step * a, b = at / other;
        if (b >= 1 && b < most && at - b * other < head_dim) return "rows of the result run into each other";
        if (b + 1 < most && (b + 1) * other - at < head_dim) return "rows of the result run into each other";
    }
    return nullptr;
}

inline const char* check_batch(int64_t n, int64_t tokens, int64_t seqs, bool listed) {
    if (n < 0 || tokens < 0) return "negative count";
    if (n > kMaxSeqs || tokens > kMaxTokens) return "too many sequences or tokens";
    if (!listed && n > seqs) return "more sequences than the cache has";
    return nullptr;
}

}  // namespace manta
