// cache.cpp -- implementation of include/manta_cache.h: argument checks,
// device memory and the launch sequences of the rotary and cache calls.
#include "manta_cache.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdlib>
#include <new>

#include "cache_kernels.hpp"
#include "cache_layout.hpp"
#include "runtime_internal.hpp"

using manta::CacheView;
using manta_rt::fail;

// Partial results of attention whose keys are split over workgroups, and the
// tickets of the last one to finish (zero between calls).
constexpr size_t kPartialBytes = (size_t)96 << 20;
constexpr size_t kAttendTickets = 65536;

struct MantaRocmRotary : manta_rt::Attached {
    MantaRocm* rt = nullptr;
    double* turns = nullptr;
    int rot = 0, layout = 0;
    float magnitude = 1.0f;
    void release() override {
        if (turns) (void)hipFree(turns);
        turns = nullptr;
        rt = nullptr;
    }
};

struct MantaRocmCache : manta_rt::Attached {
    MantaRocm* rt = nullptr;
    MantaRocmCacheShape shape{};
    CacheView view{};
    void* memory = nullptr;  // codes and largest values
    void* book = nullptr;    // refs, lengths, tables; then the scratch and the refused sequences' marks
    int64_t code_bytes = 0, max_count = 0, book_count = 0;
    manta::PageScratch scratch{};
    int32_t* free_list = nullptr;
    float* partial = nullptr;
    uint32_t* tickets = nullptr;
    int reported(void* stream) override {
        return (int)hipMemsetAsync(view.refused, 0, (size_t)view.seqs * 4, (hipStream_t)stream);
    }
    void release() override {
        if (memory) (void)hipFree(memory);
        if (book) (void)hipFree(book);
        if (partial) (void)hipFree(partial);
        memory = book = nullptr;
        partial = nullptr;
        rt = nullptr;
    }
};

namespace {

#define TRY_HIP(call, what)                                                             \
    do {                                                                                \
        hipError_t e_ = (call);                                                         \
        if (e_ != hipSuccess)                                                           \
            return fail(err, MANTA_ROCM_ERROR, "%s: %s (%s)", what, hipGetErrorName(e_), hipGetErrorString(e_)); \
    } while (0)

// A launch, counted and timed as the runtime's other kernels are.
template <class F>
int launch(MantaRocm* rt, const char* what, char** err, F f) {
    void* ev = manta_rt::launch_begin(rt);
    const hipError_t e = f((hipStream_t)manta_rt::runtime_stream(rt));
    manta_rt::launch_end(rt, what, ev);
    if (e != hipSuccess)
        return fail(err, MANTA_ROCM_ERROR, "%s: %s (%s)", what, hipGetErrorName(e), hipGetErrorString(e));
    return MANTA_ROCM_OK;
}

int check_cache(MantaRocm* rt, const MantaRocmCache* c, const char* what, char** err) {
    if (!c) return fail(err, MANTA_ROCM_ERROR, "%s: nil cache", what);
    if (!c->rt) return fail(err, MANTA_ROCM_ERROR, "%s: the cache's runtime is destroyed", what);
    if (c->rt != rt) return fail(err, MANTA_ROCM_ERROR, "%s: the cache belongs to another runtime", what);
    return manta_rt::use(rt, err);
}

bool aligned16(const void* p, int64_t a, int64_t b, int size) {
    return ((uintptr_t)p % 16) == 0 && (a * size) % 16 == 0 && (b * size) % 16 == 0;
}

int element_size(int dtype) { return dtype == MANTA_ROCM_F32 ? 4 : 2; }

}  // namespace

extern "C" {

// ------------------------------------------------------------------ rotary

int manta_rocm_rotary_freqs(int64_t rot, double base, int scaling, double factor, double low, double high,
                            double original, double* out, char** err) {
    if (!out) return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: nil output");
    if (rot <= 0 || rot % 2 != 0 || rot > manta::kMaxHeadDim)
        return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: rot must be even, 2 to %d (got %lld)", manta::kMaxHeadDim,
                    (long long)rot);
    if (!(base > 0) || !std::isfinite(base))
        return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: base must be positive");
    if (scaling < MANTA_ROCM_ROTARY_NONE || scaling > MANTA_ROCM_ROTARY_BLEND)
        return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: unknown scaling %d", scaling);
    if (scaling != MANTA_ROCM_ROTARY_NONE && (!(factor > 0) || !std::isfinite(factor)))
        return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: factor must be positive");
    if (scaling == MANTA_ROCM_ROTARY_BLEND && (!(high > low) || !(original > 0)))
        return fail(err, MANTA_ROCM_ERROR, "rotary_freqs: a blend needs high > low and original > 0");
    if (scaling == MANTA_ROCM_ROTARY_BASE && rot > 2) base *= std::pow(factor, (double)rot / (double)(rot - 2));
    for (int64_t p = 0; p < rot / 2; p++) {
        double f = std::pow(base, -2.0 * (double)p / (double)rot);
        if (scaling == MANTA_ROCM_ROTARY_LINEAR) f /= factor;
        if (scaling == MANTA_ROCM_ROTARY_BLEND) {
            const double turns = original * f / (2.0 * M_PI);
            const double g = std::fmin(1.0, std::fmax(0.0, (turns - low) / (high - low)));
            f *= (1.0 - g) / factor + g;
        }
        out[p] = f;
    }
    return MANTA_ROCM_OK;
}

int manta_rocm_rotary_bind(MantaRocm* rt, const double* freqs, int64_t rot, int layout, double magnitude,
                           MantaRocmRotary** out, char** err) {
    if (!out) return fail(err, MANTA_ROCM_ERROR, "nil output");
    *out = nullptr;
    if (!freqs) return fail(err, MANTA_ROCM_ERROR, "rotary_bind: nil frequencies");
    if (rot <= 0 || rot % 2 != 0 || rot > manta::kMaxHeadDim)
        return fail(err, MANTA_ROCM_ERROR, "rotary_bind: rot must be even, 2 to %d (got %lld)", manta::kMaxHeadDim,
                    (long long)rot);
    if (layout != MANTA_ROCM_ROTARY_HALF && layout != MANTA_ROCM_ROTARY_INTERLEAVED)
        return fail(err, MANTA_ROCM_ERROR, "rotary_bind: unknown layout %d", layout);
    if (!std::isfinite(magnitude)) return fail(err, MANTA_ROCM_ERROR, "rotary_bind: magnitude is not finite");
    for (int64_t p = 0; p < rot / 2; p++)
        if (!std::isfinite(freqs[p])) return fail(err, MANTA_ROCM_ERROR, "rotary_bind: frequency %lld is not finite",
                                                  (long long)p);
    int rc = manta_rt::use(rt, err);
    if (rc) return rc;
    double turns[manta::kMaxHeadDim / 2];
    for (int64_t p = 0; p < rot / 2; p++) turns[p] = freqs[p] / (2.0 * M_PI);
    MantaRocmRotary* r = new (std::nothrow) MantaRocmRotary();
    if (!r) return fail(err, MANTA_ROCM_ERROR, "rotary_bind: out of memory");
    hipError_t e = hipMalloc((void**)&r->turns, (size_t)(rot / 2) * sizeof(double));
    if (e == hipSuccess) e = hipMemcpy(r->turns, turns, (size_t)(rot / 2) * sizeof(double), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        r->release();
        delete r;
        return fail(err, MANTA_ROCM_ERROR, "rotary_bind: %s (%s)", hipGetErrorName(e), hipGetErrorString(e));
    }
    r->rt = rt;
    r->rot = (int)rot;
    r->layout = layout;
    r->magnitude = (float)magnitude;
    if (!manta_rt::attach(rt, r)) {
        r->release();
        delete r;
        return fail(err, MANTA_ROCM_ERROR, "rotary_bind: out of memory");
    }
    *out = r;
    return MANTA_ROCM_OK;
}

void manta_rocm_rotary_unbind(MantaRocmRotary* r) {
    if (!r) return;
    if (r->rt) manta_rt::detach(r->rt, r);
    delete r;
}

int manta_rocm_rotary(MantaRocm* rt, const MantaRocmRotary* rot, int dtype, const int32_t* positions_dev,
                      int64_t tokens, int64_t head_dim, const MantaRocmHeads* parts, int64_t nparts, int inverse,
                      char** err) {
    if (!manta::element_type(dtype)) return fail(err, MANTA_ROCM_ERROR, "rotary: unknown element type %d", dtype);
    if (tokens < 0 || tokens > manta::kMaxTokens)
        return fail(err, MANTA_ROCM_ERROR, "rotary: bad token count %lld", (long long)tokens);
    if (nparts < 1 || nparts > manta::kRotaryParts || !parts)
        return fail(err, MANTA_ROCM_ERROR, "rotary: 1 to %d tensors (got %lld)", manta::kRotaryParts,
                    (long long)nparts);
    manta::RotaryArgs a{};
    const int size = element_size(dtype), wide = 16 / size;
    a.wide = 1;
    for (int64_t i = 0; i < nparts; i++) {
        const MantaRocmHeads& h = parts[i];
        if (h.heads <= 0 || h.heads > 65535)
            return fail(err, MANTA_ROCM_ERROR, "rotary: tensor %lld: 1 to 65535 heads (got %lld)", (long long)i,
                        (long long)h.heads);
        if (tokens && (!h.x_dev || !h.out_dev))
            return fail(err, MANTA_ROCM_ERROR, "rotary: tensor %lld: nil pointer", (long long)i);
        const char* bad = manta::check_strides(tokens, h.heads, head_dim, h.x_token, h.x_head);
        if (!bad) bad = manta::check_out_strides(tokens, h.heads, head_dim, h.out_token, h.out_head);
        if (bad) return fail(err, MANTA_ROCM_ERROR, "rotary: tensor %lld: %s", (long long)i, bad);
        if (h.x_dev == h.out_dev && (h.x_token != h.out_token || h.x_head != h.out_head))
            return fail(err, MANTA_ROCM_ERROR, "rotary: tensor %lld: in place needs equal strides", (long long)i);
        a.part[i] = {h.x_dev, h.out_dev, (int)h.heads, h.x_token, h.x_head, h.out_token, h.out_head};
        a.heads += (int)h.heads;
        a.wide = a.wide && aligned16(h.x_dev, h.x_token, h.x_head, size) &&
                 aligned16(h.out_dev, h.out_token, h.out_head, size);
    }
    if (!rot) return fail(err, MANTA_ROCM_ERROR, "rotary: nil frequencies");
    if (head_dim < rot->rot || head_dim > manta::kMaxHeadDim)
        return fail(err, MANTA_ROCM_ERROR, "rotary: head_dim %lld must be %d (the rotated columns) to %d",
                    (long long)head_dim, rot->rot, manta::kMaxHeadDim);
    if (tokens && !positions_dev) return fail(err, MANTA_ROCM_ERROR, "rotary: nil positions");
    if (!rot->rt) return fail(err, MANTA_ROCM_ERROR, "rotary: the frequencies' runtime is destroyed");
    if (rot->rt != rt) return fail(err, MANTA_ROCM_ERROR, "rotary: the frequencies belong to another runtime");
    int rc = manta_rt::use(rt, err);
    if (rc || tokens == 0) return rc;
    a.parts = (int)nparts;
    a.turns = rot->turns;
    a.positions = positions_dev;
    a.tokens = tokens;
    a.head_dim = (int)head_dim;
    a.rot = rot->rot;
    a.interleaved = rot->layout == MANTA_ROCM_ROTARY_INTERLEAVED;
    a.magnitude = rot->magnitude;
    a.inverse = inverse != 0;
    a.dtype = dtype;
    // whole pieces of `wide` pairs and of `wide` copied columns
    a.wide = a.wide && (a.rot / 2) % wide == 0 && (a.head_dim - a.rot) % wide == 0;
    return launch(rt, "rotary", err, [&](hipStream_t s) { return manta::launch_rotary(a, s); });
}

// ------------------------------------------------------------------- cache

int manta_rocm_cache_create(MantaRocm* rt, const MantaRocmCacheShape* shape, MantaRocmCache** out, char** err) {
    if (!out) return fail(err, MANTA_ROCM_ERROR, "nil output");
    *out = nullptr;
    if (!shape) return fail(err, MANTA_ROCM_ERROR, "cache_create: nil shape");
    if (const char* bad = manta::check_cache_shape(*shape)) return fail(err, MANTA_ROCM_ERROR, "cache_create: %s", bad);
    int rc = manta_rt::use(rt, err);
    if (rc) return rc;
    MantaRocmCache* c = new (std::nothrow) MantaRocmCache();
    if (!c) return fail(err, MANTA_ROCM_ERROR, "cache_create: out of memory");
    c->shape = *shape;
    CacheView& v = c->view;
    v.layers = shape->layers;
    v.pages = shape->pages;
    v.page_tokens = (int)shape->page_tokens;
    v.page_shift = __builtin_ctz((unsigned)v.page_tokens);
    v.kv_heads = (int)shape->kv_heads;
    v.head_dim = (int)shape->head_dim;
    v.pitch = (v.head_dim + 31) / 32 * 32;
    v.seqs = (int)shape->seqs;
    v.table_pages = (int)shape->table_pages;
    rc = manta_rt::cache_error_words(rt, &v.err, &v.err_flag, err);
    if (rc) {
        delete c;
        return rc;
    }
    c->max_count = v.layers * v.pages * v.kv_heads;
    c->code_bytes = v.layers * v.pages * v.page_codes();
    c->book_count = v.pages + v.seqs + (int64_t)v.seqs * v.table_pages;
    const size_t max_bytes = ((size_t)c->max_count * 4 + 255) / 256 * 256;
    const size_t book_bytes = ((size_t)c->book_count * 4 + 255) / 256 * 256;
    const size_t scratch = (size_t)(4 * v.pages + 64) * 4;
    hipError_t e = hipMalloc(&c->memory, 2 * ((size_t)c->code_bytes + max_bytes));
    if (e == hipSuccess) e = hipMemset(c->memory, 0, 2 * ((size_t)c->code_bytes + max_bytes));
    const size_t marks = (size_t)v.seqs * 4;
    if (e == hipSuccess) e = hipMalloc(&c->book, book_bytes + scratch + marks);
    // refs and lengths 0, tables -1
    if (e == hipSuccess) e = hipMemset(c->book, 0, (size_t)(v.pages + v.seqs) * 4);
    if (e == hipSuccess)
        e = hipMemset((char*)c->book + (size_t)(v.pages + v.seqs) * 4, 0xFF,
                      book_bytes - (size_t)(v.pages + v.seqs) * 4);
    if (e == hipSuccess) e = hipMemset((char*)c->book + book_bytes + scratch, 0, marks);
    if (e == hipSuccess) e = hipMalloc((void**)&c->partial, kPartialBytes + kAttendTickets * 4);
    if (e == hipSuccess) e = hipMemset((char*)c->partial + kPartialBytes, 0, kAttendTickets * 4);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        c->release();
        delete c;
        return fail(err, MANTA_ROCM_ERROR, "cache_create: %s (%s)", hipGetErrorName(e), hipGetErrorString(e));
    }
    char* m = (char*)c->memory;
    v.k_codes = (int8_t*)m;
    v.v_codes = (int8_t*)(m + c->code_bytes);
    v.k_max = (float*)(m + 2 * c->code_bytes);
    v.v_max = (float*)(m + 2 * c->code_bytes + max_bytes);
    v.refs = (int32_t*)c->book;
    v.lengths = v.refs + v.pages;
    v.tables = v.lengths + v.seqs;
    int32_t* w = (int32_t*)((char*)c->book + book_bytes);
    c->scratch = {w, w + 64, w + 64 + v.pages, w + 64 + 2 * v.pages};
    c->free_list = w + 64 + 3 * v.pages;
    v.refused = (int32_t*)((char*)c->book + book_bytes + scratch);
    c->tickets = (uint32_t*)((char*)c->partial + kPartialBytes);
    c->rt = rt;
    if (!manta_rt::attach(rt, c)) {
        c->release();
        delete c;
        return fail(err, MANTA_ROCM_ERROR, "cache_create: out of memory");
    }
    *out = c;
    return MANTA_ROCM_OK;
}

void manta_rocm_cache_destroy(MantaRocmCache* c) {
    if (!c) return;
    if (c->rt) manta_rt::detach(c->rt, c);
    delete c;
}

int manta_rocm_cache_shape(const MantaRocmCache* c, MantaRocmCacheShape* out) {
    if (!c || !out) return MANTA_ROCM_ERROR;
    *out = c->shape;
    return MANTA_ROCM_OK;
}

int manta_rocm_cache_buffers(const MantaRocmCache* c, MantaRocmCacheBuffers* out) {
    if (!c || !out || !c->rt) return MANTA_ROCM_ERROR;
    const CacheView& v = c->view;
    *out = {v.k_codes, v.v_codes, v.k_max, v.v_max, v.refs, v.pitch, c->code_bytes, c->max_count, c->book_count};
    return MANTA_ROCM_OK;
}

int manta_rocm_cache_extend(MantaRocm* rt, MantaRocmCache* c, const int32_t* seqs, const int32_t* counts, int64_t n,
                            char** err) {
    int rc = check_cache(rt, c, "cache_extend", err);
    if (rc) return rc;
    if (n < 0 || n > c->shape.seqs)
        return fail(err, MANTA_ROCM_ERROR, "cache_extend: bad sequence count %lld", (long long)n);
    if (n == 0) return MANTA_ROCM_OK;
    if (!seqs || !counts) return fail(err, MANTA_ROCM_ERROR, "cache_extend: nil pointer");
    rc = launch(rt, "cache_pages", err, [&](hipStream_t s) {
        return manta::launch_cache_extend(c->view, c->scratch, seqs, counts, (int)n, c->free_list, s);
    });
    if (rc) return rc;
    return launch(rt, "cache_copy", err, [&](hipStream_t s) {
        return manta::launch_cache_copy(c->view, c->scratch.from, c->scratch.to, c->scratch.count, (int)n, nullptr, s);
    });
}

int manta_rocm_cache_fork(MantaRocm* rt, MantaRocmCache* c, const int32_t* parents, const int32_t* children,
                          const int32_t* tokens, int64_t n, char** err) {
    int rc = check_cache(rt, c, "cache_fork", err);
    if (rc) return rc;
    if (n < 0 || n > c->shape.seqs)
        return fail(err, MANTA_ROCM_ERROR, "cache_fork: bad sequence count %lld", (long long)n);
    if (n == 0) return MANTA_ROCM_OK;
    if (!parents || !children) return fail(err, MANTA_ROCM_ERROR, "cache_fork: nil pointer");
    return launch(rt, "cache_pages", err, [&](hipStream_t s) {
        return manta::launch_cache_fork(c->view, parents, children, tokens, (int)n, s);
    });
}

int manta_rocm_cache_release(MantaRocm* rt, MantaRocmCache* c, const int32_t* seqs, const int32_t* keep, int64_t n,
                             char** err) {
    int rc = check_cache(rt, c, "cache_release", err);
    if (rc) return rc;
    if (n < 0 || n > c->shape.seqs)
        return fail(err, MANTA_ROCM_ERROR, "cache_release: bad sequence count %lld", (long long)n);
    if (n == 0) return MANTA_ROCM_OK;
    if (!seqs) return fail(err, MANTA_ROCM_ERROR, "cache_release: nil pointer");
    return launch(rt, "cache_pages", err,
                  [&](hipStream_t s) { return manta::launch_cache_release(c->view, seqs, keep, (int)n, s); });
}

int manta_rocm_cache_compact(MantaRocm* rt, MantaRocmCache* c, int32_t* live, char** err) {
    int rc = check_cache(rt, c, "cache_compact", err);
    if (rc) return rc;
    rc = launch(rt, "cache_pages", err,
                [&](hipStream_t s) { return manta::launch_cache_compact(c->view, c->scratch, live, s); });
    if (rc) return rc;
    return launch(rt, "cache_copy", err, [&](hipStream_t s) {
        return manta::launch_cache_copy(c->view, c->scratch.from, c->scratch.to, c->scratch.count, (int)c->view.pages,
                                        c->scratch.remap, s);
    });
}

int manta_rocm_cache_copy_pages(MantaRocm* rt, MantaRocmCache* c, const int32_t* src, const int32_t* dst, int64_t n,
                                char** err) {
    int rc = check_cache(rt, c, "cache_copy_pages", err);
    if (rc) return rc;
    if (n < 0 || n > c->shape.pages)
        return fail(err, MANTA_ROCM_ERROR, "cache_copy_pages: bad page count %lld", (long long)n);
    if (n == 0) return MANTA_ROCM_OK;
    if (!src || !dst) return fail(err, MANTA_ROCM_ERROR, "cache_copy_pages: nil pointer");
    return launch(rt, "cache_copy", err, [&](hipStream_t s) {
        return manta::launch_cache_copy(c->view, src, dst, nullptr, (int)n, nullptr, s);
    });
}

}  // extern "C"

namespace {

// What append, read and attention check alike.
int check_rows(MantaRocm* rt, const MantaRocmCache* c, const char* what, int64_t layer, const int32_t* offsets,
               const int32_t* seqs, int64_t n, int64_t tokens, char** err) {
    int rc = check_cache(rt, c, what, err);
    if (rc) return rc;
    if (layer < 0 || layer >= c->shape.layers)
        return fail(err, MANTA_ROCM_ERROR, "%s: layer %lld out of range", what, (long long)layer);
    if (const char* bad = manta::check_batch(n, tokens, c->shape.seqs, seqs != nullptr))
        return fail(err, MANTA_ROCM_ERROR, "%s: %s", what, bad);
    if (n > 0 && !offsets) return fail(err, MANTA_ROCM_ERROR, "%s: nil offsets", what);
    return MANTA_ROCM_OK;
}

int kv_rows(const MantaRocmCache* c, const char* what, int dtype, void* k, int64_t k_token, int64_t k_head, void* v,
            int64_t v_token, int64_t v_head, int64_t tokens, bool written, manta::KvRows* out, char** err) {
    if (!manta::element_type(dtype)) return fail(err, MANTA_ROCM_ERROR, "%s: unknown element type %d", what, dtype);
    if (tokens > 0 && (!k || !v)) return fail(err, MANTA_ROCM_ERROR, "%s: nil pointer", what);
    const auto check = written ? manta::check_out_strides : manta::check_strides;
    const char* bad = check(tokens, c->shape.kv_heads, c->shape.head_dim, k_token, k_head);
    if (!bad) bad = check(tokens, c->shape.kv_heads, c->shape.head_dim, v_token, v_head);
    if (bad) return fail(err, MANTA_ROCM_ERROR, "%s: %s", what, bad);
    const int size = element_size(dtype);
    *out = {k, v, k_token, k_head, v_token, v_head, dtype,
            aligned16(k, k_token, k_head, size) && aligned16(v, v_token, v_head, size)};
    return MANTA_ROCM_OK;
}

}  // namespace

extern "C" {

int manta_rocm_cache_append(MantaRocm* rt, MantaRocmCache* c, int64_t layer, int dtype, const void* k, int64_t k_token,
                            int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const int32_t* offsets,
                            const int32_t* seqs, int64_t n, int64_t tokens, char** err) {
    int rc = check_rows(rt, c, "cache_append", layer, offsets, seqs, n, tokens, err);
    if (rc) return rc;
    manta::KvRows x;
    rc = kv_rows(c, "cache_append", dtype, (void*)k, k_token, k_head, (void*)v, v_token, v_head, tokens, false, &x, err);
    if (rc || n == 0 || tokens == 0) return rc;
    const manta::RaggedRows r{offsets, seqs, (int)n, (int)tokens};
    return launch(rt, "cache_append", err,
                  [&](hipStream_t s) { return manta::launch_cache_append(c->view, layer, r, x, s); });
}

int manta_rocm_cache_read(MantaRocm* rt, const MantaRocmCache* c, int64_t layer, int dtype, void* k, int64_t k_token,
                          int64_t k_head, void* v, int64_t v_token, int64_t v_head, const int32_t* offsets,
                          const int32_t* seqs, int64_t n, int64_t tokens, char** err) {
    int rc = check_rows(rt, c, "cache_read", layer, offsets, seqs, n, tokens, err);
    if (rc) return rc;
    manta::KvRows x;
    rc = kv_rows(c, "cache_read", dtype, k, k_token, k_head, v, v_token, v_head, tokens, true, &x, err);
    if (rc || n == 0 || tokens == 0) return rc;
    const manta::RaggedRows r{offsets, seqs, (int)n, (int)tokens};
    return launch(rt, "cache_read", err,
                  [&](hipStream_t s) { return manta::launch_cache_read(c->view, layer, r, x, s); });
}

int manta_rocm_cache_attention(MantaRocm* rt, const MantaRocmCache* c, int64_t layer, int dtype,
                               const MantaRocmHeads* q, float* lse, const int32_t* offsets, const int32_t* seqs,
                               int64_t n, int64_t tokens, double scale, int causal, int64_t window, int64_t longest,
                               char** err) {
    int rc = check_rows(rt, c, "cache_attention", layer, offsets, seqs, n, tokens, err);
    if (rc) return rc;
    if (dtype != MANTA_ROCM_F16 && dtype != MANTA_ROCM_BF16)
        return fail(err, MANTA_ROCM_UNSUPPORTED, "cache_attention: queries must be f16 or bf16");
    if (!q) return fail(err, MANTA_ROCM_ERROR, "cache_attention: nil queries");
    const int64_t d = c->shape.head_dim;
    if (q->heads <= 0 || q->heads % c->shape.kv_heads != 0 || q->heads > 65535)
        return fail(err, MANTA_ROCM_ERROR, "cache_attention: %lld query heads over %lld kv heads", (long long)q->heads,
                    (long long)c->shape.kv_heads);
    if (tokens > 0 && (!q->x_dev || !q->out_dev)) return fail(err, MANTA_ROCM_ERROR, "cache_attention: nil pointer");
    const char* bad = manta::check_strides(tokens, q->heads, d, q->x_token, q->x_head);
    if (!bad) bad = manta::check_out_strides(tokens, q->heads, d, q->out_token, q->out_head);
    if (bad) return fail(err, MANTA_ROCM_ERROR, "cache_attention: %s", bad);
    if (q->x_dev == q->out_dev && (q->x_token != q->out_token || q->x_head != q->out_head))
        return fail(err, MANTA_ROCM_ERROR, "cache_attention: in place needs equal strides");
    if (!std::isfinite(scale)) return fail(err, MANTA_ROCM_ERROR, "cache_attention: scale is not finite");
    if (window < 0 || (window > 0 && !causal))
        return fail(err, MANTA_ROCM_ERROR, "cache_attention: a window must be positive and causal");
    if (longest < 0) return fail(err, MANTA_ROCM_ERROR, "cache_attention: negative length");
    if (tokens * q->heads > ((int64_t)1 << 28))
        return fail(err, MANTA_ROCM_ERROR, "cache_attention: too many rows (%lld tokens of %lld heads)", (long long)tokens,
                    (long long)q->heads);
    if (n == 0 || tokens == 0) return MANTA_ROCM_OK;
    manta::AttendArgs a{};
    a.q = q->x_dev;
    a.out = q->out_dev;
    a.lse = lse;
    a.q_token = q->x_token;
    a.q_head = q->x_head;
    a.o_token = q->out_token;
    a.o_head = q->out_head;
    a.dtype = dtype;
    a.heads = (int)q->heads;
    a.group = (int)(q->heads / c->shape.kv_heads);
    a.scale = (float)(scale * M_LOG2E / 127.0);
    a.causal = causal != 0;
    a.window = window > manta::kMaxInt32 ? 0 : (int)window;
    a.longest = (int)(longest < manta::kMaxInt32 ? longest : manta::kMaxInt32);
    a.wide = aligned16(q->x_dev, q->x_token, q->x_head, 2) && aligned16(q->out_dev, q->out_token, q->out_head, 2);
    a.partial = c->partial;
    a.partial_bytes = (int64_t)kPartialBytes;
    a.tickets = c->tickets;
    a.ntickets = (int64_t)kAttendTickets;
    a.cus = manta_rt::runtime_cus(rt);
    const manta::RaggedRows r{offsets, seqs, (int)n, (int)tokens};
    return launch(rt, "cache_attention", err,
                  [&](hipStream_t s) { return manta::launch_cache_attention(c->view, layer, r, a, s); });
}

int manta_rocm_copy(MantaRocm* rt, void* dst, const void* src, size_t bytes, char** err) {
    int rc = manta_rt::use(rt, err);
    if (rc || bytes == 0) return rc;
    if (!dst || !src) return fail(err, MANTA_ROCM_ERROR, "copy: nil pointer");
    const uintptr_t a = (uintptr_t)dst, b = (uintptr_t)src;
    if (a < b + bytes && b < a + bytes) return fail(err, MANTA_ROCM_ERROR, "copy: the ranges overlap");
    TRY_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToDevice, (hipStream_t)manta_rt::runtime_stream(rt)),
            "hipMemcpyDtoD");
    return MANTA_ROCM_OK;
}

}  // extern "C"
