// decode.cpp -- implementation of include/manta_decode.h (but for the calls
// on rotary tables and caches, which are in cache.cpp): argument checks,
// device memory and launches.
#include "manta_decode.h"

#include <hip/hip_runtime.h>

#include <new>

#include "decode_kernels.hpp"
#include "decode_layout.hpp"
#include "launch_common.hpp"
#include "runtime_internal.hpp"

using manta_rt::element_size;
using manta_rt::fail;
using manta_rt::launch;

struct MantaRocmWeight : manta_rt::Attached {
    MantaRocm* rt = nullptr;
    int64_t width = 0, n = 0, pitch = 0;
    int gate = 0;
    void* memory = nullptr;  // codes, then scales
    int8_t* codes = nullptr;
    float* scales = nullptr;
    void release() override {
        if (memory) (void)hipFree(memory);
        memory = nullptr;
        rt = nullptr;
    }
};

struct MantaRocmBeams : manta_rt::Attached {
    MantaRocm* rt = nullptr;
    int64_t groups = 0, beams = 0, best = 0;
    size_t words = 0;
    void* memory = nullptr;  // parts, then tickets
    void release() override {
        if (memory) (void)hipFree(memory);
        memory = nullptr;
        rt = nullptr;
    }
};

namespace {

// Frees what a failed bind has made.
template <class H>
int give_up(H* h, int rc) {
    h->release();
    delete h;
    return rc;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------- products

int manta_rocm_weight_bind(MantaRocm* rt, const int8_t* codes, const float* scales, int64_t width, int64_t n, int gate,
                           MantaRocmWeight** out, char** err) {
    if (!out) return fail(err, MANTA_ROCM_ERROR, "nil output");
    *out = nullptr;
    if (const char* bad = manta::check_weight(width, n, gate)) return fail(err, MANTA_ROCM_ERROR, "weight_bind: %s", bad);
    if (!codes || !scales) return fail(err, MANTA_ROCM_ERROR, "weight_bind: nil pointer");
    int rc = manta_rt::use(rt, err);
    if (rc) return rc;
    const bool gated = gate != MANTA_ROCM_GATE_NONE;
    const int64_t pitch = manta::product_pitch(width), rows = manta::weight_rows(n, gated);
    const size_t bytes = (size_t)pitch * (size_t)rows, tail = (size_t)rows * sizeof(float);
    const int64_t columns = gated ? 2 * n : n;
    MantaRocmWeight* w = new (std::nothrow) MantaRocmWeight();
    if (!w) return fail(err, MANTA_ROCM_ERROR, "weight_bind: out of memory");
    // laid out on the device, from a copy as it came
    const size_t raw = (size_t)width * (size_t)columns, raw_tail = (size_t)columns * sizeof(float);
    const size_t raw_scales = (raw + 255) / 256 * 256;
    void* came = nullptr;
    const hipStream_t s = (hipStream_t)manta_rt::runtime_stream(rt);
    hipError_t e = hipMalloc(&w->memory, bytes + tail);
    if (e == hipSuccess) e = hipMalloc(&came, raw_scales + raw_tail);
    if (e == hipSuccess) e = hipMemcpyAsync(came, codes, raw, hipMemcpyHostToDevice, s);
    if (e == hipSuccess) e = hipMemcpyAsync((char*)came + raw_scales, scales, raw_tail, hipMemcpyHostToDevice, s);
    if (e == hipSuccess)
        e = manta::launch_weight_layout((const int8_t*)came, (const float*)((char*)came + raw_scales), width, n, gated,
                                        (int8_t*)w->memory, (float*)((char*)w->memory + bytes), s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (came) (void)hipFree(came);
    if (e != hipSuccess)
        return give_up(w, fail(err, MANTA_ROCM_ERROR, "weight_bind: %s (%s)", hipGetErrorName(e), hipGetErrorString(e)));
    w->codes = (int8_t*)w->memory;
    w->scales = (float*)((char*)w->memory + bytes);
    w->width = width;
    w->n = n;
    w->pitch = pitch;
    w->gate = gate;
    w->rt = rt;
    if (!manta_rt::attach(rt, w)) return give_up(w, fail(err, MANTA_ROCM_ERROR, "weight_bind: out of memory"));
    *out = w;
    return MANTA_ROCM_OK;
}

void manta_rocm_weight_unbind(MantaRocmWeight* w) {
    if (!w) return;
    if (w->rt) manta_rt::detach(w->rt, w);
    delete w;
}

int64_t manta_rocm_quantized_bytes(int64_t rows, int64_t width) {
    if (rows < 0 || rows > manta::kMaxTokens || width < 1 || width > manta::kMaxWidth) return -1;
    return manta::product_rows(rows) * manta::product_pitch(width);
}

int manta_rocm_quantize_rows(MantaRocm* rt, int dtype, const void* x, int64_t x_row, int64_t rows, int64_t width,
                             const float* norm, double eps, int8_t* codes, float* scales, char** err) {
    if (!manta::element_type(dtype)) return fail(err, MANTA_ROCM_ERROR, "quantize_rows: unknown element type %d", dtype);
    if (manta_rocm_quantized_bytes(rows, width) < 0)
        return fail(err, MANTA_ROCM_ERROR, "quantize_rows: bad shape [%lld, %lld]", (long long)rows, (long long)width);
    if (x_row < 0 || (rows > 1 && x_row < width))
        return fail(err, MANTA_ROCM_ERROR, "quantize_rows: rows of %lld columns are %lld elements apart",
                    (long long)width, (long long)x_row);
    if (norm)
        if (const char* bad = manta::check_eps(eps)) return fail(err, MANTA_ROCM_ERROR, "quantize_rows: %s", bad);
    if (rows > 0 && (!x || !codes || !scales)) return fail(err, MANTA_ROCM_ERROR, "quantize_rows: nil pointer");
    if ((uintptr_t)codes % 16 != 0) return fail(err, MANTA_ROCM_ERROR, "quantize_rows: codes must start on 16 bytes");
    if ((uintptr_t)x % element_size(dtype) != 0)
        return fail(err, MANTA_ROCM_ERROR, "quantize_rows: rows are not aligned to their elements");
    int rc = manta_rt::use(rt, err);
    if (rc || rows == 0) return rc;
    manta::QuantizeArgs a{};
    a.x = x;
    a.x_row = x_row;
    a.rows = rows;
    a.width = (int)width;
    a.pitch = (int)manta::product_pitch(width);
    a.norm = norm;
    a.eps = eps;
    a.codes = codes;
    a.scales = scales;
    a.dtype = dtype;
    return launch(rt, "quantize_rows", err, [&](hipStream_t s) { return manta::launch_quantize_rows(a, s); });
}

int manta_rocm_matmul_q8(MantaRocm* rt, const MantaRocmWeight* w, const int8_t* codes, const float* scales,
                         int64_t rows, int dtype, const void* add, int64_t add_row, void* out, int64_t out_row,
                         char** err) {
    if (!w) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: nil weight");
    if (!w->rt) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: the weight's runtime is destroyed");
    if (w->rt != rt) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: the weight belongs to another runtime");
    if (!manta::element_type(dtype)) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: unknown element type %d", dtype);
    if (rows < 0 || rows > manta::kMaxTokens)
        return fail(err, MANTA_ROCM_ERROR, "matmul_q8: bad row count %lld", (long long)rows);
    if (rows > 0 && (!codes || !scales || !out)) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: nil pointer");
    if ((uintptr_t)codes % 16 != 0) return fail(err, MANTA_ROCM_ERROR, "matmul_q8: codes must start on 16 bytes");
    if (out_row < 0 || add_row < 0 || (rows > 1 && (out_row < w->n || (add && add_row < w->n))))
        return fail(err, MANTA_ROCM_ERROR, "matmul_q8: rows of %lld columns are %lld and %lld elements apart",
                    (long long)w->n, (long long)out_row, (long long)add_row);
    if ((uintptr_t)out % element_size(dtype) != 0 || (uintptr_t)add % element_size(dtype) != 0)
        return fail(err, MANTA_ROCM_ERROR, "matmul_q8: results are not aligned to their elements");
    if (add && w->gate != MANTA_ROCM_GATE_NONE)
        return fail(err, MANTA_ROCM_ERROR, "matmul_q8: nothing is added to a gated product");
    if (add && add == out && rows > 1 && add_row != out_row)
        return fail(err, MANTA_ROCM_ERROR, "matmul_q8: in place needs equal strides");
    int rc = manta_rt::use(rt, err);
    if (rc || rows == 0) return rc;
    manta::ProductArgs a{};
    a.x = codes;
    a.x_scales = scales;
    a.w = w->codes;
    a.w_scales = w->scales;
    a.add = add;
    a.out = out;
    a.add_row = add_row;
    a.out_row = out_row;
    a.rows = rows;
    a.n = (int)w->n;
    a.steps = (int)(w->pitch / 64);
    a.w_blocks = (int)(manta::weight_rows(w->n, w->gate != MANTA_ROCM_GATE_NONE) / 16);
    a.dtype = dtype;
    a.gate = w->gate;
    a.cus = manta_rt::runtime_cus(rt);
    return launch(rt, "matmul_q8", err, [&](hipStream_t s) { return manta::launch_product(a, s); });
}

// ------------------------------------------------------------------- beams

int manta_rocm_beams_create(MantaRocm* rt, int64_t groups, int64_t beams, int64_t best, MantaRocmBeams** out,
                            char** err) {
    if (!out) return fail(err, MANTA_ROCM_ERROR, "nil output");
    *out = nullptr;
    if (const char* bad = manta::check_beams(groups, beams, best))
        return fail(err, MANTA_ROCM_ERROR, "beams_create: %s", bad);
    if (groups < 1) return fail(err, MANTA_ROCM_ERROR, "beams_create: no groups");
    int rc = manta_rt::use(rt, err);
    if (rc) return rc;
    MantaRocmBeams* b = new (std::nothrow) MantaRocmBeams();
    if (!b) return fail(err, MANTA_ROCM_ERROR, "beams_create: out of memory");
    b->groups = groups;
    b->beams = beams;
    b->best = best;
    b->words = (size_t)(manta::beam_parts_in_all(groups * beams) * manta::beam_part_words(best));
    hipError_t e = hipMalloc(&b->memory, b->words * 8 + (size_t)groups * 4);
    if (e == hipSuccess) e = hipMemset((char*)b->memory + b->words * 8, 0, (size_t)groups * 4);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess)
        return give_up(b, fail(err, MANTA_ROCM_ERROR, "beams_create: %s (%s)", hipGetErrorName(e), hipGetErrorString(e)));
    b->rt = rt;
    if (!manta_rt::attach(rt, b)) return give_up(b, fail(err, MANTA_ROCM_ERROR, "beams_create: out of memory"));
    *out = b;
    return MANTA_ROCM_OK;
}

void manta_rocm_beams_destroy(MantaRocmBeams* b) {
    if (!b) return;
    if (b->rt) manta_rt::detach(b->rt, b);
    delete b;
}

int manta_rocm_beam_select(MantaRocm* rt, MantaRocmBeams* b, int dtype, const void* logits, int64_t logits_row,
                           int64_t groups, int64_t beams, int64_t vocab, const float* scores, const int32_t* ended,
                           int64_t end_token, int64_t best, int32_t* parents, int32_t* tokens, float* totals,
                           int32_t* now_ended, char** err) {
    if (!b) return fail(err, MANTA_ROCM_ERROR, "beam_select: nil beams");
    if (!b->rt) return fail(err, MANTA_ROCM_ERROR, "beam_select: the beams' runtime is destroyed");
    if (b->rt != rt) return fail(err, MANTA_ROCM_ERROR, "beam_select: the beams belong to another runtime");
    if (!manta::element_type(dtype)) return fail(err, MANTA_ROCM_ERROR, "beam_select: unknown element type %d", dtype);
    if (const char* bad = manta::check_beams(groups, beams, best))
        return fail(err, MANTA_ROCM_ERROR, "beam_select: %s", bad);
    if (groups > b->groups || beams > b->beams || best > b->best)
        return fail(err, MANTA_ROCM_ERROR, "beam_select: %lld groups of %lld beams, %lld results: made for %lld, %lld, %lld",
                    (long long)groups, (long long)beams, (long long)best, (long long)b->groups, (long long)b->beams,
                    (long long)b->best);
    if (vocab < 1 || vocab > manta::kMaxInt32 - 16)
        return fail(err, MANTA_ROCM_ERROR, "beam_select: bad vocabulary %lld", (long long)vocab);
    if (logits_row < 0 || (groups * beams > 1 && logits_row < vocab))
        return fail(err, MANTA_ROCM_ERROR, "beam_select: rows of %lld logits are %lld elements apart", (long long)vocab,
                    (long long)logits_row);
    if ((ended || now_ended) && (end_token < 0 || end_token >= vocab))
        return fail(err, MANTA_ROCM_ERROR, "beam_select: end token %lld of %lld", (long long)end_token, (long long)vocab);
    if (groups > 0 && (!logits || !scores || !parents || !tokens || !totals))
        return fail(err, MANTA_ROCM_ERROR, "beam_select: nil pointer");
    if (best != beams && groups > 0 && (totals == scores || (ended && now_ended == ended)))
        return fail(err, MANTA_ROCM_ERROR, "beam_select: in place needs as many results as beams (%lld, %lld)",
                    (long long)best, (long long)beams);
    if ((uintptr_t)logits % element_size(dtype) != 0)
        return fail(err, MANTA_ROCM_ERROR, "beam_select: logits are not aligned to their elements");
    int rc = manta_rt::use(rt, err);
    if (rc || groups == 0) return rc;
    manta::BeamArgs a{};
    a.logits = logits;
    a.logits_row = logits_row;
    a.groups = (int)groups;
    a.beams = (int)beams;
    a.parts = manta::beam_parts(groups * beams, vocab);
    a.best = (int)best;
    a.vocab = vocab;
    a.scores = scores;
    a.ended = ended;
    a.end_token = (int)end_token;
    a.parents = parents;
    a.tokens = tokens;
    a.totals = totals;
    a.now_ended = now_ended;
    a.work = (uint64_t*)b->memory;
    a.tickets = (uint32_t*)((char*)b->memory + b->words * 8);
    a.dtype = dtype;
    return launch(rt, "beam_select", err, [&](hipStream_t s) { return manta::launch_beam_select(a, s); });
}

int manta_rocm_beam_inputs(MantaRocm* rt, const int32_t* tokens, int64_t n, int64_t instead, int32_t* out, char** err) {
    if (n < 0 || n > manta::kMaxTokens) return fail(err, MANTA_ROCM_ERROR, "beam_inputs: bad token count %lld", (long long)n);
    if (instead < 0 || instead > manta::kMaxInt32)
        return fail(err, MANTA_ROCM_ERROR, "beam_inputs: token %lld", (long long)instead);
    if (n > 0 && (!tokens || !out)) return fail(err, MANTA_ROCM_ERROR, "beam_inputs: nil pointer");
    int rc = manta_rt::use(rt, err);
    if (rc || n == 0) return rc;
    return launch(rt, "beam_inputs", err, [&](hipStream_t s) {
        return manta::launch_beam_inputs(tokens, (int)n, (int)instead, out, s);
    });
}

}  // extern "C"
