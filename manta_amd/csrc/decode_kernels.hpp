// decode_kernels.hpp -- host-side launchers of the product and beam kernels
// (internal to libmanta_rocm.so; the public surface is
// include/manta_decode.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_layout.hpp"

namespace manta {

struct QuantizeArgs {
    const void* x;
    int64_t x_row;  // elements between rows
    int64_t rows;
    int width, pitch;
    const float* norm;  // [width] or nullptr
    double eps;
    int8_t* codes;
    float* scales;
    int dtype;
};
hipError_t launch_quantize_rows(const QuantizeArgs& a, hipStream_t s);

// codes [width, columns] and their scales as the products read them (columns n,
// or n and n when gated)
hipError_t launch_weight_layout(const int8_t* codes, const float* scales, int64_t width, int64_t n, bool gated,
                                int8_t* out, float* out_scales, hipStream_t s);

struct ProductArgs {
    const int8_t* x;  // quantised rows
    const float* x_scales;
    const int8_t* w;  // weight rows, in the same blocks
    const float* w_scales;  // by weight row
    const void* add;
    void* out;
    int64_t add_row, out_row;
    int64_t rows;
    int n;            // output columns
    int steps;        // blocks of 64 summed columns
    int w_blocks;     // blocks of 16 weight rows
    int dtype, gate;
    int cus;
};
hipError_t launch_product(const ProductArgs& a, hipStream_t s);

struct BeamArgs {
    const void* logits;
    int64_t logits_row;
    int groups, beams, parts, best;
    int64_t vocab;
    const float* scores;
    const int32_t* ended;
    int end_token;
    int32_t* parents;
    int32_t* tokens;
    float* totals;
    int32_t* now_ended;  // or nullptr
    uint64_t* work;     // [groups * beams][parts][beam_part_words(best)]
    uint32_t* tickets;  // [groups], zero between calls
    int dtype;
};
hipError_t launch_beam_select(const BeamArgs& a, hipStream_t s);
hipError_t launch_beam_inputs(const int32_t* tokens, int n, int instead, int32_t* out, hipStream_t s);

}  // namespace manta
