// decode_layout.hpp -- where quantised rows, bound weights and the parts of
// beams lie, and the checks of the decoding calls' arguments.  Plain C++ (no
// HIP), shared by the kernels, the C ABI and the CPU tests.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "cache_layout.hpp"
#include "manta_decode.h"

namespace manta {

// ---- products in 8 bits ----
// Both operands lie in blocks of 16 rows (tokens or output columns) and 64 of
// the summed columns, 1 KB: four runs of 16 columns, each of them row after
// row.  Lane l of a wave that reads 16 bytes at 16 l has row l % 16, columns
// 16 (l / 16) to + 15: an operand of v_mfma_i32_16x16x64_i8.
constexpr int64_t kMaxWidth = 131072;  // 127 * 128 * 131072 < 2^31
constexpr int64_t kMaxColumns = 1 << 24;
constexpr double kMinEps = 0x1p-126;

MANTA_HD int64_t product_pitch(int64_t width) { return (width + 127) / 128 * 128; }
MANTA_HD int64_t product_rows(int64_t rows) { return (rows + 15) / 16 * 16; }
MANTA_HD int64_t product_at(int64_t pitch, int64_t r, int64_t c) {
    return ((r >> 4) * (pitch >> 6) + (c >> 6)) * 1024 + ((c & 63) >> 4) * 256 + (r & 15) * 16 + (c & 15);
}
// Rows of a bound weight: a gated weight's G and U take turns in blocks of 16,
// so that a wave has both factors of a result.
MANTA_HD int64_t weight_rows(int64_t n, bool gated) { return product_rows(n) * (gated ? 2 : 1); }

// Which kernel and tile (rows x weight rows): figures are bf16, 4096 summed
// columns, us on 256 compute units.
enum ProductForm {
    kFew16x16, kFew16x32, kFew32x32, kFew64x32,  // all the rows of a strip, the summed columns split over waves
    kTile64Deep, kTile64Row, kTile64, kTile128, kTile256,  // tiles through LDS
};
inline ProductForm product_form(int64_t rows, int64_t w_blocks, bool gated, int64_t cus) {
    const int64_t rb = (rows + 15) / 16, wb = w_blocks;
    auto few = [&](int mt, int nt) { return ((rb + mt - 1) / mt) * ((wb + nt - 1) / nt); };
    // The smallest tile that still is a workgroup a compute unit or less: more
    // of them share the reading of the weight, and its latency (32 rows x 4096
    // columns: 16 x 32 tiles 5.9, 32 x 32 7.3; 64 x 4096: 64 x 32 9.1, tiles of
    // 64 x 64 through LDS 14.9)
    if (!gated && few(1, 1) <= cus) return kFew16x16;
    if (few(1, 2) <= cus) return kFew16x32;
    if (few(2, 2) <= cus) return kFew32x32;
    if (few(4, 2) <= cus) return kFew64x32;
    // Up to 32 rows of more columns, where the weight's bytes are all that
    // counts (16 rows x 24576 columns: 16.6, tiles 18.2; 32 rows are even)
    if (rb == 1) return kFew16x32;
    if (rb == 2) return kFew32x32;
    // Tiles of 64 x 64 while those are few: a larger tile of a unit's own takes
    // as long as several of them (512 x 4096: 15.1, 128 x 128 26.9; 1024 x 4096
    // 27.1, 30.8; 512 x 12288 40.2, 37.9)
    const int64_t t64 = ((rows + 63) / 64) * ((wb + 3) / 4), t128 = ((rows + 127) / 128) * ((wb + 7) / 8);
    if (t64 <= 4 * cus) {
        // a tile a unit or less: a deep ring, 128 columns a barrier (589 x 832 of
        // 7936 summed: 19.4, two stages 28.5, four of 64 columns 23.9)
        if (t64 <= cus) return kTile64Deep;
        // one row of tiles reads its weight out of memory, four stages of 64
        // columns (48 rows x 2 x 12288: 18.3, and 19.1 with less LDS)
        if (rb <= 4) return kTile64Row;
        // several a unit wait for each other's data with little LDS each: two
        // stages of 128 (512 x 4096: 15.1, four stages 16.4, of 64 columns 18.3;
        // 1024 x 4096: 27.1, 30.5, 29.6)
        return kTile64;
    }
    // 256 x 256 needs half of the operands' reads of 128 x 128, but comes in
    // whole rounds of a tile a unit, 57 each, against 17.5 a tile for the unit
    // that has most of 128 x 128, and 9 (1024 x 12288: 60.1 and 66.0; 2048 x 4096:
    // 57.7 and 43; 8192 x 4096: 121 and 158; 16384 x 640: 54.8 and 63.8)
    const int64_t t256 = ((rows + 255) / 256) * ((wb + 15) / 16);
    return (t256 + cus - 1) / cus * 13 <= (t128 + cus - 1) / cus * 4 + 2 ? kTile256 : kTile128;
}

inline const char* check_weight(int64_t width, int64_t n, int gate) {
    if (width < 1 || width > kMaxWidth) return "width must be 1 to 131072";
    if (n < 1 || n > kMaxColumns) return "columns must be 1 to 16777216";
    if (gate < MANTA_ROCM_GATE_NONE || gate > MANTA_ROCM_GATE_GELU) return "unknown gate";
    return nullptr;
}
inline const char* check_eps(double eps) {
    return eps >= kMinEps && isfinite((float)eps) ? nullptr : "eps must be at least 2^-126 and finite";
}

// ---- beams ----
constexpr int kMaxBeams = 64, kMaxBest = 64;
constexpr int64_t kMaxBeamRows = 1 << 20;
constexpr int kBeamPiece = 4096;  // logits that a workgroup holds at a time
constexpr int kBeamParts = 64;    // workgroups of a row, at most
// 64-bit words of a part: its best keys, its largest logit, its sum
MANTA_HD int64_t beam_part_words(int64_t best) { return best + 2; }
// Workgroups of a row: 1,024 in all are what the card holds at a time (4 a
// compute unit), and a longer part finds more of its logits below its best ones
// so far.
MANTA_HD int beam_parts(int64_t rows, int64_t vocab) {
    const int64_t pieces = (vocab + kBeamPiece - 1) / kBeamPiece;
    int64_t parts = rows < 1024 ? 1024 / rows : 1;
    parts = parts < pieces ? parts : pieces;
    return (int)(parts < kBeamParts ? parts : kBeamParts);
}
// Parts that any call of up to so many rows has.
MANTA_HD int64_t beam_parts_in_all(int64_t rows) {
    if (rows >= 1024) return rows;
    return rows * kBeamParts < 1024 ? rows * kBeamParts : 1024;
}

inline const char* check_beams(int64_t groups, int64_t beams, int64_t best) {
    if (groups < 0 || beams < 1 || beams > kMaxBeams) return "1 to 64 beams";
    if (best < 1 || best > kMaxBest) return "1 to 64 results a group";
    if (groups > kMaxBeamRows / beams) return "more than 1048576 beams in all";
    return nullptr;
}

// ---- reorder ----
constexpr int64_t kMaxReorder = 4096, kMaxReorderGroup = 1024;
constexpr int kReorderInts = 8192;   // table entries that a workgroup holds
// columns of the tables that a workgroup takes: a power of two
MANTA_HD int reorder_columns(int64_t group) {
    int c = 64;
    while (c > 8 && c * group > kReorderInts) c /= 2;
    return c;
}

}  // namespace manta
