// kernels_product.hip -- products in 8 bits for gfx950: rows quantised with a
// scale each, times a weight with a scale a column, summed in int32 on
// v_mfma_i32_16x16x64_i8.
#include <atomic>

#include "cache_kernels.hpp"
#include "code_common.hpp"
#include "decode_kernels.hpp"
#include "mq_common.hpp"

#pragma clang fp contract(off)

namespace manta {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- quantise

// A row's codes are (z by) / low, `by` 127 and `low` the row's largest |z|; from
// 2^121 on both are 2^-7 times that, the same quotient of numbers in range.
struct Ratio {
    float by, low;
    __device__ __forceinline__ explicit Ratio(float big)
        : by(big >= 0x1p121f ? 127.0f * 0x1p-7f : 127.0f), low(big >= 0x1p121f ? big * 0x1p-7f : big) {}
    __device__ __forceinline__ int code(float z) const { return (int)__builtin_rintf(__fdiv_rn(z * by, low)); }
};

// One row a workgroup at a time.
template <class E>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantizeArgs a) {
    typedef typename E::T T;
    __shared__ uint32_t tops[kThreads / 64];
    __shared__ double sums[kThreads / 64];
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.x_row;
        uint32_t top = 0;
        double sum = 0.0;
        for (int c = tid; c < a.width; c += kThreads) {
            const float v = E::load(x[c]);
            sum = fma((double)v, (double)v, sum);
            top = max(top, __float_as_uint(a.norm ? v * a.norm[c] : v) & 0x7FFFFFFFu);
        }
        for (int s = 32; s; s >>= 1) {
            top = max(top, (uint32_t)__shfl_xor((int)top, s));
            sum += __shfl_xor(sum, s);
        }
        if ((tid & 63) == 0) {
            tops[tid >> 6] = top;
            sums[tid >> 6] = sum;
        }
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < kThreads / 64; w++) {
            top = max(top, tops[w]);
            sum += sums[w];
        }
        const bool bad = top >= 0x7F800000u;
        const float big = __uint_as_float(top);
        const bool zero = bad || big < 0x1p-126f;
        if (tid == 0) {
            float scale = 0.0f;
            if (bad) scale = __builtin_nanf("");
            else if (!zero) scale = a.norm ? (float)((double)big / 127.0 / sqrt(sum / a.width + a.eps)) : __fdiv_rn(big, 127.0f);
            a.scales[row] = scale;
        }
        const Ratio ratio(big);
        for (int c0 = tid * 16; c0 < a.pitch; c0 += kThreads * 16) {
            uint32_t words[4];
            for (int k = 0; k < 4; k++) {
                uint32_t word = 0;
                for (int j = 0; j < 4; j++) {
                    const int c = c0 + 4 * k + j;
                    int code = 0;
                    if (!zero && c < a.width) {
                        const float v = E::load(x[c]);
                        code = ratio.code(a.norm ? v * a.norm[c] : v);
                    }
                    word |= (uint32_t)(code & 0xFF) << (8 * j);
                }
                words[k] = word;
            }
            *(uint4*)(a.codes + product_at(a.pitch, row, c0)) = make_uint4(words[0], words[1], words[2], words[3]);
        }
        __syncthreads();  // tops and sums have been read
    }
}

// The same results for rows of up to 32768 columns, each read once: 16 columns
// a piece, NP pieces a thread, held in registers from the load until they are
// coded.  Rows may start anywhere (16-byte loads take any alignment of their
// elements).  WAVES waves a row; the rows of a block of 16 are taken on one XCD
// (workgroup i runs on XCD i % 8), whose L2 joins their 16-byte runs into whole
// lines.
template <class E, bool NORM, int WAVES, int NP>
__global__ __launch_bounds__(kThreads) void quantize_wide_kernel(QuantizeArgs a) {
    typedef typename E::T T;
    constexpr int V = E::kWide, L = 16 / V, RPW = kThreads / 64 / WAVES;  // rows of a workgroup
    struct alignas(16) Pack16 {
        T v[V];
    };
    __shared__ uint32_t tops[kThreads / 64];
    __shared__ double sums[kThreads / 64];
    constexpr int PER = 128 / RPW;  // workgroups of 8 blocks of rows
    const int wave = threadIdx.x >> 6, in = blockIdx.x % PER;
    const int64_t block = (int64_t)(blockIdx.x / PER) * 8 + in % 8;
    const int64_t row = block * 16 + in / 8 * RPW + wave / WAVES;
    const bool live = row < a.rows;
    const int tid = threadIdx.x % (64 * WAVES);
    const T* x = (const T*)a.x + (live ? row : 0) * a.x_row;
    Pack16 held[NP][L];
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const int c0 = (tid + 64 * WAVES * p) * 16;
#pragma unroll
        for (int l = 0; l < L; l++) {
            held[p][l] = Pack16{};
            const int c = c0 + l * V;
            if (!live || c >= a.width) continue;
            if (c + V <= a.width) held[p][l] = load16_any<Pack16>(x + c);
            else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (c + j < a.width) held[p][l].v[j] = x[c + j];
            }
        }
    }
    // z of piece p, element e
    float w[NP][NORM ? 16 : 1];
    if (NORM) {
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = (tid + 64 * WAVES * p) * 16 + e;
                if (c + 4 <= a.width) {
                    struct alignas(16) F4 {
                        float v[4];
                    };
                    const F4 f = load16_any<F4>(a.norm + c);
#pragma unroll
                    for (int j = 0; j < 4; j++) w[p][NORM ? e + j : 0] = f.v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) w[p][NORM ? e + j : 0] = c + j < a.width ? a.norm[c + j] : 0.0f;
                }
            }
    }
    auto value = [&](int p, int e) { return E::load(held[p][e / V].v[e % V]); };
    auto z = [&](int p, int e) { return NORM ? value(p, e) * w[p][NORM ? e : 0] : value(p, e); };
    uint32_t top = 0;
    double sum = 0.0;
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (NORM) {
                const double v = (double)value(p, e);
                sum = fma(v, v, sum);
            }
            top = max(top, __float_as_uint(z(p, e)) & 0x7FFFFFFFu);
        }
    for (int s = 32; s; s >>= 1) {
        top = max(top, (uint32_t)__shfl_xor((int)top, s));
        if (NORM) sum += __shfl_xor(sum, s);
    }
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) {
            tops[wave] = top;
            sums[wave] = sum;
        }
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < WAVES; k++) {
            top = max(top, tops[wave / WAVES * WAVES + k]);
            sum += sums[wave / WAVES * WAVES + k];
        }
    }
    if (!live) return;
    const bool bad = top >= 0x7F800000u;
    const float big = __uint_as_float(top);
    const bool zero = bad || big < 0x1p-126f;
    if (tid == 0) {
        float scale = 0.0f;
        if (bad) scale = __builtin_nanf("");
        else if (!zero) scale = NORM ? (float)((double)big / 127.0 / sqrt(sum / a.width + a.eps)) : __fdiv_rn(big, 127.0f);
        a.scales[row] = scale;
    }
    const Ratio ratio(big);
    const float inv = 1.0f / ratio.low;
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const int c0 = (tid + 64 * WAVES * p) * 16;
        if (c0 >= a.pitch) continue;
        uint32_t word[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float t[4];
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = z(p, 4 * k + j) * ratio.by;
            word[k] = zero ? 0 : ratio_codes(t, ratio.low, inv, false);
        }
        *(uint4*)(a.codes + product_at(a.pitch, row, c0)) = make_uint4(word[0], word[1], word[2], word[3]);
    }
}

template <class E, bool NORM>
hipError_t quantize_of(const QuantizeArgs& a, hipStream_t s) {
    const int64_t blocks = (a.rows + 127) / 128;
    // a wave a row up to 1024 columns, a workgroup a row up to 32768
    if (a.width <= 1024) {
        quantize_wide_kernel<E, NORM, 1, 1><<<(unsigned)(blocks * 32), kThreads, 0, s>>>(a);
    } else if (a.width <= 32768 && blocks < (1 << 16)) {
        const dim3 grid((unsigned)(blocks * 128));
        if (a.width <= 4096) quantize_wide_kernel<E, NORM, 4, 1><<<grid, kThreads, 0, s>>>(a);
        else if (a.width <= 8192) quantize_wide_kernel<E, NORM, 4, 2><<<grid, kThreads, 0, s>>>(a);
        else if (a.width <= 16384) quantize_wide_kernel<E, NORM, 4, 4><<<grid, kThreads, 0, s>>>(a);
        else quantize_wide_kernel<E, NORM, 4, 8><<<grid, kThreads, 0, s>>>(a);
    } else {
        quantize_kernel<E><<<(unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20), kThreads, 0, s>>>(a);
    }
    return hipGetLastError();
}

// --------------------------------------------------------- a weight's layout

// A wave lays out blocks: lane l takes 16 of the summed columns of weight row
// l % 16, whose codes lie a row of `columns` apart (16 lanes read 16 bytes of
// each; the caches join the rest).
__global__ __launch_bounds__(kThreads) void weight_layout_kernel(const int8_t* codes, const float* scales, int64_t width,
                                                                 int64_t n, int gated, int64_t steps, int64_t blocks,
                                                                 int8_t* out, float* out_scales) {
    const int lane = threadIdx.x & 63;
    const int64_t columns = gated ? 2 * n : n, waves = (int64_t)gridDim.x * (kThreads / 64);
    for (int64_t b = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); b < blocks * steps; b += waves) {
        // neighbouring waves take neighbouring columns of the same rows
        const int64_t wb = b % blocks, step = b / blocks;
        const int64_t r = wb * 16 + (lane & 15);
        const int64_t c = gated ? (wb >> 1) * 16 + (lane & 15) : r;
        const int64_t from = gated && (wb & 1) ? n + c : c;
        const int64_t k0 = step * 64 + (lane >> 4) * 16;
        uint32_t word[4] = {0, 0, 0, 0};
        if (c < n)
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (k0 + k < width) word[k / 4] |= (uint32_t)(uint8_t)codes[(k0 + k) * columns + from] << (8 * (k % 4));
        *(uint4*)(out + (wb * steps + step) * 1024 + lane * 16) = make_uint4(word[0], word[1], word[2], word[3]);
        if (step == 0 && lane < 16) out_scales[r] = c < n ? scales[from] : 0.0f;
    }
}

// ----------------------------------------------------------------- product

// v times the logistic function of u = v (c0 + c1 v^2): c1 is 0 for silu, and for
// gelu u is twice the argument of its tanh form.  With e = exp(-|u|) that function
// is 1 / (1 + e), or e / (1 + e) below 0.  e is the hardware's 2^t, t = -|u| log2(e)
// in two parts, of which the lower enters as a factor 1 + lower ln 2: within 3 *
// 2^-24 of it (0 below 2^-126; past 200 nothing changes, and infinities stay out
// of the parts); 1 / (1 + e) is the hardware's, within 2^-23.  (expf, a division
// and the polynomial of both, twice the instructions: bf16, 3001 x 4096 x 2 x
// 12288 284 us, 271 so; 10580 x 128 x 2 x 8320 147, 116.)
struct Gate {
    float c0, c1;
    __device__ __forceinline__ explicit Gate(int gate)
        : c0(gate == MANTA_ROCM_GATE_SILU ? 1.0f : 2.0f * 0.7978845608f),
          c1(gate == MANTA_ROCM_GATE_SILU ? 0.0f : 2.0f * 0.7978845608f * 0.044715f) {}
    __device__ __forceinline__ float operator()(float v) const {
        constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0cp-26f;
        const float u = v * fmaf(c1, fminf(v * v, 0x1p127f), c0);  // (no 0 times infinity)
        const float a = -fminf(fabsf(u), 200.0f);
        const float t = a * kLog2e, lower = fmaf(a, kRest, fmaf(a, kLog2e, -t));
        float e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e, lower * 0.6931471806f, e);
        return v * ((u >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e));
    }
};

// Four results of a row, columns c .. c + 3.
template <class E>
__device__ __forceinline__ void store4(const ProductArgs& a, int64_t row, int c, const float* y) {
    typedef typename E::T T;
    typedef typename E::T Four __attribute__((ext_vector_type(4)));
    typedef Four FourAny __attribute__((aligned(sizeof(T))));  // (one access at any alignment)
    T* out = (T*)a.out + row * a.out_row + c;
    const T* add = a.add ? (const T*)a.add + row * a.add_row + c : nullptr;
    if (c + 3 < a.n) {
        Four o, p{};
        if (add) p = *(const FourAny*)add;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = E::store(add ? y[j] + E::load(p[j]) : y[j]);
        *(FourAny*)out = o;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j < a.n) out[j] = E::store(add ? y[j] + E::load(add[j]) : y[j]);
}

// Scales of NT weight blocks from wb on: lane l has those of rows
// 4 (l / 16) + 0 .. 3 of each, as it has their sums (16 x 16 tiles: weight rows
// 4 (l / 16) + 0 .. 3 of token l % 16).
template <int NT>
struct BlockScales {
    float4 v[NT];
    __device__ __forceinline__ BlockScales(const ProductArgs& a, int wb) {
        const int c0 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int t = 0; t < NT; t++) v[t] = *(const float4*)(a.w_scales + min(wb + t, a.w_blocks - 1) * 16 + c0);
    }
    __device__ __forceinline__ void times(int t, float row_scale, v4i sums, float* y) const {
        const float f[4] = {v[t].x, v[t].y, v[t].z, v[t].w};
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (float)sums[j] * (row_scale * f[j]);
    }
};

// The results of NT weight blocks from block wb on for this lane's token
// (row; stored if it is one).  Of 16-bit elements, two blocks' halves change
// places between neighbouring rows of 16 lanes, so that a lane has 8 columns in
// a row and a row of lanes 32 bytes of each token: half as many stores, of whole
// 64-byte pieces where rows are aligned (they need not be).
template <class E, bool GATED, int NT>
struct Added {  // what such a lane adds, asked for ahead
    static constexpr int NR = NT / (GATED ? 2 : 1);  // result blocks
    static constexpr bool kPairs = E::kWide == 8 && NR % 2 == 0;
    struct alignas(8 * sizeof(typename E::T)) Eight {
        typename E::T v[8];
    };
    Eight v[NR / 2 + 1];
    __device__ __forceinline__ void fetch(const ProductArgs& a, int64_t row, int wb) {
        if constexpr (!GATED && kPairs) {
            if (!a.add || row >= a.rows) return;
            const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
            for (int r = 0; r + 1 < NR; r += 2) {
                const int c = (wb + r + (g & 1)) * 16 + (g >> 1) * 8;
                if (c + 8 <= a.n) 
                    v[r / 2] = load16_any<Eight>((const typename E::T*)a.add + row * a.add_row + c);
            }
        }
    }
};
template <class E, bool GATED, int NT>
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t row, float row_scale, int wb,
                                       const BlockScales<NT>& scales, const v4i* sums,
                                       const Added<E, GATED, NT>& added) {
    constexpr int G = GATED ? 2 : 1, NR = NT / G;
    const int g = (threadIdx.x & 63) >> 4;
    const int first = GATED ? wb / 2 : wb, end = GATED ? a.w_blocks / 2 : a.w_blocks;
    const Gate activate(a.gate);
    float y[NR][4];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        scales.times(r * G, row_scale, sums[r * G], y[r]);
        if (GATED) {
            float u[4];
            scales.times(r * G + G - 1, row_scale, sums[r * G + G - 1], u);
#pragma unroll
            for (int j = 0; j < 4; j++) y[r][j] = activate(y[r][j]) * u[j];
        }
    }
    if constexpr (Added<E, GATED, NT>::kPairs) {
        typedef typename E::T T;
        typedef typename Added<E, GATED, NT>::Eight Eight;
#pragma unroll
        for (int r = 0; r < NR; r += 2) {
            float z[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[r][j]), __float_as_uint(y[r + 1][j]),
                                                                false, false);
                z[j] = __uint_as_float(p[0]);
                z[4 + j] = __uint_as_float(p[1]);
            }
            const int c = (first + r + (g & 1)) * 16 + (g >> 1) * 8;
            if (row >= a.rows || first + r + (g & 1) >= end) continue;
            T* out = (T*)a.out + row * a.out_row + c;
            const T* add = a.add ? (const T*)a.add + row * a.add_row + c : nullptr;
            if (c + 8 <= a.n) {
                Eight o;
                const Eight& q = added.v[r / 2];
#pragma unroll
                for (int j = 0; j < 8; j++) o.v[j] = E::store(add ? z[j] + E::load(q.v[j]) : z[j]);
                store16_any(out, o);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < a.n) out[j] = E::store(add ? z[j] + E::load(add[j]) : z[j]);
            }
        }
        return;
    }
    if (row >= a.rows) return;
#pragma unroll
    for (int r = 0; r < NR; r++)
        if (first + r < end) store4<E>(a, row, (first + r) * 16 + 4 * g, y[r]);
}

// Few rows: the weight's bytes are what is read.  A workgroup takes all the
// rows (16 MT at most) and 16 NT weight rows; its waves take U steps of the
// summed columns in turn, read both operands where they lie (16 bytes a lane,
// a block's KB in all) a turn ahead of their use, and join their sums, whole
// numbers, in LDS.
template <class E, bool GATED, int WAVES, int MT, int NT, int U>
__global__ __launch_bounds__(WAVES * 64) void product_few_kernel(ProductArgs a) {
    __shared__ v4i joined[WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wb = blockIdx.x * NT;
    const int64_t blocks = (a.rows + 15) / 16, rb = (int64_t)blockIdx.y * MT;
    const int8_t* xp[MT];
    const int8_t* wp[NT];
#pragma unroll
    for (int m = 0; m < MT; m++) xp[m] = a.x + min(rb + m, blocks - 1) * a.steps * 1024 + lane * 16;
#pragma unroll
    for (int t = 0; t < NT; t++) wp[t] = a.w + (int64_t)min(wb + t, a.w_blocks - 1) * a.steps * 1024 + lane * 16;
    v4i sums[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) sums[m][t] = v4i{0, 0, 0, 0};
    v4i xv[2][U][MT], wv[2][U][NT];
    auto fetch = [&](int k0, int into) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t at = (int64_t)min(k0 + u, a.steps - 1) * 1024;
#pragma unroll
            for (int t = 0; t < NT; t++) wv[into][u][t] = __builtin_nontemporal_load((const v4i*)(wp[t] + at));
#pragma unroll
            for (int m = 0; m < MT; m++) xv[into][u][m] = *(const v4i*)(xp[m] + at);
        }
    };
    auto multiply = [&](int k0, int from) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (k0 + u >= a.steps) break;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++)
                    sums[m][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[from][u][t], xv[from][u][m], sums[m][t], 0, 0, 0);
        }
    };
    constexpr int TURN = WAVES * U;
    fetch(wave * U, 0);
    for (int k = wave * U; k < a.steps; k += 2 * TURN) {
        fetch(k + TURN, 1);
        multiply(k, 0);
        fetch(k + 2 * TURN, 0);
        multiply(k + TURN, 1);
    }
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) joined[wave][m * NT + t][lane] = sums[m][t];
    __syncthreads();
    constexpr int G = GATED ? 2 : 1;  // tiles that finish together
    for (int i = wave; i < MT * NT / G; i += WAVES) {
        const int m = i / (NT / G), t = i % (NT / G) * G;
        v4i all[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            all[g] = joined[0][m * NT + t + g][lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) all[g] += joined[w][m * NT + t + g][lane];
        }
        const int64_t row = (rb + m) * 16 + (lane & 15);
        Added<E, GATED, G> added;
        added.fetch(a, row, wb + t);
        finish<E, GATED, G>(a, row, a.x_scales[min(row, a.rows - 1)], wb + t, BlockScales<G>(a, wb + t), all, added);
    }
}

// Many rows: a workgroup of WM x WN waves takes 16 WM MT tokens and 16 WN NT
// weight rows, a wave MT x NT tiles of 16 x 16.  Blocks of both operands
// stream through LDS, ST stages of SUB steps of the summed columns ahead of the
// products, by direct-to-LDS loads: a block is 1 KB in a row where it lies and
// where it goes, and a wave reads it back 16 bytes a lane in order, so neither
// side has a bank conflict.
//
// 8192 x 4096 x 4096 bf16: 121 to 124 us, 2.2 POP/s (torch's int8 product of that
// size, without scales: 130).  What bounds it: a step's products alone take 54
// of a 256 x 256 tile's 67 us when the whole card works on random codes (the
// clock falls with the matrix cores' load: 43 us on 16 compute units), the
// fill of 32 KB a step about 45 bytes a clock.
template <class E, bool GATED, int WM, int WN, int MT, int NT, int ST, int SUB>
__global__ __launch_bounds__(WM* WN * 64) void product_tile_kernel(
    ProductArgs a, int row_tiles, int w_tiles) {
    constexpr int TM = WM * MT, TN = WN * NT, WAVES = WM * WN;
    constexpr int LPW = (TM + TN) * SUB / WAVES;  // blocks that a wave loads a stage
    static_assert(LPW * WAVES == (TM + TN) * SUB && SUB <= 2, "a stage's blocks split evenly over the waves");
    constexpr int STAGE = (TM + TN) * SUB * 1024;
    const int stages = a.steps / SUB;  // (steps is even)
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroup i runs on XCD i % 8: each XCD takes a run of tiles, in strips
    // of 8 row tiles, so that its 32 workgroups share 8 + 4 tiles' operands in
    // its L2.
    int rt, wt;
    {
        const int total = row_tiles * w_tiles, xcd = blockIdx.x & 7;
        const int t = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
        const int strip = 8 * w_tiles, first = t / strip * 8, rows = min(8, row_tiles - first), in = t % strip;
        rt = first + in % rows;
        wt = in / rows;
    }
    const int64_t x_blocks = (a.rows + 15) / 16;
    const int8_t* src[LPW];
#pragma unroll
    for (int i = 0; i < LPW; i++) {
        const int b = (wave * LPW + i) / SUB;
        // (blocks past the operand read its last one; nothing of theirs is stored)
        const int8_t* p = b < TM ? a.x + min((int64_t)rt * TM + b, x_blocks - 1) * a.steps * 1024
                                 : a.w + (int64_t)min(wt * TN + b - TM, a.w_blocks - 1) * a.steps * 1024;
        src[i] = p + (wave * LPW + i) % SUB * 1024 + lane * 16;
    }
    const uint32_t base = lds_addr(smem) + wave * LPW * 1024;
    auto issue = [&](int k) {
        const uint32_t dst = __builtin_amdgcn_readfirstlane(base + (k % ST) * STAGE);
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            lds_load16(src[i], dst + i * 1024);
            src[i] += SUB * 1024;
        }
    };
#pragma unroll
    for (int k = 0; k < ST; k++)
        if (k < stages) issue(k);
    v4i sums[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) sums[m][t] = v4i{0, 0, 0, 0};
    const int m0 = wave % WM * MT, t0 = wave / WM * NT;  // this wave's blocks of the tile
    v4i wv[2][SUB][NT], xv[2][SUB][MT];
    auto read = [&](int k, int into) {
        const uint8_t* stage = smem + (k % ST) * STAGE + lane * 16;
#pragma unroll
        for (int u = 0; u < SUB; u++) {
#pragma unroll
            for (int t = 0; t < NT; t++) wv[into][u][t] = *(const v4i*)(stage + ((TM + t0 + t) * SUB + u) * 1024);
#pragma unroll
            for (int m = 0; m < MT; m++) xv[into][u][m] = *(const v4i*)(stage + ((m0 + m) * SUB + u) * 1024);
        }
    };
    auto multiply = [&](int from) {
#pragma unroll
        for (int u = 0; u < SUB; u++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++)
                    sums[m][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[from][u][t], xv[from][u][m], sums[m][t], 0, 0, 0);
    };
    // Stage k's products run while stage k + 1's operands come out of LDS.  At
    // the barrier stage k + 1 has arrived and every wave holds stage k, whose
    // place stage k + ST takes.
    auto step = [&](int k, int now) {
        if (k + 1 < stages) {
            mq_wait_barrier<LPW, ST - 2>(stages - 2 - k);
            if (k + ST < stages) issue(k + ST);
            read(k + 1, now ^ 1);
        }
        multiply(now);
    };
    mq_wait_barrier<LPW, ST - 1>(stages - 1);
    read(0, 0);
    for (int k = 0; k < stages; k += 2) {
        step(k, 0);
        if (SUB == 1 || k + 1 < stages) step(k + 1, 1);
    }
    const int64_t row0 = ((int64_t)rt * TM + m0) * 16 + (lane & 15);
    const BlockScales<NT> scales(a, wt * TN + t0);
    float row_scales[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) row_scales[m] = a.x_scales[min(row0 + 16 * m, a.rows - 1)];
    Added<E, GATED, NT> added[2];
    added[0].fetch(a, row0, wt * TN + t0);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        if (m + 1 < MT) added[(m + 1) & 1].fetch(a, row0 + 16 * (m + 1), wt * TN + t0);
        finish<E, GATED, NT>(a, row0 + 16 * m, row_scales[m], wt * TN + t0, scales, sums[m], added[m & 1]);
    }
}

template <class E, bool GATED, int WM, int WN, int MT, int NT, int ST, int SUB>
hipError_t product_tiles(const ProductArgs& a, hipStream_t s) {
    constexpr int TM = WM * MT, TN = WN * NT;
    const size_t lds = (size_t)ST * (TM + TN) * SUB * 1024;
    int device = 0;
    if (const hipError_t e = hipGetDevice(&device)) return e;
    static std::atomic<uint64_t> set{0};  // devices whose kernel may use that much LDS
    if (!(set.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
        const hipError_t e = hipFuncSetAttribute((const void*)product_tile_kernel<E, GATED, WM, WN, MT, NT, ST, SUB>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
        set.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    }
    const int64_t row_tiles = (a.rows + 16 * TM - 1) / (16 * TM), w_tiles = (a.w_blocks + TN - 1) / TN;
    product_tile_kernel<E, GATED, WM, WN, MT, NT, ST, SUB>
        <<<(unsigned)(row_tiles * w_tiles), WM * WN * 64, lds, s>>>(a, (int)row_tiles, (int)w_tiles);
    return hipGetLastError();
}

template <class E, bool GATED, int WAVES, int MT, int NT, int U>
hipError_t product_few(const ProductArgs& a, hipStream_t s) {
    const dim3 grid((a.w_blocks + NT - 1) / NT, (unsigned)((a.rows + 16 * MT - 1) / (16 * MT)));
    product_few_kernel<E, GATED, WAVES, MT, NT, U><<<grid, WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}

// (decode_layout.hpp has the rule)
template <class E, bool GATED>
hipError_t product_of(const ProductArgs& a, hipStream_t s) {
    switch (product_form(a.rows, a.w_blocks, GATED, a.cus)) {
        case kFew16x16:
            if constexpr (!GATED) return product_few<E, GATED, 8, 1, 1, 4>(a, s);
            break;  // (not of gated weights)
        case kFew16x32: return product_few<E, GATED, 8, 1, 2, 2>(a, s);
        case kFew32x32: return product_few<E, GATED, 8, 2, 2, 2>(a, s);
        case kFew64x32: return product_few<E, GATED, 4, 4, 2, 2>(a, s);
        case kTile64Deep: return product_tiles<E, GATED, 2, 2, 2, 2, 4, 2>(a, s);
        case kTile64Row: return product_tiles<E, GATED, 2, 2, 2, 2, 4, 1>(a, s);
        case kTile64: return product_tiles<E, GATED, 2, 2, 2, 2, 2, 2>(a, s);
        case kTile128: return product_tiles<E, GATED, 2, 2, 4, 4, 2, 1>(a, s);
        case kTile256: return product_tiles<E, GATED, 2, 4, 8, 4, 2, 1>(a, s);
    }
    return hipErrorInvalidValue;
}

template <class E>
hipError_t product_type(const ProductArgs& a, hipStream_t s) {
    return a.gate == MANTA_ROCM_GATE_NONE ? product_of<E, false>(a, s) : product_of<E, true>(a, s);
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeArgs& a, hipStream_t s) {
    const bool norm = a.norm != nullptr;
    if (a.dtype == MANTA_ROCM_F32) return norm ? quantize_of<F32, true>(a, s) : quantize_of<F32, false>(a, s);
    if (a.dtype == MANTA_ROCM_F16) return norm ? quantize_of<F16, true>(a, s) : quantize_of<F16, false>(a, s);
    return norm ? quantize_of<Bf16, true>(a, s) : quantize_of<Bf16, false>(a, s);
}

hipError_t launch_weight_layout(const int8_t* codes, const float* scales, int64_t width, int64_t n, bool gated,
                                int8_t* out, float* out_scales, hipStream_t s) {
    const int64_t steps = product_pitch(width) / 64, blocks = weight_rows(n, gated) / 16;
    const int64_t groups = (steps * blocks + kThreads / 64 - 1) / (kThreads / 64);
    weight_layout_kernel<<<(unsigned)(groups < 65536 ? groups : 65536), kThreads, 0, s>>>(codes, scales, width, n, gated,
                                                                                        steps, blocks, out, out_scales);
    return hipGetLastError();
}

hipError_t launch_product(const ProductArgs& a, hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F32) return product_type<F32>(a, s);
    if (a.dtype == MANTA_ROCM_F16) return product_type<F16>(a, s);
    return product_type<Bf16>(a, s);
}

}  // namespace manta
