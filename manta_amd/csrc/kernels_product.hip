// kernels_product.hip -- products in 8 bits for gfx950: rows quantised with a
// scale each, times a weight with a scale a column, summed in int32 on
// v_mfma_i32_16x16x64_i8.
#include "cache_kernels.hpp"
#include "decode_kernels.hpp"

#pragma clang fp contract(off)

namespace manta {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256;

// ---------------------------------------------------------------- quantise

__device__ __forceinline__ int row_code(float z, float max) {
    const float r = __builtin_rintf(__fdiv_rn(z * 127.0f, max));
    return (int)fminf(127.0f, fmaxf(-127.0f, r));
}

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
        for (int c0 = tid * 16; c0 < a.pitch; c0 += kThreads * 16) {
            uint32_t words[4];
            for (int k = 0; k < 4; k++) {
                uint32_t word = 0;
                for (int j = 0; j < 4; j++) {
                    const int c = c0 + 4 * k + j;
                    int code = 0;
                    if (!zero && c < a.width) {
                        const float v = E::load(x[c]);
                        code = row_code(a.norm ? v * a.norm[c] : v, big);
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

// ----------------------------------------------------------------- product

__device__ __forceinline__ float activate(float v, int gate) {
    // silu v / (1 + exp(-v)); gelu likewise, its tanh form being v times the
    // logistic function of 2 u
    const float u = gate == MANTA_ROCM_GATE_SILU ? v : 2.0f * 0.7978845608f * (v + 0.044715f * (v * v * v));
    return v / (1.0f + expf(-u));
}

// Four results of a row, columns c .. c + 3.
template <class E>
__device__ __forceinline__ void store4(const ProductArgs& a, int64_t row, int c, const float* y) {
    typedef typename E::T T;
    struct alignas(4 * sizeof(T)) Four {
        T v[4];
    };
    T* out = (T*)a.out + row * a.out_row + c;
    const T* add = a.add ? (const T*)a.add + row * a.add_row + c : nullptr;
    if (a.wide && c + 3 < a.n) {
        Four o, p{};
        if (add) p = *(const Four*)add;
#pragma unroll
        for (int j = 0; j < 4; j++) o.v[j] = E::store(add ? y[j] + E::load(p.v[j]) : y[j]);
        *(Four*)out = o;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j < a.n) out[j] = E::store(add ? y[j] + E::load(add[j]) : y[j]);
}

// A 16 x 16 tile of sums: lane l has weight rows 16 wb + 4 (l / 16) + 0 .. 3
// of token l % 16.
__device__ __forceinline__ void scaled(const ProductArgs& a, int wb, float row_scale, v4i sums, float* y) {
    const float4 t = *(const float4*)(a.w_scales + wb * 16 + 4 * ((threadIdx.x & 63) >> 4));
    const float f[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = (float)sums[j] * (row_scale * f[j]);
}

// The results of NT weight blocks from block wb on for the token of this
// lane (row, in range).
template <class E, bool GATED, int NT>
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t row, int wb, const v4i* sums) {
    const float scale = a.x_scales[row];
    const int c0 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int t = 0; t < NT; t += GATED ? 2 : 1) {
        if (wb + t >= a.w_blocks) break;
        float y[4];
        scaled(a, wb + t, scale, sums[t], y);
        if (GATED) {
            float u[4];
            scaled(a, wb + t + 1, scale, sums[t + (GATED ? 1 : 0)], u);
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = activate(y[j], a.gate) * u[j];
        }
        store4<E>(a, row, (GATED ? (wb + t) / 2 : wb + t) * 16 + c0, y);
    }
}

// A wave takes 16 MT tokens and 16 NT weight rows and reads both operands
// where they lie: each is 16 bytes a lane, a block's KB in all.
template <class E, bool GATED, int MT, int NT>
__global__ __launch_bounds__(kThreads) void product_kernel(ProductArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wb = (blockIdx.x * (kThreads / 64) + wave) * NT;
    if (wb >= a.w_blocks) return;
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
    for (int k = 0; k < a.steps; k++) {
        v4i xv[MT], wv[NT];
#pragma unroll
        for (int m = 0; m < MT; m++) xv[m] = *(const v4i*)(xp[m] + (int64_t)k * 1024);
#pragma unroll
        for (int t = 0; t < NT; t++) wv[t] = *(const v4i*)(wp[t] + (int64_t)k * 1024);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < NT; t++) sums[m][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[t], xv[m], sums[m][t], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int64_t row = (rb + m) * 16 + (lane & 15);
        if (row < a.rows) finish<E, GATED, NT>(a, row, wb, sums[m]);
    }
}

template <class E, bool GATED>
hipError_t product_of(const ProductArgs& a, hipStream_t s) {
    constexpr int MT = 4, NT = 4;
    const int64_t row_tiles = ((a.rows + 15) / 16 + MT - 1) / MT;
    for (int64_t r0 = 0; r0 < row_tiles; r0 += 32768) {  // (a grid's second axis is 16 bits)
        ProductArgs p = a;
        const int64_t first = r0 * MT * 16;
        p.x += first * a.steps * 64;
        p.x_scales += first;
        p.rows = a.rows - first;
        p.out = (typename E::T*)a.out + first * a.out_row;
        if (a.add) p.add = (const typename E::T*)a.add + first * a.add_row;
        const dim3 grid((a.w_blocks + 4 * NT - 1) / (4 * NT), (unsigned)(row_tiles - r0 < 32768 ? row_tiles - r0 : 32768));
        product_kernel<E, GATED, MT, NT><<<grid, kThreads, 0, s>>>(p);
    }
    return hipGetLastError();
}

template <class E>
hipError_t product_type(const ProductArgs& a, hipStream_t s) {
    return a.gate == MANTA_ROCM_GATE_NONE ? product_of<E, false>(a, s) : product_of<E, true>(a, s);
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20));
    if (a.dtype == MANTA_ROCM_F32) quantize_kernel<F32><<<grid, kThreads, 0, s>>>(a);
    else if (a.dtype == MANTA_ROCM_F16) quantize_kernel<F16><<<grid, kThreads, 0, s>>>(a);
    else quantize_kernel<Bf16><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_product(const ProductArgs& a, hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F32) return product_type<F32>(a, s);
    if (a.dtype == MANTA_ROCM_F16) return product_type<F16>(a, s);
    return product_type<Bf16>(a, s);
}

}  // namespace manta
