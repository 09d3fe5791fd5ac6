// kernels_rotary.hip -- rotary positions for gfx950.
//
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
//   a = 2 pi * position * turns[p]
//
// per token, head and pair p; the gradient is the same with -a.  Bytes bound:
// each element is read and written once.  The angles of a token are shared by
// its heads: a workgroup takes one token and some of its heads, works the
// rot/2 (cos, sin) out once into LDS and streams the heads past them in
// 16-byte pieces (8192 tokens of 40 heads of 128, bf16: 33.6 us, 5.0 TB/s; a
// copy reaches 4.75).  The turns are reduced to [-1/2, 1/2] in f64: at position
// 10^6 an f32 product is off by 0.06 radians, the f64 one by 1e-10.
#include "cache_kernels.hpp"

namespace manta {

namespace {

constexpr int kThreads = 256;

template <class E, int V>
struct alignas(sizeof(typename E::T) * V) Pack {
    typename E::T v[V];
};

// V elements at once: V pairs of a head, or V columns past the rotated ones.
template <class E, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
    typedef typename E::T T;
    __shared__ float cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
    const int half = a.rot >> 1;
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        __syncthreads();  // an earlier token's angles have been used
        const double pos = (double)a.positions[token];
        for (int p = threadIdx.x; p < half; p += kThreads) {
            const double t = pos * a.turns[p];
            const float r = (float)(t - rint(t));
            float s, c;
            sincospif(2.0f * r, &s, &c);
            cs[p] = a.magnitude * c;
            sn[p] = a.inverse ? -(a.magnitude * s) : a.magnitude * s;
        }
        __syncthreads();
        const int turned = half / V;                     // pieces of V pairs
        const int rest = (a.head_dim - a.rot) / V;       // pieces of V copied columns
        const int pieces = turned + rest;
        const int per = (a.heads + gridDim.y - 1) / gridDim.y;
        const int h0 = blockIdx.y * per, h1 = min(a.heads, h0 + per);
        for (int i = threadIdx.x; i < (h1 - h0) * pieces; i += kThreads) {
            int h = h0 + i / pieces;
            const int piece = i % pieces;
            int k = 0;
            while (h >= a.part[k].heads) h -= a.part[k++].heads;
            const RotaryPart& q = a.part[k];
            const T* x = (const T*)q.x + token * q.x_token + h * q.x_head;
            T* y = (T*)q.out + token * q.out_token + h * q.out_head;
            if (piece >= turned) {
                const int at = a.rot + (piece - turned) * V;
                if (x != y) *(Pack<E, V>*)(y + at) = *(const Pack<E, V>*)(x + at);
                continue;
            }
            const int p = piece * V;
            Pack<E, V> lo, hi;
            if (INTERLEAVED) {
                lo = *(const Pack<E, V>*)(x + 2 * p);
                hi = *(const Pack<E, V>*)(x + 2 * p + V);
            } else {
                lo = *(const Pack<E, V>*)(x + p);
                hi = *(const Pack<E, V>*)(x + half + p);
            }
            Pack<E, V> ylo, yhi;
#pragma unroll
            for (int j = 0; j < V; j++) {
                // element j of the first halves' and of the second halves' run
                const int e = 2 * j;
                const T t1 = !INTERLEAVED ? lo.v[j] : e < V ? lo.v[e % V] : hi.v[e % V];
                const T t2 = !INTERLEAVED ? hi.v[j] : e + 1 < V ? lo.v[(e + 1) % V] : hi.v[(e + 1) % V];
                const float x1 = E::load(t1), x2 = E::load(t2), c = cs[p + j], s = sn[p + j];
                const T y1 = E::store(x1 * c - x2 * s), y2 = E::store(x2 * c + x1 * s);
                if (!INTERLEAVED) {
                    ylo.v[j] = y1;
                    yhi.v[j] = y2;
                } else {
                    (e < V ? ylo : yhi).v[e % V] = y1;
                    (e + 1 < V ? ylo : yhi).v[(e + 1) % V] = y2;
                }
            }
            if (INTERLEAVED) {
                *(Pack<E, V>*)(y + 2 * p) = ylo;
                *(Pack<E, V>*)(y + 2 * p + V) = yhi;
            } else {
                *(Pack<E, V>*)(y + p) = ylo;
                *(Pack<E, V>*)(y + half + p) = yhi;
            }
        }
    }
}

// The same of heads that are RMS normed first: y = rotate(x r w), r = 1 /
// sqrt(mean(x^2) + eps).  `lanes` (a power of two) lanes hold a head, NP
// pieces each, from its load to its store, so a head is read once and its sum
// of squares is one exchange among them.  Sums of squares are f64: no number
// of f32 leaves its range.
template <class E, int V, bool INTERLEAVED, int NP>
__global__ __launch_bounds__(kThreads) void rotary_normed_kernel(RotaryArgs a, RotaryNorms n, int lanes) {
    typedef typename E::T T;
    __shared__ float cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
    const int half = a.rot >> 1;
    const int turned = half / V;                // pieces of V pairs
    const int rest = (a.head_dim - a.rot) / V;  // pieces of V columns past them
    const int pieces = turned + rest;
    const int per = (a.heads + gridDim.y - 1) / gridDim.y;
    const int h0 = blockIdx.y * per, h1 = min(a.heads, h0 + per);
    const int gl = threadIdx.x & (lanes - 1), g0 = threadIdx.x / lanes, step = kThreads / lanes;
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        __syncthreads();  // an earlier token's angles have been used
        const double pos = (double)a.positions[token];
        for (int p = threadIdx.x; p < half; p += kThreads) {
            const double t = pos * a.turns[p];
            const float r = (float)(t - rint(t));
            float s, c;
            sincospif(2.0f * r, &s, &c);
            cs[p] = a.magnitude * c;
            sn[p] = a.magnitude * s;
        }
        __syncthreads();
        for (int hb = h0; hb < h1; hb += step) {  // (all lanes stay for the exchange)
            int h = hb + g0;
            const bool live = h < h1;
            int k = 0;
            if (live)
                while (h >= a.part[k].heads) h -= a.part[k++].heads;
            const RotaryPart& q = a.part[k];
            const float* w = n.weight[k];
            const T* x = (const T*)q.x + token * q.x_token + h * q.x_head;
            T* y = (T*)q.out + token * q.out_token + h * q.out_head;
            Pack<E, V> lo[NP], hi[NP];
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int piece = gl + lanes * i;
                lo[i] = Pack<E, V>{};
                hi[i] = Pack<E, V>{};
                if (live && piece < turned) {
                    const int p = piece * V;
                    lo[i] = *(const Pack<E, V>*)(x + (INTERLEAVED ? 2 * p : p));
                    hi[i] = *(const Pack<E, V>*)(x + (INTERLEAVED ? 2 * p + V : half + p));
                } else if (live && piece < pieces) {
                    lo[i] = *(const Pack<E, V>*)(x + a.rot + (piece - turned) * V);
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const double u = E::load(lo[i].v[j]), v = E::load(hi[i].v[j]);
                    sum = fma(u, u, sum);
                    sum = fma(v, v, sum);
                }
            }
            for (int s = lanes >> 1; s; s >>= 1) sum += __shfl_xor(sum, s);
            if (!live) continue;
            const float r = w ? (float)(1.0 / sqrt(sum / a.head_dim + n.eps)) : 1.0f;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int piece = gl + lanes * i;
                if (piece >= pieces) continue;
                if (piece >= turned) {
                    const int at = a.rot + (piece - turned) * V;
                    Pack<E, V> o;
#pragma unroll
                    for (int j = 0; j < V; j++)
                        o.v[j] = w ? E::store(E::load(lo[i].v[j]) * r * w[at + j]) : lo[i].v[j];
                    *(Pack<E, V>*)(y + at) = o;
                    continue;
                }
                const int p = piece * V;
                // the run of columns that lo holds, and hi
                const int at0 = INTERLEAVED ? 2 * p : p, at1 = INTERLEAVED ? 2 * p + V : half + p;
                float u[2 * V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    u[j] = E::load(lo[i].v[j]);
                    u[V + j] = E::load(hi[i].v[j]);
                    if (w) {
                        u[j] = u[j] * r * w[at0 + j];
                        u[V + j] = u[V + j] * r * w[at1 + j];
                    }
                }
                T o[2 * V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    // pair p + j: elements 2j and 2j + 1 of the run, or j of each half
                    const int e1 = INTERLEAVED ? 2 * j : j, e2 = INTERLEAVED ? 2 * j + 1 : V + j;
                    const float c = cs[p + j], s = sn[p + j];
                    o[e1] = E::store(u[e1] * c - u[e2] * s);
                    o[e2] = E::store(u[e2] * c + u[e1] * s);
                }
                Pack<E, V> ylo, yhi;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    ylo.v[j] = o[j];
                    yhi.v[j] = o[V + j];
                }
                *(Pack<E, V>*)(y + at0) = ylo;
                *(Pack<E, V>*)(y + at1) = yhi;
            }
        }
    }
}

template <class E>
hipError_t launch_normed(const RotaryArgs& a, const RotaryNorms& n, hipStream_t s) {
    int split = 1;
    while (split < 8 && split * 2 <= a.heads && a.tokens * split < 512) split *= 2;
    const dim3 grid((unsigned)(a.tokens < (1 << 20) ? a.tokens : 1 << 20), split);
    const int v = a.wide ? E::kWide : 1;
    const int pieces = (a.rot / 2 + a.head_dim - a.rot) / v;
    int lanes = 1;
    while (lanes < pieces && lanes < 64) lanes *= 2;  // pieces <= 255, <= 64 when wide
    if (a.wide) {
        if (a.interleaved) rotary_normed_kernel<E, E::kWide, true, 1><<<grid, kThreads, 0, s>>>(a, n, lanes);
        else rotary_normed_kernel<E, E::kWide, false, 1><<<grid, kThreads, 0, s>>>(a, n, lanes);
    } else {
        if (a.interleaved) rotary_normed_kernel<E, 1, true, 4><<<grid, kThreads, 0, s>>>(a, n, lanes);
        else rotary_normed_kernel<E, 1, false, 4><<<grid, kThreads, 0, s>>>(a, n, lanes);
    }
    return hipGetLastError();
}

template <class E>
hipError_t launch(const RotaryArgs& a, hipStream_t s) {
    // few tokens: a token's heads over several workgroups, so that the card
    // is full
    int split = 1;
    while (split < 8 && split * 2 <= a.heads && a.tokens * split < 512) split *= 2;
    const dim3 grid((unsigned)(a.tokens < (1 << 20) ? a.tokens : 1 << 20), split);
    if (a.wide) {
        if (a.interleaved) rotary_kernel<E, E::kWide, true><<<grid, kThreads, 0, s>>>(a);
        else rotary_kernel<E, E::kWide, false><<<grid, kThreads, 0, s>>>(a);
    } else {
        if (a.interleaved) rotary_kernel<E, 1, true><<<grid, kThreads, 0, s>>>(a);
        else rotary_kernel<E, 1, false><<<grid, kThreads, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F32) return launch<F32>(a, s);
    if (a.dtype == MANTA_ROCM_F16) return launch<F16>(a, s);
    return launch<Bf16>(a, s);
}

hipError_t launch_rotary_normed(const RotaryArgs& a, const RotaryNorms& n, hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F32) return launch_normed<F32>(a, n, s);
    if (a.dtype == MANTA_ROCM_F16) return launch_normed<F16>(a, n, s);
    return launch_normed<Bf16>(a, n, s);
}

}  // namespace manta
