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

}  // namespace manta
