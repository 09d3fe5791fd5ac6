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
#include "code_common.hpp"

namespace manta {

namespace {

constexpr int kThreads = 256;

template <class E, int V>
struct alignas(sizeof(typename E::T) * V) Pack {
    typename E::T v[V];
};

// The part of a turn that pos * turns leaves, in [-1/2, 1/2]: of the exact
// product, whose f64 rounding is 3e-8 turns off at position 2^31.
__device__ __forceinline__ float turn_left(double pos, double turns) {
    return (float)fma(pos, turns, -rint(pos * turns));
}
// A pair turned: a product and a fused one, so two roundings.
__device__ __forceinline__ float turn_1(float x1, float x2, float c, float s) { return fmaf(x1, c, -(x2 * s)); }
__device__ __forceinline__ float turn_2(float x1, float x2, float c, float s) { return fmaf(x2, c, x1 * s); }

// A result, rounded to f32 and then to its type.  (Else the compiler fuses f16's
// rounding with the operation before it for some elements of a piece and not for
// others: a result would depend on its place, and two lanes that work out the
// same element could write two.)
template <class E>
__device__ __forceinline__ typename E::T stored(float y) {
    asm("" : "+v"(y));
    return E::store(y);
}

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
            const float r = turn_left(pos, a.turns[p]);
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
                const T y1 = stored<E>(turn_1(x1, x2, c, s)), y2 = stored<E>(turn_2(x1, x2, c, s));
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
// of f32 leaves its range.  The weights are fetched into LDS once for a
// workgroup's `tokens`, whose heads it takes as one run, the first ones' data
// on their way while the angles are worked out.  Bytes bound: 8192 tokens of 40
// heads of 128, bf16, out of memory: 29 to 35 us, 4.8 to 5.7 TB/s.
//
// PIECES says how a head splits into pieces of 16 bytes:
//   kEven   whole ones at their alignment, pairs and rest alike;
//   kShared at any alignment, the last one of the pairs and of the rest ending
//           where they do: it shares its first elements with the piece before,
//           which works out the same for them (the sum takes them once);
//   kShort  as kShared where there are too few for one piece: the last is taken
//           element by element.
// (4169 tokens of 36 heads of 80, 50 of them rotated, bf16: kShared 22 us, kShort
// 33.)
enum { kEven, kShared, kShort };
constexpr int kNormTokens = 8;
template <class E, bool INTERLEAVED, int PIECES, int NP>
__global__ __launch_bounds__(kThreads) void rotary_normed_kernel(RotaryArgs a, RotaryNorms n, int lanes, int tokens) {
    typedef typename E::T T;
    constexpr int V = E::kWide;
    typedef Pack<E, V> Piece;
    // (a last piece reads on past what there is, and stores none of it)
    __shared__ alignas(16) float cs[kNormTokens][kMaxHeadDim / 2 + V], sn[kNormTokens][kMaxHeadDim / 2 + V];
    __shared__ alignas(16) float weight[kRotaryParts][kMaxHeadDim + 2 * V];
    const int half = a.rot >> 1;
    const int turned = (half + V - 1) / V;                // pieces of V pairs
    const int rest = (a.head_dim - a.rot + V - 1) / V;    // pieces of V columns past them
    const int pieces = turned + rest;
    // the first pair of a piece, or column past the pairs
    auto start = [&](int piece) {
        if (piece < turned) return PIECES == kShared ? min(piece * V, half - V) : piece * V;
        const int c = a.rot + (piece - turned) * V;
        return PIECES == kShared ? min(c, a.head_dim - V) : c;
    };
    const int per = (a.heads + gridDim.y - 1) / gridDim.y;
    const int h0 = blockIdx.y * per, heads = min(a.heads, h0 + per) - h0;
    const int gl = threadIdx.x & (lanes - 1), g0 = threadIdx.x / lanes, step = kThreads / lanes;
    auto put = [&](T* p, Piece v) {
        if (n.past) store16_past(p, v);
        else *(Piece*)p = v;
    };
    for (int k = 0; k < a.parts; k++)
        if (n.weight[k])
            for (int c = threadIdx.x; c < a.head_dim; c += kThreads) weight[k][c] = n.weight[k][c];
    for (int64_t t0 = (int64_t)blockIdx.x * tokens; t0 < a.tokens; t0 += (int64_t)gridDim.x * tokens) {
        const int count = (int)min((int64_t)tokens, a.tokens - t0), all = count * heads;

        // a head's elements as this lane has them
        Piece lo[NP], hi[NP];
        T* out = nullptr;
        int token = 0, part = 0;
        auto fetch = [&](int i) {
            token = i / heads;
            int h = h0 + i - token * heads;
            // (the parts' fields are picked with constant indices: they stay in
            // scalar registers, where a lane's own index would read them from memory)
            part = 0;
            const T* src = (const T*)a.part[0].x + (t0 + token) * a.part[0].x_token + h * a.part[0].x_head;
            out = (T*)a.part[0].out + (t0 + token) * a.part[0].out_token + h * a.part[0].out_head;
#pragma unroll
            for (int k = 1; k < kRotaryParts; k++) {
                if (k >= a.parts || h < a.part[k - 1].heads) break;
                h -= a.part[k - 1].heads;
                part = k;
                src = (const T*)a.part[k].x + (t0 + token) * a.part[k].x_token + h * a.part[k].x_head;
                out = (T*)a.part[k].out + (t0 + token) * a.part[k].out_token + h * a.part[k].out_head;
            }
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const int piece = gl + lanes * p, at = start(piece);
                const T* from0 = src + (INTERLEAVED && piece < turned ? 2 * at : at);
                const T* from1 = src + (INTERLEAVED ? 2 * at + V : half + at);
                const bool whole = PIECES != kShort || at + V <= (piece < turned ? half : a.head_dim);
                if (whole && piece < pieces) lo[p] = PIECES == kEven ? *(const Piece*)from0 : load16_any<Piece>(from0);
                if (whole && piece < turned) hi[p] = PIECES == kEven ? *(const Piece*)from1 : load16_any<Piece>(from1);
                if constexpr (PIECES == kShort) {
                    if (whole || piece >= pieces) continue;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const bool pairs = piece < turned;
                        const int end = !pairs ? a.head_dim : INTERLEAVED ? a.rot - at : half;
                        if (at + j < end) lo[p].v[j] = from0[j];
                        if (pairs && at + (INTERLEAVED ? V + j : j) < end) hi[p].v[j] = from1[j];
                    }
                }
            }
        };
        int twice[NP];  // elements of a piece that the piece before it has too
#pragma unroll
        for (int p = 0; p < NP; p++) {
            lo[p] = hi[p] = Piece{};  // (what is not fetched counts as 0)
            const int piece = gl + lanes * p;
            twice[p] = PIECES != kShared || piece >= pieces ? 0
                       : piece < turned                     ? (INTERLEAVED ? 2 : 1) * (piece * V - start(piece))
                                                            : a.rot + (piece - turned) * V - start(piece);
        }
        if (g0 < all) fetch(g0);
        for (int e = threadIdx.x; e < count * half; e += kThreads) {
            const int token = e / half, p = e - token * half;
            const float r = turn_left((double)a.positions[t0 + token], a.turns[p]);
            float s, c;
            sincospif(2.0f * r, &s, &c);
            cs[token][p] = a.magnitude * c;
            sn[token][p] = a.magnitude * s;
        }
        __syncthreads();
        for (int base = 0; base < all; base += step) {  // (all lanes stay for the exchange)
            const bool live = base + g0 < all;
            double sum = 0.0;
#pragma unroll
            for (int p = 0; p < NP; p++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float u = E::load(lo[p].v[j]), v = E::load(hi[p].v[j]);
                    if (PIECES == kShared) {
                        u = j < twice[p] ? 0.0f : u;
                        v = (INTERLEAVED ? V + j : j) < twice[p] ? 0.0f : v;
                    }
                    sum = fma((double)u, (double)u, sum);
                    sum = fma((double)v, (double)v, sum);
                }
            for (int s = lanes >> 1; s; s >>= 1) sum += __shfl_xor(sum, s);
            bool norm = n.weight[0] != nullptr;
#pragma unroll
            for (int k = 1; k < kRotaryParts; k++)
                if (part == k) norm = n.weight[k] != nullptr;
            // the hardware's 2^-23 and a step of Newton's, of the error squared
            const double mean = fma(sum, n.inv_dim, n.eps), r0 = __builtin_amdgcn_rsq(mean);
            // (of infinity 0 as it is: the step would be 0 times infinity)
            const double r1 = mean < HUGE_VAL ? fma(0.5 * r0, fma(-mean * r0, r0, 1.0), r0) : r0;
            const float r = norm ? (float)r1 : 1.0f;
            const float* w = weight[part];
            if (live) {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int piece = gl + lanes * i;
                    if (piece >= pieces) continue;
                    if (piece >= turned) {
                        const int at = start(piece);
                        Piece o;
#pragma unroll
                        for (int j = 0; j < V; j++)
                            o.v[j] = norm ? stored<E>(E::load(lo[i].v[j]) * r * w[at + j]) : lo[i].v[j];
                        if constexpr (PIECES == kEven) {
                            put(out + at, o);
                        } else if (PIECES == kShared || at + V <= a.head_dim) {
                            store16_any(out + at, o);
                        } else if constexpr (PIECES == kShort) {
#pragma unroll
                            for (int j = 0; j < V; j++)
                                if (at + j < a.head_dim) out[at + j] = o.v[j];
                        }
                        continue;
                    }
                    const int p = start(piece);
                    // the run of columns that lo holds, and hi
                    const int at0 = INTERLEAVED ? 2 * p : p, at1 = INTERLEAVED ? 2 * p + V : half + p;
                    float u[2 * V];
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        u[j] = E::load(lo[i].v[j]);
                        u[V + j] = E::load(hi[i].v[j]);
                        if (norm) {
                            u[j] = u[j] * r * w[at0 + j];
                            u[V + j] = u[V + j] * r * w[at1 + j];
                        }
                    }
                    T o[2 * V];
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        // pair p + j: elements 2j and 2j + 1 of the run, or j of each half
                        const int e1 = INTERLEAVED ? 2 * j : j, e2 = INTERLEAVED ? 2 * j + 1 : V + j;
                        const float c = cs[token][p + j], s = sn[token][p + j];
                        o[e1] = stored<E>(turn_1(u[e1], u[e2], c, s));
                        o[e2] = stored<E>(turn_2(u[e1], u[e2], c, s));
                    }
                    Piece ylo, yhi;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        ylo.v[j] = o[j];
                        yhi.v[j] = o[V + j];
                    }
                    if constexpr (PIECES == kEven) {
                        put(out + at0, ylo);
                        put(out + at1, yhi);
                    } else if (PIECES == kShared || p + V <= half) {
                        store16_any(out + at0, ylo);
                        store16_any(out + at1, yhi);
                    } else if constexpr (PIECES == kShort) {
#pragma unroll
                        for (int j = 0; j < V; j++) {
                            if (INTERLEAVED ? at0 + j < a.rot : p + j < half) out[at0 + j] = ylo.v[j];
                            if (INTERLEAVED ? at1 + j < a.rot : p + j < half) out[at1 + j] = yhi.v[j];
                        }
                    }
                }
            }
            if (base + step + g0 < all) fetch(base + step + g0);
        }
        __syncthreads();  // the angles have been used
    }
}

template <class E>
hipError_t launch_normed(const RotaryArgs& a, RotaryNorms n, hipStream_t s) {
    // results past the 32 MB of the L2s are not found there by what reads them
    // next: written past them, they leave the room to what is being read
    // (8192 x 40 heads of 128, bf16, out of memory and back: 42 us, 35 so; with
    // a rotary that reads it 73, 70)
    n.past = a.tokens * a.heads * a.head_dim * (int64_t)sizeof(typename E::T) > ((int64_t)32 << 20);
    constexpr int V = E::kWide;
    const int pieces = (a.rot / 2 + V - 1) / V + (a.head_dim - a.rot + V - 1) / V;  // 65 at most
    int lanes = 1;
    while (lanes < pieces && lanes < 64) lanes *= 2;
    // few tokens: a token's heads over several workgroups, so that the card is
    // full; many: as many a workgroup as give it about six rounds of its
    // lanes, while there are 1,024 workgroups (8192 x 40 heads of 128: bf16 1
    // token 39.3 us, 2 33.7, 4 31.3; f32 68.5, 67.1, 73.9; 5001 x 24 of 64, f32:
    // 22.9, 18.7, 18.1)
    int split = 1;
    while (split < 8 && split * 2 <= a.heads && a.tokens * split < 512) split *= 2;
    int64_t tokens = 1536 / (a.heads * lanes);
    if (tokens > a.tokens / 1024) tokens = a.tokens / 1024;
    tokens = tokens < 1 ? 1 : tokens > kNormTokens ? kNormTokens : tokens;
    const int64_t runs = (a.tokens + tokens - 1) / tokens;
    const dim3 grid((unsigned)(runs < (1 << 20) ? runs : 1 << 20), split);
    // (pieces at any alignment where all are aligned: 49.7 us against 42 for 8192
    // tokens of 40 heads of 128, bf16, out of memory)
    const int t = (int)tokens, over = a.head_dim - a.rot;
    if (a.wide) {  // 64 pieces at most
        if (a.interleaved) rotary_normed_kernel<E, true, kEven, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
        else rotary_normed_kernel<E, false, kEven, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
    } else if (a.rot / 2 >= V && (over == 0 || over >= V)) {  // 64 as well: 4 pairs take two pieces' columns
        if (a.interleaved) rotary_normed_kernel<E, true, kShared, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
        else rotary_normed_kernel<E, false, kShared, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
    } else if (pieces <= 64) {
        if (a.interleaved) rotary_normed_kernel<E, true, kShort, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
        else rotary_normed_kernel<E, false, kShort, 1><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
    } else if constexpr (V == 4) {  // a pair and 254 columns of f32
        if (a.interleaved) rotary_normed_kernel<E, true, kShort, 2><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
        else rotary_normed_kernel<E, false, kShort, 2><<<grid, kThreads, 0, s>>>(a, n, lanes, t);
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
