// kernels_beams.hip -- the choice of the next beams for gfx950: the best of
//   scores[g, b] + logits[g, b, t] - log(sum over u of exp(logits[g, b, u]))
// over a group's beams b and the vocabulary t.
//
// One launch, and every logit is read once.  A workgroup holds 8,192 of a
// row's logits in registers: their largest, the sum of exp(x - largest) and
// the row's `best` largest of them, which is all that the total's order within
// a row can ask for.  The last workgroup of a group (a ticket) joins the parts
// of each beam, and takes the best of the beams' candidates.
//
// Sums and totals are f64: totals of different beams lie a few 1e-2 apart
// where `best` of them are taken from a vocabulary, so an error of f32 (1e-7
// of a sum) would exchange two of them once in 10^5 choices, and this one
// (1e-15) does not.  A vector instruction of f64 takes as long as one of f32
// here.
#include "best_common.hpp"
#include "cache_kernels.hpp"
#include "decode_kernels.hpp"

namespace manta {

namespace {

constexpr int kThreads = 256;
constexpr int kHeld = kBeamPiece / kThreads;  // logits a thread holds
constexpr int kFound = 1024;                  // candidates that the last workgroup ranks at once

// exp(d) for d <= 0 (0 below -708), within 2e-16 of it: d = k ln 2 + r, and the
// series of exp(r) to r^13 / 13!, |r| <= ln(2) / 2.
__device__ __forceinline__ double exp_neg(double d) {
    if (d < -708.0) d = -HUGE_VAL;
    const double k = rint(d * 1.4426950408889634);
    double r = fma(k, -0x1.62e42fefa39efp-1, d);  // ln 2 in two parts
    r = fma(k, -0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return d < -708.0 ? 0.0 : ldexp(p, (int)k);
}

// Order-preserving map of f64 (not NaN, -0 made +0) to u64; 0 is below all.
__device__ __forceinline__ uint64_t total_order(double t) {
    const uint64_t u = (uint64_t)__double_as_longlong(t + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double order_total(uint64_t o) {
    return __longlong_as_double((long long)(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
}

// Order of a logit: never 0, every NaN above the numbers.
__device__ __forceinline__ uint32_t logit_order(float x) { return x != x ? 0xFFC00000u : float_order(x); }

struct Joined {  // of a row or a part: exp(largest) * sum
    double largest, sum;
};
// Both may be empty (sum 0); a NaN in either stays.
__device__ __forceinline__ Joined join(Joined a, Joined b) {
    if (b.sum == 0.0) return a;
    if (a.sum == 0.0) return b;
    const double m = fmax(a.largest, b.largest);
    return {m, a.sum * exp_neg(a.largest - m) + b.sum * exp_neg(b.largest - m)};
}

struct Candidate {
    uint64_t total, place;  // order of the total (0: none), beam << 32 | token
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
    return a.total > b.total || (a.total == b.total && a.place < b.place);
}

__device__ __forceinline__ uint64_t load_part(const uint64_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_part(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct MergeShared {
    double largest[kMaxBeams], log_sum[kMaxBeams], score[kMaxBeams];
    int ended[kMaxBeams];
    Candidate found[kFound];
    Candidate wave_best[kThreads / 64];
    uint32_t tops[kThreads];
    uint32_t floor;
    int count;
};

// The last workgroup of group g: the best totals over its beams' parts.
__device__ __forceinline__ void merge_group(const BeamArgs& a, int g, MergeShared& M, BestShared& B) {
    const int tid = threadIdx.x;
    const int words = (int)beam_part_words(a.best);
    const uint64_t* work = a.work + (int64_t)g * a.beams * a.parts * words;
    for (int b = tid; b < a.beams; b += kThreads) {
        const int row = g * a.beams + b;
        M.score[b] = (double)a.scores[row];
        M.ended[b] = a.ended && a.ended[row] != 0;
        if (!M.ended[b]) {
            Joined j{0.0, 0.0};
            for (int p = 0; p < a.parts; p++) {
                const uint64_t* part = work + ((int64_t)b * a.parts + p) * words + a.best;
                j = join(j, {__longlong_as_double((long long)load_part(part)),
                             __longlong_as_double((long long)load_part(part + 1))});
            }
            M.largest[b] = j.largest;
            M.log_sum[b] = log(j.sum);
        }
    }
    if (tid == 0) M.count = 0;
    __syncthreads();
    const int per = a.parts * a.best;  // candidates of a beam
    const int n = a.beams * per;
    auto candidate = [&](int i) {
        const int b = i / per, k = i - b * per;
        Candidate c{0, 0};
        double t;
        if (M.ended[b]) {
            if (k) return c;
            t = M.score[b];
            c.place = ((uint64_t)b << 32) | (uint32_t)a.end_token;
        } else {
            const uint64_t key = load_part(work + ((int64_t)b * a.parts + k / a.best) * words + k % a.best);
            if (!key) return c;
            // (apart: the largest may be a number that swallows the logarithm)
            t = M.score[b] + (((double)key_score(key, 0) - M.largest[b]) - M.log_sum[b]);
            c.place = ((uint64_t)b << 32) | key_index(key);
        }
        if (t > -HUGE_VAL) c.total = total_order(t);
        return c;
    };
    // Candidates at or above the best-th largest of the threads' own best
    // (compared as f32: narrowing keeps the order) are few and hold the result.
    auto coarse = [](const Candidate& c) { return c.total ? float_order((float)order_total(c.total)) : 0u; };
    uint32_t top = 0;
    for (int i = tid; i < n; i += kThreads) top = max(top, coarse(candidate(i)));
    M.tops[tid] = top;
    __syncthreads();
    find_floor<4>(M.tops, a.best, B);
    __syncthreads();
    const uint32_t floor = B.floor;
    for (int i = tid; i < n; i += kThreads) {
        const Candidate c = candidate(i);
        if (c.total && coarse(c) >= floor) {
            const int at = atomicAdd(&M.count, 1);
            if (at < kFound) M.found[at] = c;
        }
    }
    __syncthreads();
    const int found = M.count;
    auto put = [&](int k, const Candidate& c) {
        const int64_t at = (int64_t)g * a.best + k;
        a.parents[at] = c.total ? (int)(c.place >> 32) : -1;
        a.tokens[at] = c.total ? (int)(uint32_t)c.place : -1;
        a.totals[at] = c.total ? (float)order_total(c.total) : -__builtin_inff();
    };
    if (found <= kFound) {
        for (int i = tid; i < found; i += kThreads) {
            const Candidate mine = M.found[i];
            int rank = 0;
            for (int k = 0; k < found; k++) rank += better(M.found[k], mine) ? 1 : 0;
            if (rank < a.best) put(rank, mine);
        }
        for (int k = found + tid; k < a.best; k += kThreads) put(k, Candidate{0, 0});
        return;
    }
    // more of them than fit (totals equal in masses): one after the other
    Candidate last{~0ull, 0};
    for (int k = 0; k < a.best; k++) {
        Candidate mine{0, ~0ull};
        for (int i = tid; i < n; i += kThreads) {
            const Candidate c = candidate(i);
            if (c.total && better(last, c) && better(c, mine)) mine = c;
        }
        for (int s = 32; s; s >>= 1) {
            const Candidate o{(uint64_t)__shfl_xor((long long)mine.total, s), (uint64_t)__shfl_xor((long long)mine.place, s)};
            if (better(o, mine)) mine = o;
        }
        if ((tid & 63) == 0) M.wave_best[tid >> 6] = mine;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; w++)
            if (better(M.wave_best[w], mine)) mine = M.wave_best[w];
        if (tid == 0) put(k, mine);
        last = mine;
        __syncthreads();
    }
}

template <class E>
__global__ __launch_bounds__(kThreads) void beam_kernel(BeamArgs a) {
    typedef typename E::T T;
    constexpr int V = E::kWide;
    // Which thread and workgroup takes a logit depends on its place in the row
    // alone, so that rows of equal logits have equal sums to the last bit and
    // their totals tie; rows start anywhere, and the loads are 16 bytes all the
    // same (memory takes them at any alignment).
    struct alignas(sizeof(T)) Pack16 {
        T v[V];
    };
    __shared__ BestShared B;
    __shared__ MergeShared M;
    __shared__ uint64_t kept_keys[kMaxBest];
    __shared__ uint32_t wave_top[kThreads / 64];
    __shared__ double wave_sum[kThreads / 64];
    __shared__ int last;
    const int tid = threadIdx.x, part = blockIdx.x, row = blockIdx.y;
    const int g = row / a.beams;
    const bool over = a.ended && a.ended[row] != 0;
    uint64_t* dst = a.work + ((int64_t)row * a.parts + part) * beam_part_words(a.best);
    if (!over) {
        const T* src = (const T*)a.logits + (int64_t)row * a.logits_row;
        const int64_t end = a.vocab, pieces = (end + kBeamPiece - 1) / kBeamPiece;
        const int64_t p0 = pieces * part / a.parts, p1 = pieces * (part + 1) / a.parts;
        Joined all{0.0, 0.0};
        int kept = 0;
        for (int64_t p = p0; p < p1; p++) {
            const int64_t v0 = p * kBeamPiece;
            auto at = [&](int j) { return v0 + ((j / V) * kThreads + tid) * V + j % V; };
            uint32_t o[kHeld];  // order of a logit; 0 where there is none
#pragma unroll
            for (int j = 0; j < kHeld; j += V) {
                const int64_t v = at(j);
                if (v + V <= end) {
                    const Pack16 x = *(const Pack16*)(src + v);
#pragma unroll
                    for (int k = 0; k < V; k++) o[j + k] = logit_order(E::load(x.v[k]));
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++)
                        o[j + k] = v + k < end ? logit_order(E::load(src[v + k])) : 0u;
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < kHeld; j++) top = max(top, o[j]);
            for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
            if ((tid & 63) == 0) wave_top[tid >> 6] = top;
            __syncthreads();
            for (int w = 0; w < kThreads / 64; w++) top = max(top, wave_top[w]);
            const double largest = (double)order_float(top);
            // (all masked: 0 stands in for -inf, and the sum is 0)
            const double from = largest == -HUGE_VAL ? 0.0 : largest;
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < kHeld; j++)
                if (o[j]) sum += exp_neg((double)order_float(o[j]) - from);
            for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
            if ((tid & 63) == 0) wave_sum[tid >> 6] = sum;
            __syncthreads();
            sum = 0.0;
            for (int w = 0; w < kThreads / 64; w++) sum += wave_sum[w];
            all = join(all, {from, sum});
            // the piece's best, and with those of the pieces before
            auto token = [&](int j) { return o[j] ? (int)at(j) : -1; };
            int now = block_best<kHeld>([&](int j) { return o[j]; }, token, kHeld, a.best, B);
            if (now < 0)
                now = best_streamed(
                    [&](int64_t i) {
                        const int64_t v = v0 + i;
                        return v < end ? make_key(E::load(src[v]), (uint32_t)v, 0) : 0ull;
                    },
                    kBeamPiece, 1ull, a.best, B);
            if (p > p0) {
                __syncthreads();
                for (int i = tid; i < kept; i += kThreads) B.keys[now + i] = kept_keys[i];
                __syncthreads();
                now = best_of(now + kept, a.best, B);
            }
            kept = now;
            __syncthreads();
            if (p + 1 < p1) {
                for (int i = tid; i < kept; i += kThreads) kept_keys[i] = B.keys[i];
                __syncthreads();
            }
        }
        for (int i = tid; i < a.best; i += kThreads) store_part(dst + i, i < kept ? B.keys[i] : 0ull);
        if (tid == 0) {
            store_part(dst + a.best, (uint64_t)__double_as_longlong(all.largest));
            store_part(dst + a.best + 1, (uint64_t)__double_as_longlong(all.sum));
        }
    }
    // Publication: agent-scope stores, retired before the ticket.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
        last = __hip_atomic_fetch_add(&a.tickets[g], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               (uint32_t)(a.beams * a.parts - 1);
        if (last) __hip_atomic_store(&a.tickets[g], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last) merge_group(a, g, M, B);
}

template <class E>
hipError_t launch_type(const BeamArgs& a, hipStream_t s) {
    // rows are a grid's second axis, 16 bits of it: whole groups at a time
    const int most = 65535 / a.beams;
    for (int g0 = 0; g0 < a.groups; g0 += most) {
        BeamArgs p = a;
        const int64_t rows = (int64_t)g0 * a.beams;
        p.groups = a.groups - g0 < most ? a.groups - g0 : most;
        p.logits = (const typename E::T*)a.logits + rows * a.logits_row;
        p.scores += rows;
        if (a.ended) p.ended += rows;
        p.parents += (int64_t)g0 * a.best;
        p.tokens += (int64_t)g0 * a.best;
        p.totals += (int64_t)g0 * a.best;
        p.work += rows * a.parts * beam_part_words(a.best);
        p.tickets += g0;
        beam_kernel<E><<<dim3(a.parts, p.groups * a.beams), kThreads, 0, s>>>(p);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F32) return launch_type<F32>(a, s);
    if (a.dtype == MANTA_ROCM_F16) return launch_type<F16>(a, s);
    return launch_type<Bf16>(a, s);
}

}  // namespace manta
