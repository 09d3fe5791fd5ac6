// kernels_beams.hip -- the choice of the next beams for gfx950: the best of
//   scores[g, b] + logits[g, b, t] - log(sum over u of exp(logits[g, b, u]))
// over a group's beams b and the vocabulary t.
//
// One launch, and every logit is read once.  A workgroup takes a part of a row,
// 4,096 logits at a time, and a wave its quarter of them in registers (the next
// ones on their way): it keeps the largest it has seen, the sum of exp(x -
// largest), and the `best` largest logits, which is all that the total's order
// within a row can ask for, a lane each in order.  After the first piece few
// logits reach the last of those, so no wave waits for another before the part
// is done.  The last workgroup of a group (a ticket) joins the parts of each
// beam, and takes the best of the beams' candidates.
//
// 64 groups of 8 beams of 130001 logits: f32 76 us, 3.5 TB/s, bf16 73, f16 81; what
// bounds it are the exponentials, 16 of about 30 vector instructions a logit,
// which fill two thirds of the SIMDs' cycles (with 22 of them, to 1e-11, 90).
//
// Sums and totals are f64: totals of different beams lie a few 1e-2 apart
// where `best` of them are taken from a vocabulary, so an error of f32 (1e-7
// of a sum) would exchange two of them once in 10^5 choices, and this one
// (below 1e-10) does not.  A vector instruction of f64 takes as long as one of
// f32 here.
#include <type_traits>

#include "best_common.hpp"
#include "cache_kernels.hpp"
#include "code_common.hpp"
#include "decode_kernels.hpp"

namespace manta {

namespace {

constexpr int kThreads = 256;
constexpr int kHeld = kBeamPiece / kThreads;  // logits a thread holds
constexpr int kAhead = 4;                     // candidates that a thread of it holds
constexpr int kFound = 512;                   // candidates that the last workgroup ranks at once

// exp(d) for -700 <= d <= 0 (NaN stays), within 1e-10 of it: d = k ln 2 + r, |r|
// <= ln(2) / 2, and exp(r) as 1 + r + r^2 / 2 + r^3 times a polynomial of degree
// 4, whose coefficients make the largest relative error over that range the
// least (reweighted least squares; 9.6e-11.  The series to r^9 / 9! has 7e-12
// and two steps more).  Adding 1.5 * 2^52 rounds to k and leaves it in the low
// word, and k goes into the exponent by an addition.  The constants stay in
// scalar registers: as literals each would cost two moves a use.
struct Exp {
    double magic = 6755399441055744.0, log2e = 1.4426950408889634, ln2 = -0x1.62e42fefa39efp-1;
    double c7 = 0.0001973345940007819, c6 = 0.0013935234389446138, c5 = 0.008333586300566968,
           c4 = 0.041666461302453994, c3 = 0.1666666558083848;
    __device__ __forceinline__ Exp() {
        asm("" : "+s"(magic), "+s"(log2e), "+s"(ln2));
        asm("" : "+s"(c7), "+s"(c6), "+s"(c5), "+s"(c4), "+s"(c3));
    }
    __device__ __forceinline__ double operator()(double d) const {
        const double t = fma(d, log2e, magic);
        const double r = fma(t - magic, ln2, d);
        double p = fma(c7, r, c6);
        p = fma(p, r, c5);
        p = fma(p, r, c4);
        p = fma(p, r, c3);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        // (a NaN's low word has no bits that reach the exponent)
        uint32_t hi = (uint32_t)__double2hiint(p);
        const uint32_t k = (uint32_t)__double2loint(t);
        asm("v_lshl_add_u32 %0, %1, 20, %0" : "+v"(hi) : "v"(k));
        return __hiloint2double((int)hi, __double2loint(p));
    }
};
__device__ __forceinline__ double exp_neg(double d) { return d < -700.0 ? 0.0 : Exp()(d); }

// Order-preserving map of f64 (not NaN, -0 made +0) to u64; 0 is below all.
__device__ __forceinline__ uint64_t total_order(double t) {
    const uint64_t u = (uint64_t)__double_as_longlong(t + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double order_total(uint64_t o) {
    return __longlong_as_double((long long)(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
}

// Sums and maxima over a wave's 64 lanes, all of them active, in every lane:
// row shifts by 1, 2, 4 and 8, after which lane 15 of a row has its row's, and
// two broadcasts, after which lane 63 has the wave's.  A lane whose source lies
// outside takes `none`.  (A tenth of the cycles of exchanges through LDS.)
template <class F>
__device__ __forceinline__ void wave_steps(F step) {
    step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
    step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
}
__device__ __forceinline__ float wave_max(float x) {
    const int none = (int)0xFF800000u;  // -inf
    wave_steps([&](auto ctrl, auto rows) {
        x = fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(none, (int)__float_as_uint(x), ctrl(), rows(),
                                                                           0xf, false)));
    });
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
template <class Op>
__device__ __forceinline__ double wave_join(double x, double none, Op op) {
    const int nlo = __double2loint(none), nhi = __double2hiint(none);
    wave_steps([&](auto ctrl, auto rows) {
        const int lo = __builtin_amdgcn_update_dpp(nlo, __double2loint(x), ctrl(), rows(), 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(nhi, __double2hiint(x), ctrl(), rows(), 0xf, false);
        x = op(x, __hiloint2double(hi, lo));
    });
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), 63), __builtin_amdgcn_readlane(__double2loint(x), 63));
}
__device__ __forceinline__ double wave_sum(double x) {
    return wave_join(x, 0.0, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double wave_max(double x) {
    return wave_join(x, -HUGE_VAL, [](double a, double b) { return fmax(a, b); });
}

// A wave's lanes' shares exp(largest) * sum of one total (sum 0: none; a NaN in
// any stays), joined: *largest and the sum, in every lane.
__device__ __forceinline__ double joined(double sum, double* largest) {
    const double most = wave_max(sum == 0.0 ? -HUGE_VAL : *largest);
    sum = sum == 0.0 ? 0.0 : sum * exp_neg(*largest - most);
    *largest = most;
    return wave_sum(sum);
}

// Equal totals: the lower beam, of one beam the larger logit (a score may swallow
// their difference), then the lower token.  Candidate i of a beam stands for its
// token: parts lie in the tokens' order, and a part's keys too where logits are
// equal.
constexpr int kPlaceBits = 18;
static_assert(kMaxBeams * kBeamParts * kMaxBest <= 1 << kPlaceBits, "i fits its bits");
struct Candidate {
    uint64_t total, place;  // order of the total (0: none); beam, the logit's order complemented, i
    __device__ __forceinline__ int beam() const { return (int)(place >> (32 + kPlaceBits)); }
    __device__ __forceinline__ int index() const { return (int)(place & ((1u << kPlaceBits) - 1)); }
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

struct Floor {
    uint32_t floor;
};
struct MergeShared {
    double largest[kMaxBeams], log_sum[kMaxBeams], score[kMaxBeams];
    int ended[kMaxBeams];
    Candidate found[kFound];
    int token[kFound];
    Candidate wave_best[kThreads / 64];
    uint32_t tops[kThreads];
    Floor floor;
    int count;
};

// The last workgroup of group g: the best totals over its beams' parts.
__device__ __forceinline__ void merge_group(const BeamArgs& a, int g, MergeShared& M) {
    const int tid = threadIdx.x;
    const int words = (int)beam_part_words(a.best);
    const uint64_t* work = a.work + (int64_t)g * a.beams * a.parts * words;
    const int per = a.parts * a.best;  // candidates of a beam
    const int n = a.beams * per;
    // (keys of ended beams are whatever an earlier call left: not looked at)
    auto key_at = [&](int i) { return load_part(work + (int64_t)(i / a.best) * words + i % a.best); };
    uint64_t keys[kAhead];  // this thread's first ones, on their way
#pragma unroll
    for (int r = 0; r < kAhead; r++) keys[r] = tid + kThreads * r < n ? key_at(tid + kThreads * r) : 0ull;
    // A lane a part: a wave a beam, or of more beams than waves with few parts as
    // many side by side as there is room for, since each round of them waits for
    // its loads (81 groups of 12 beams of 6661, f16: 30 us a wave a beam, 27 so;
    // where a round is all there is the wave's exchanges are 1.5 faster).
    int lanes = 64;
    if (a.beams > kThreads / 64 && a.parts <= 16)
        for (lanes = 1; lanes < a.parts;) lanes *= 2;
    const int lane = tid & (lanes - 1);
    for (int b = tid / lanes; b < a.beams; b += kThreads / lanes) {
        const int row = g * a.beams + b;
        const uint64_t* part = work + ((int64_t)b * a.parts + min(lane, a.parts - 1)) * words + a.best;
        double largest = __longlong_as_double((long long)load_part(part));
        double sum = __longlong_as_double((long long)load_part(part + 1));
        const bool over = a.ended && a.ended[row] != 0;  // (then the parts are an earlier call's)
        if (lane >= a.parts) sum = 0.0;
        if (lanes == 64) {
            sum = joined(sum, &largest);
        } else {
            double most = sum == 0.0 ? -HUGE_VAL : largest;
            for (int s = lanes >> 1; s; s >>= 1) most = fmax(most, __shfl_xor(most, s));
            sum = sum == 0.0 ? 0.0 : sum * exp_neg(largest - most);
            for (int s = lanes >> 1; s; s >>= 1) sum += __shfl_xor(sum, s);
            largest = most;
        }
        if (lane == 0) {
            M.score[b] = (double)a.scores[row];
            M.ended[b] = over;
            M.largest[b] = largest;
            M.log_sum[b] = log(sum);
        }
    }
    if (tid == 0) M.count = 0;
    __syncthreads();
    auto candidate = [&](int i, uint64_t key) {
        const int b = i / per, k = i - b * per;
        Candidate c{0, (((uint64_t)b << 32) | (uint32_t)~(key >> 32)) << kPlaceBits | (uint32_t)i};
        double t;
        if (M.ended[b]) {
            if (k) return c;
            t = M.score[b];
        } else {
            if (!key) return c;
            // (apart: the largest may be a number that swallows the logarithm)
            t = M.score[b] + (((double)key_score(key, 0) - M.largest[b]) - M.log_sum[b]);
        }
        if (t > -HUGE_VAL) c.total = total_order(t);
        return c;
    };
    // Candidates at or above the best-th largest of the threads' own best
    // (compared as f32: narrowing keeps the order) are few and hold the result.
    auto coarse = [](const Candidate& c) { return c.total ? float_order((float)order_total(c.total)) : 0u; };
    uint32_t top = 0;
    auto each = [&](auto f) {
#pragma unroll
        for (int r = 0; r < kAhead; r++)
            if (tid + kThreads * r < n) f(candidate(tid + kThreads * r, keys[r]), keys[r]);
        for (int i = tid + kThreads * kAhead; i < n; i += kThreads) {
            const uint64_t key = key_at(i);
            f(candidate(i, key), key);
        }
    };
    auto token_of = [&](const Candidate& c, uint64_t key) { return M.ended[c.beam()] ? a.end_token : (int)key_index(key); };
    each([&](const Candidate& c, uint64_t) { top = max(top, coarse(c)); });
    M.tops[tid] = top;
    __syncthreads();
    find_floor<4>(M.tops, a.best, M.floor);
    __syncthreads();
    const uint32_t floor = M.floor.floor;
    each([&](const Candidate& c, uint64_t key) {
        if (c.total && coarse(c) >= floor) {
            const int at = atomicAdd(&M.count, 1);
            if (at < kFound) {
                M.found[at] = c;
                M.token[at] = token_of(c, key);
            }
        }
    });
    __syncthreads();
    const int found = M.count;
    auto put = [&](int k, const Candidate& c, int token) {
        const int64_t at = (int64_t)g * a.best + k;
        a.parents[at] = c.total ? c.beam() : -1;
        a.tokens[at] = token;
        a.totals[at] = c.total ? (float)order_total(c.total) : -__builtin_inff();
        if (a.now_ended) a.now_ended[at] = token == a.end_token ? 1 : 0;
    };
    if (found <= kFound) {
        for (int i = tid; i < found; i += kThreads) {
            const Candidate mine = M.found[i];
            int rank = 0;
            for (int k = 0; k < found; k++) rank += better(M.found[k], mine) ? 1 : 0;
            if (rank < a.best) put(rank, mine, M.token[i]);
        }
        for (int k = found + tid; k < a.best; k += kThreads) put(k, Candidate{0, 0}, -1);
        return;
    }
    // more of them than fit (totals equal in masses): one after the other
    Candidate last{~0ull, 0};
    for (int k = 0; k < a.best; k++) {
        Candidate mine{0, ~0ull};
        each([&](const Candidate& c, uint64_t) {
            if (c.total && better(last, c) && better(c, mine)) mine = c;
        });
        for (int s = 32; s; s >>= 1) {
            const Candidate o{(uint64_t)__shfl_xor((long long)mine.total, s), (uint64_t)__shfl_xor((long long)mine.place, s)};
            if (better(o, mine)) mine = o;
        }
        if ((tid & 63) == 0) M.wave_best[tid >> 6] = mine;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; w++)
            if (better(M.wave_best[w], mine)) mine = M.wave_best[w];
        if (tid == 0) put(k, mine, mine.total ? token_of(mine, key_at(mine.index())) : -1);
        last = mine;
        __syncthreads();
    }
}

// What a wave has seen: the largest, and a lane's sum of exp(x - largest).
struct Seen {
    float top = -__builtin_inff();
    double sum = 0.0;
    unsigned long long odd = 0;  // lanes that have met a NaN, or +inf
    // Returns the wave's largest of these.
    template <int N>
    __device__ __forceinline__ float add(const float (&x)[N], const Exp& exp) {
        float now = x[0];
#pragma unroll
        for (int j = 1; j < N; j++) now = fmaxf(now, x[j]);  // (a NaN shows below)
        now = wave_max(now);
        if (now > top) {
            sum *= exp_neg((double)top - (double)now);
            top = now;
        }
        // (all masked: 0 stands in for -inf, and the sum does not count)
        const float from = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const double d = (double)x[j] - (double)from;
            odd |= __ballot(!(d == d));
            sum += exp(fmax(d, -600.0));  // (1e-261 of the largest for less)
            // four at a time: sixteen at once do not fit the registers
            if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        return now;
    }
};

// A wave's `best` largest logits: lane i has the key of the i-th (0: none).
struct Kept {
    uint64_t key = 0;
    float tau = -__builtin_inff();  // the last one's logit and token, once there are so many:
    int tau_token = -1;             // what is to come in lies above it

    // Begin with the lanes' own largest of the first piece, sorted by counting
    // (and taken out of x): few others are left to come in one by one.
    template <int N, class Token>
    __device__ __forceinline__ void start(float (&x)[N], Token token, int best, uint64_t* room) {
        const uint32_t lane = threadIdx.x & 63;
        float high = x[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < N; j++)
            if (x[j] > high || !(high == high)) {
                high = x[j];
                at = j;
            }
        // (lanes without one come last, and apart from each other)
        const bool none = !(high > -__builtin_inff());
        int t = 0;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j == at) t = token(j);
        const uint64_t mine = none ? (uint64_t)(63 - lane) : make_key(high, (uint32_t)t, 0);
        room[lane] = mine;  // (the wave's own 64: its accesses are in order)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int rank = rank_in(room, 64, mine);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_permute(rank * 4, (int)(uint32_t)mine);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_permute(rank * 4, (int)(uint32_t)(mine >> 32));
        key = hi && (int)lane < best ? ((uint64_t)hi << 32) | lo : 0ull;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j == at && !none) x[j] = -__builtin_inff();
        look(best);
    }
    __device__ __forceinline__ void look(int best) {
        const uint64_t end = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(key >> 32), best - 1) << 32) |
                             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, best - 1);
        if (end) {
            tau = key_score(end, 0);
            tau_token = (int)key_index(end);
        }
    }
    template <class Token>
    __device__ __forceinline__ void offer(float x, Token token, int best) {
        unsigned long long m = __ballot(x >= tau);
        if (!m) return;
        const int t = token();
        m &= __ballot(x > tau || t < tau_token);
        while (m) {
            const int from = __ffsll(m) - 1;
            m &= m - 1;
            const uint64_t one =
                make_key(__uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), from)),
                         (uint32_t)__builtin_amdgcn_readlane(t, from), 0);
            const int place = __popcll(__ballot(key > one)), lane = threadIdx.x & 63;
            if (place >= best) continue;
            const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)key, 0x138, 0xf, 0xf, false);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(key >> 32), 0x138, 0xf, 0xf, false);
            const uint64_t before = ((uint64_t)hi << 32) | lo;  // the lane before's
            if (lane >= place) key = lane == place ? one : before;
        }
        look(best);
    }
};

template <class E>
__global__ __launch_bounds__(kThreads, 4) void beam_kernel(BeamArgs a) {
    typedef typename E::T T;
    constexpr int V = E::kWide, LOADS = kHeld / V;
    // Which thread and workgroup takes a logit depends on its place in the row
    // alone, so that rows of equal logits have equal sums to the last bit and
    // their totals tie; rows start anywhere, and the loads are 16 bytes all the
    // same (memory takes them at any alignment).
    struct alignas(16) Pack16 {
        T v[V];
    };
    __shared__ union Shared {
        BestShared best;
        MergeShared merge;
        __device__ Shared() {}
    } S;
    __shared__ double tops[kThreads / 64], sums[kThreads / 64];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x, row = blockIdx.y;
    const int g = row / a.beams;
    const bool over = a.ended && a.ended[row] != 0;
    uint64_t* dst = a.work + ((int64_t)row * a.parts + part) * beam_part_words(a.best);
    if (!over) {
        const T* src = (const T*)a.logits + (int64_t)row * a.logits_row;
        const int64_t end = a.vocab, pieces = (end + kBeamPiece - 1) / kBeamPiece;
        const int64_t p0 = pieces * part / a.parts, p1 = pieces * (part + 1) / a.parts;
        const int64_t mine = wave * (kBeamPiece / 4);
        Pack16 held[LOADS];
        auto fetch = [&](int64_t p) {
#pragma unroll
            for (int l = 0; l < LOADS; l++) {
                const int64_t v = p * kBeamPiece + mine + (l * 64 + lane) * V;
                if (v + V <= end) {
                    held[l] = load16_any<Pack16>(src + v);
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++)
                        if (v + k < end) held[l].v[k] = src[v + k];
                }
            }
        };
        const Exp exp;
        Seen seen;
        Kept kept;
        if (p0 < p1) fetch(p0);
        for (int64_t p = p0; p < p1; p++) {
            const int first = (int)(p * kBeamPiece + mine) + lane * V;
            auto at = [&](int j) { return first + (j / V) * 64 * V + j % V; };
            float x[kHeld];  // (-inf where there is none)
#pragma unroll
            for (int j = 0; j < kHeld; j++) x[j] = E::load(held[j / V].v[j % V]);
            if ((p + 1) * kBeamPiece > end) {
#pragma unroll
                for (int j = 0; j < kHeld; j++)
                    if (at(j) >= end) x[j] = -__builtin_inff();
            }
            if (p + 1 < p1) fetch(p + 1);
            const float top = seen.add(x, exp);
            if (p == p0) kept.start(x, at, a.best, S.best.keys + wave * 64);
            if (top >= kept.tau && top > -__builtin_inff()) {
#pragma unroll
                for (int q = 0; q < kHeld / 4; q++) {
                    const float most = fmaxf(fmaxf(x[4 * q], x[4 * q + 1]), fmaxf(x[4 * q + 2], x[4 * q + 3]));
                    if (!__ballot(most >= kept.tau)) continue;
#pragma unroll
                    for (int j = 4 * q; j < 4 * q + 4; j++) kept.offer(x[j], [&] { return at(j); }, a.best);
                }
            }
        }
        const double sum = seen.odd ? __builtin_nan("") : wave_sum(seen.sum);
        if (lane == 0) {
            const bool none = seen.top == -__builtin_inff();
            tops[wave] = none ? 0.0 : (double)seen.top;
            sums[wave] = none && sum == sum ? 0.0 : sum;
        }
        // The waves' lists by rank (merged by halving, 16 x 8 beams with 64 results
        // are 0.7 us of 72 faster, and calls of few results 0.2 slower).
        uint64_t* lists = S.best.keys + kThreads;  // (the first were ranked before these)
        const uint64_t key = lane < a.best ? kept.key : 0ull;
        if (lane < a.best) lists[wave * a.best + lane] = key;
        const int live = __syncthreads_count(key != 0);
        if (key) {
            const int rank = rank_in(lists, kThreads / 64 * a.best, key);
            if (rank < a.best) store_part(dst + rank, key);
        }
        for (int i = live + tid; i < a.best; i += kThreads) store_part(dst + i, 0ull);
        if (wave == kThreads / 64 - 1) {
            double largest = lane < kThreads / 64 ? tops[lane] : 0.0;
            const double all = joined(lane < kThreads / 64 ? sums[lane] : 0.0, &largest);
            if (lane == 0) {
                store_part(dst + a.best, (uint64_t)__double_as_longlong(largest));
                store_part(dst + a.best + 1, (uint64_t)__double_as_longlong(all));
            }
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
    if (last) merge_group(a, g, S.merge);
}

__global__ __launch_bounds__(kThreads) void inputs_kernel(const int32_t* tokens, int n, int instead, int32_t* out) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i < n) out[i] = tokens[i] < 0 ? instead : tokens[i];
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
        if (a.now_ended) p.now_ended += (int64_t)g0 * a.best;
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

hipError_t launch_beam_inputs(const int32_t* tokens, int n, int instead, int32_t* out, hipStream_t s) {
    inputs_kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, s>>>(tokens, n, instead, out);
    return hipGetLastError();
}

}  // namespace manta
