// kernels_cache_prompt.hip -- softmax(scale q k^T) v over the 8-bit cache,
// many rows of a sequence at a time: prompts, and passages after a cached
// prefix.
//
// Bound by the instructions of the softmax and of staging beside the products:
// 4 sequences of up to 4096 rows, 32 heads of 128 over 8, bf16: 657 us, 872
// TFLOP/s (a large product reaches 1174).  A workgroup takes 256 or 128 rows
// (the query heads of a kv head, and tokens) and goes over the keys 64 at a
// time: the codes become f16 (bf16 for k of bf16 queries) once per workgroup,
// in LDS, and its waves multiply them with 32 rows each.
#include "cache_attend.hpp"

namespace manta {

namespace {

constexpr int kMaxSplits = 16;

constexpr int kKeys = 64;  // of a step

// Scores are k q^T in tiles of 32 keys by 32 rows: lane (h, c) = (lane / 32,
// lane % 32) holds 16 scores of row c.  Row 8 i + 4 h + j of the k operand is
// key 16 h + 4 i + j of the 32, so those 16 are keys of one block (of one
// page, with one scale), and the product v^T p takes its p from the registers
// that hold them.
//
// A weight carries its page's v_max in its exponent (p of cache_attend.hpp), and
// codes stay exact.  (Codes scaled as they are staged would be rounded with
// their scale: 1.8 times the rounding error of an f16 result, not 1.4.)  A row's
// m and D move when they are exceeded by 8 or more (p is at most 2^15), so most
// steps leave the sums alone.  (Weights against the largest v_max of all the
// tile's keys instead: 633 us for the 657 above, and rows that see only pages of
// small v lose their weights to a page that they do not see.)
constexpr float kSlack = 8.0f, kLift = 7.0f;
template <class E, int DP, int WAVES, int OCC, bool ONE_PAGE>
__global__ __launch_bounds__(64 * WAVES, OCC) void attend_many_kernel(CacheView c, int64_t layer, RaggedRows r,
                                                                  AttendArgs a) {
    typedef typename E::T T;
    typedef typename MmaOf<E>::M M;
    typedef typename M::V V8;
    constexpr int kThreads = 64 * WAVES;
    constexpr int D = 32 * DP, KS = 2 * DP, RT = WAVES * 32, OP = D + 4;
    constexpr int KPITCH = D + 8, VPITCH = kKeys + 8;  // (elements: rows start 4 banks apart)
    constexpr int CHUNKS = kKeys * D / 16, EACH = (CHUNKS + kThreads - 1) / kThreads;
    __shared__ T k_lds[2][kKeys * KPITCH];
    __shared__ _Float16 v_lds[2][D * VPITCH];
    // of each block of 16 keys: the factor of its scores, log2 of its v_max, its kind
    __shared__ f32x4 block_lds[2][4];

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // kv heads first: workgroups go round the dies, so a head's stay on one
    // (of 8 heads), whose cache then holds its keys.  The last rows see the
    // most keys: they go first.
    const int kv = blockIdx.x % c.kv_heads, split = blockIdx.y;
    const int64_t slot = gridDim.x / c.kv_heads - 1 - blockIdx.x / c.kv_heads;
    const Tile t = my_tile(c, r, a, slot, RT);
    if (t.rows == 0) return;
    int c0 = t.begin >> 6, c1 = t.end > t.begin ? (t.end + 63) >> 6 : c0;
    const int parts = min(max((c1 - c0 + a.rounds - 1) / a.rounds, 1), a.splits);
    if (split >= parts) return;
    {
        const int n = c1 - c0, first = c0;
        c0 = first + (int)((int64_t)n * split / parts);
        c1 = first + (int)((int64_t)n * (split + 1) / parts);
    }

    const int32_t* table = c.tables + (int64_t)t.seq * c.table_pages;
    const int mask = c.page_tokens - 1, last_page = (t.end - 1) >> c.page_shift;
    const uint32_t page_codes = (uint32_t)c.page_codes();  // (at most 65535 * 128 * 256)
    const int64_t slab0 = c.slab(layer, 0), head_codes = (int64_t)kv * c.page_tokens * c.pitch;
    const int8_t* kbase = c.k_codes + slab0 * page_codes + head_codes;
    const int8_t* vbase = c.v_codes + slab0 * page_codes + head_codes;
    const float* kmax = c.k_max + slab0 * c.kv_heads + kv;
    const float* vmax = c.v_max + slab0 * c.kv_heads + kv;

    // the wave's rows, clamped (the doubles are not stored), as operands
    const int d = c.head_dim, wave_row = wave * 32;
    V8 q[KS];
    int lo, hi;
    {
        const int row = t.r0 + min(wave_row + col, t.rows - 1);
        const int token = row / a.group, head = kv * a.group + row % a.group;
        const int pos = t.length - t.count + token;
        lo = key_begin(a, pos);
        hi = key_end(a, t.length, pos);
        const T* src = (const T*)a.q + (int64_t)(t.row0 + token) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int at = 16 * s + 8 * h;
            V8 x;
            if (a.wide && at + 8 <= d) {
                x = *(const V8*)(src + at);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = at + j < d ? src[at + j] : (T)0.0f;
            }
            q[s] = a.scale < 0.0f ? -x : x;  // (the scores' order is that of the products)
        }
    }
    // keys that some of the wave's rows see, and that all of them do
    int some_lo, some_hi, all_lo, all_hi;
    {
        const int first = t.length - t.count + (t.r0 + min(wave_row, t.rows - 1)) / a.group;
        const int last = t.length - t.count + (t.r0 + min(wave_row + 31, t.rows - 1)) / a.group;
        some_lo = key_begin(a, first);
        all_lo = key_begin(a, last);
        all_hi = key_end(a, t.length, first);
        some_hi = wave_row < t.rows ? key_end(a, t.length, last) : 0;
    }

    // codes on their way to LDS
    u32x4 kc[EACH], vc[EACH];
    float v_big = 0.0f, k_big = 0.0f;  // block tid % 4: largest v, largest k
    bool bad = false;
    auto page_of = [&](int x, int block) { return table[min((64 * x + 16 * block) >> c.page_shift, last_page)]; };
    // Vector loads, though their addresses are the same for all: a scalar load
    // on its way would make every wait for LDS a wait for memory.
    int zero = 0;
    asm("" : "+v"(zero));
    int page_k[EACH], page_v;
    auto look = [&](int x) {
        x = min(x, c1 - 1);
        if (ONE_PAGE) {
            page_v = page_of(x, zero);
            return;
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int key = min((tid + kThreads * i) / KS, kKeys - 1);
            page_k[i] = page_of(x, key >> 4);
        }
        page_v = page_of(x, tid & 3);
    };
    auto fetch = [&](int x) {
        x = min(x, c1 - 1);
        bad = (unsigned)page_v >= (unsigned)c.pages;
        if (bad && tid < 4) cache_report(c, kCacheBadPage, page_v, 0);
        const unsigned page = bad ? 0 : page_v;
        k_big = kmax[(int64_t)page * c.kv_heads];
        v_big = vmax[(int64_t)page * c.kv_heads];
        if (ONE_PAGE) {
            // one address for the workgroup, and offsets that stay
            const uint64_t at0 = (uint64_t)__builtin_amdgcn_readfirstlane(page) * page_codes;
            const int8_t* k = kbase + at0 + ((64 * x) & mask) * c.pitch;
            const int8_t* v = vbase + at0 + ((64 * x) & mask);
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const unsigned at = tid + kThreads * i;
                if (CHUNKS % kThreads == 0 || at < CHUNKS) {
                    kc[i] = *(const u32x4*)(k + at * 16u);
                    vc[i] = *(const u32x4*)(v + ((at >> 2) * (unsigned)c.page_tokens + 16u * (at & 3)));
                }
            }
        } else {
            const int8_t* v = vbase + (uint64_t)page * page_codes + ((64 * x + 16 * (tid & 3)) & mask);
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int at = tid + kThreads * i, key = at / KS, part = at % KS;
                const unsigned pk = (unsigned)page_k[i] < (unsigned)c.pages ? page_k[i] : 0;
                if (CHUNKS % kThreads == 0 || at < CHUNKS) {
                    kc[i] = *(const u32x4*)(kbase + (uint64_t)pk * page_codes + ((64 * x + key) & mask) * c.pitch + 16 * part);
                    vc[i] = *(const u32x4*)(v + (at >> 2) * c.page_tokens);
                }
            }
        }
    };
    auto stage = [&](int buf) {
        T* kl = k_lds[buf];
        _Float16* vl = v_lds[buf];
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int at = tid + kThreads * i, key = at / KS, part = at % KS;
            const int row = (key & 32) + 8 * ((key >> 2) & 3) + 4 * ((key >> 4) & 1) + (key & 3);
            if (CHUNKS % kThreads == 0 || at < CHUNKS) {
                V8* dst = (V8*)(kl + row * KPITCH + 16 * part);
                dst[0] = M::codes(kc[i][0], kc[i][1]);
                dst[1] = M::codes(kc[i][2], kc[i][3]);
            }
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int at = tid + kThreads * i;
            if (CHUNKS % kThreads == 0 || at < CHUNKS) {
                half8* dst = (half8*)(vl + (at >> 2) * VPITCH + 16 * (at & 3));
                dst[0] = codes_f16(vc[i][0], vc[i][1]);
                dst[1] = codes_f16(vc[i][2], vc[i][3]);
            }
        }
        if (tid < 4) {
            block_lds[buf][tid] = f32x4{k_big * fabsf(a.scale), lead_of(v_big), (float)block_kind(bad, v_big), 0.0f};
        }
    };

    float m = -INFINITY, D_max = -INFINITY, l = 0.0f;
    float D0 = -kLift;  // D as p takes it: less the lift, and a margin
    f32x16 o[DP];
#pragma unroll
    for (int i = 0; i < DP; i++) o[i] = f32x16{};

    auto compute = [&](int x, int buf) {
        const T* kl = k_lds[buf];
        const _Float16* vl = v_lds[buf];
        if (64 * x >= some_hi || 64 * x + 63 < some_lo) return;  // (the wave's rows see none of them)
        // Operands are read a group ahead of the products that use them.  (The
        // scheduler on its own reads two ahead, and every product then waits
        // for LDS.)
        f32x16 s[2];
        V8 kf[2][4];
        auto read_k = [&](int j) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
                    kf[j & 1][2 * u + b] = *(const V8*)(kl + (32 * b + col) * KPITCH + 16 * (2 * j + u) + 8 * h);
        };
        read_k(0);
#pragma unroll
        for (int j = 0; j < DP; j++) {
            if (j + 1 < DP) read_k(j + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int b = 0; b < 2; b++)
                    s[b] = M::mma(kf[j & 1][2 * u + b], q[2 * j + u], j + u ? s[b] : f32x16{});
            __builtin_amdgcn_sched_barrier(0);
        }
        half8 vf[2][DP];
        auto read_v = [&](int g) {
#pragma unroll
            for (int i = 0; i < DP; i++)
                vf[g & 1][i] = *(const half8*)(vl + (32 * i + col) * VPITCH + 32 * (g >> 1) + 16 * h + 8 * (g & 1));
        };
        read_v(0);
        const f32x4 block0 = block_lds[buf][h], block1 = block_lds[buf][2 + h];
        const float ks0 = block0[0], ks1 = block1[0];
        const bool odd = __any(block0[2] != kBlockUsual || block1[2] != kBlockUsual);
        const bool whole = 64 * x >= all_lo && 64 * x + 63 < all_hi && !odd;
        half8 p[2][2];
        float factor0 = ks0, factor1 = ks1;
        const int from = lo - 64 * x - 16 * h, to = hi - 64 * x - 16 * h;
        if (!whole) {
            // (the scale first: it may be zero or NaN, which a key that is not seen must not meet)
#pragma unroll
            for (int k = 0; k < 16; k++) {
                s[0][k] = k >= from && k < to && block0[2] != kBlockNone ? s[0][k] * ks0 : -INFINITY;
                s[1][k] = k + 32 >= from && k + 32 < to && block1[2] != kBlockNone ? s[1][k] * ks1 : -INFINITY;
            }
            factor0 = factor1 = 1.0f;
        }
        float top0 = s[0][0], top1 = s[1][0];
#pragma unroll
        for (int k = 1; k < 16; k++) {
            top0 = fmaxf(top0, s[0][k]);
            top1 = fmaxf(top1, s[1][k]);
        }
        top0 = rounded(top0 * factor0);
        top1 = rounded(top1 * factor1);
        float base = or_zero(m);
        const float top = max_halves(fmaxf(top0, top1));
        const float most = max_halves(fmaxf(top0 - base + block0[1], top1 - base + block1[1]));
        const bool move = top > m + kSlack || most > D_max + kSlack;
        if (__any(move)) {
            // (each row by itself: its result does not depend on the others)
            const float m2 = move ? fmaxf(m, top) : m, base2 = or_zero(m2), up = base2 - base;
            const float D2 = move ? fmaxf(D_max, most) - up : D_max;
            // (Large scores: p may pass what D says by the steps of the score and of
            // the shift below, 2^-23 of them together.  Up to 2^28 there is room.)
            const float margin = fminf(0x1p-22f * fabsf(base2), 30.0f), D3 = or_zero(D2) - kLift + margin;
            const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(D0 - up - D3);
#pragma unroll
            for (int i = 0; i < DP; i++) o[i] *= shrink;
            l *= __builtin_amdgcn_exp2f(m - base2);
            m = m2;
            D_max = D2;
            D0 = D3;
            base = base2;
        }
        const float scale[2] = {fmaxf(block0[1], D0 - kFar) - D0, fmaxf(block1[1], D0 - kFar) - D0};
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const float factor = b ? factor1 : factor0, shift = scale[b] - base;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const float e = __builtin_amdgcn_exp2f(s[b][k] * factor + shift);
                sum[b] += e;
                p[b][k >> 3][k & 7] = (_Float16)e;
            }
        }
        l += sum[0] * __builtin_amdgcn_exp2f(-scale[0]) + sum[1] * __builtin_amdgcn_exp2f(-scale[1]);
        if (odd) {
            int from2 = from, to2 = to;
            asm("" : "+v"(from2), "+v"(to2));  // (compared anew: nothing of this is kept for the usual step)
            const bool change0 = block0[2] >= kBlockPoison, change1 = block1[2] >= kBlockPoison;
            const _Float16 all0 = block0[2] == kBlockPoison ? (_Float16)NAN : (_Float16)0.0f;
            const _Float16 all1 = block1[2] == kBlockPoison ? (_Float16)NAN : (_Float16)0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                if (k >= from2 && k < to2 && change0) p[0][k >> 3][k & 7] = all0;
                if (k + 32 >= from2 && k + 32 < to2 && change1) p[1][k >> 3][k & 7] = all1;
            }
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {
            __builtin_amdgcn_sched_barrier(0);
            if (g < 3) read_v(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < DP; i++)
                o[i] = MmaF16::mma(vf[g & 1][i], p[g >> 1][g & 1], o[i]);
        }
    };

    if (c0 < c1) {
        look(c0);
        fetch(c0);
        look(c0 + 1);
        stage(0);
        fetch(c0 + 1);
        for (int x = c0; x < c1; x++) {
            // One barrier a step: what a step stages, the step before it has
            // read.  The last steps fetch and stage the last keys once more:
            // no branch here, after which every load on its way would be
            // waited for.
            const int buf = (x - c0) & 1;
            look(x + 2);
            __syncthreads();
            stage(buf ^ 1);
            fetch(x + 2);
            compute(x, buf);
        }
        __syncthreads();  // (the staged keys have been used)
    }

    const Parts mem(a);
    const int64_t tile = slot * c.kv_heads + kv;
    const int base_at = parts > 1 ? (int)(tile * a.splits) * (RT * OP * 4) : 0;
    l = sum_halves(l);
    const int row = wave_row + col;
    if (row < t.rows) {
        // (a part that saw no key joins as zeros)
        Unit unit(D0, l);
        if (parts > 1 && l == 0.0f) unit.a = 0.0f;
        const int at = base_at + (split * RT + row) * (OP * 4);
#pragma unroll
        for (int i = 0; i < DP; i++) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int k = 32 * i + 8 * u + 4 * h;
                const f32x4 y = unit(f32x4{o[i][4 * u], o[i][4 * u + 1], o[i][4 * u + 2], o[i][4 * u + 3]});
                if (parts > 1) mem.store(at + 4 * k, y);
                else store_out<T>(a, t, kv, d, row, k, y, m, l);
            }
        }
        if (parts > 1 && h == 0) mem.store(at + 4 * D, f32x2{m, l});
    }
    if (parts == 1) return;
    if (!last_part(&a.tickets[tile], parts)) return;
    static_assert(sizeof(k_lds) >= (4 * kThreads + kMaxSplits * RT) * 4 || D < 96, "");
    constexpr bool OVER = D >= 96;
    __shared__ float join_lds[OVER ? 1 : 4 * kThreads + kMaxSplits * RT];
    float* so = OVER ? (float*)k_lds : join_lds;
    join_parts<T, RT, D, kThreads, kMaxSplits>(
        a, t, kv, d, mem, [&](int s) { return base_at + s * (RT * OP * 4); }, parts, so, so + 4 * kThreads);
}

template <class E, int DP, int WAVES>
hipError_t launch_many(const CacheView& c, int64_t layer, const RaggedRows& r, AttendArgs a, hipStream_t s) {
    constexpr int OCC = DP <= 4 ? 2 : 1;  // waves a SIMD: wider heads need its registers
    constexpr int kThreads = 64 * WAVES, RT = WAVES * 32, OP = 32 * DP + 4;
    const int64_t slots = tile_slots(r.tokens, r.n, a.group, RT), tiles = slots * c.kv_heads;
    // about: keys that a tile sees in steps of 64, tiles that hold rows
    const int64_t each = (r.tokens + r.n - 1) / r.n;
    const int64_t keys = a.window > 0 && a.window + RT / a.group < a.longest ? a.window + RT / a.group : a.longest;
    const int64_t chunks = (keys + 63) / 64;
    int64_t live = r.n * ((each * a.group + RT - 1) / RT) * c.kv_heads;
    if (live > tiles) live = tiles;
    // Joining parts of 128 rows and more is dear (a prompt of 2048: 65 us whole,
    // 100 in two parts): only for tiles that leave compute units empty (4 of 30
    // tokens over 30000 keys: 381 us in two parts, 112 in 16).  A prompt of 1000
    // is near that line, and split: 49 us, whole 36.
    int64_t splits = OCC * 4 / WAVES * a.cus / live;
    if (splits > chunks / 8) splits = chunks / 8;
    const int64_t fit = a.partial_bytes / (tiles * RT * OP * 4);
    if (splits > fit) splits = fit;
    if (splits > kMaxSplits) splits = kMaxSplits;
    if (splits < 1 || tiles > a.ntickets) splits = 1;
    a.splits = (int)splits;
    const int64_t rounds = (chunks + splits - 1) / splits;
    a.rounds = rounds < 8 ? 8 : (int)rounds;
    const dim3 grid((unsigned)tiles, (unsigned)splits);
    if (c.page_tokens >= kKeys) attend_many_kernel<E, DP, WAVES, OCC, true><<<grid, kThreads, 0, s>>>(c, layer, r, a);
    else attend_many_kernel<E, DP, WAVES, OCC, false><<<grid, kThreads, 0, s>>>(c, layer, r, a);
    return hipGetLastError();
}

// Tiles of 256 rows stage the keys half as often; of 128, two of which fit a
// compute unit, they fill the card with fewer rows.  4 sequences of up to 4096,
// 32 heads over 8 (1400 tiles of 256): 651 us and 675; 8 of up to 512 (512): 74
// and 71; one of 2048 (256): 76 and 65; 4 of 30 tokens, 8 heads over 1 (16): 144
// and 112.
template <class E, int DP>
hipError_t launch_rows(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a, hipStream_t s) {
    const int64_t rows = ((int64_t)r.tokens + r.n - 1) / r.n * a.group;  // a sequence's, about
    if (DP <= 4 && r.n * ((rows + 255) / 256) * c.kv_heads > 2 * a.cus)
        return launch_many<E, DP, DP <= 4 ? 8 : 4>(c, layer, r, a, s);
    return launch_many<E, DP, 4>(c, layer, r, a, s);
}

template <class E>
hipError_t launch_width(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a, hipStream_t s) {
    switch (c.pitch / 32) {
        case 1: return launch_rows<E, 1>(c, layer, r, a, s);
        case 2: return launch_rows<E, 2>(c, layer, r, a, s);
        case 3: return launch_rows<E, 3>(c, layer, r, a, s);
        case 4: return launch_rows<E, 4>(c, layer, r, a, s);
        case 5: return launch_rows<E, 5>(c, layer, r, a, s);
        case 6: return launch_rows<E, 6>(c, layer, r, a, s);
        case 7: return launch_rows<E, 7>(c, layer, r, a, s);
        default: return launch_rows<E, 8>(c, layer, r, a, s);
    }
}

}  // namespace

hipError_t launch_attend_many(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                              hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F16) return launch_width<F16>(c, layer, r, a, s);
    return launch_width<Bf16>(c, layer, r, a, s);
}

}  // namespace manta
