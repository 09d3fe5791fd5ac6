// kernels_cache_attn.hip -- softmax(scale q k^T) v over the 8-bit cache, few
// rows at a time: a sequence's newest token, or a handful of them.
//
// Bytes bound: every code is read once for all query heads of its kv head
// (2 * head_dim bytes a key), and nothing else is large.  262145 keys of 8
// heads of 128 in 97 us: 5.55 TB/s.
#include "cache_attend.hpp"

namespace manta {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxSplits = 128;


// A load of what one tile of rows reads once (262145 keys of 8 heads of 128:
// 108 us without the hint, 97 with it; 64 ragged sequences of up to 8192: 145
// and 132).  Pages that branches share are read once a branch, and lose by it:
// 64 branches of 16000 tokens 195 us without, 257 with it; of 1000, 35 and 36.
template <bool ONCE, class V>
__device__ __forceinline__ V stream(const V* p) {
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}

struct Share {  // a workgroup's part of a tile's keys
    int kv;
    int c0, c1;         // the keys 64 c0 .. 64 c1 - 1,
    int first, step;    // of which wave w takes c0 + first + w, that + step, ...
    int part, parts;    // which of the tile's parts this is
    uint32_t* ticket;
    int at0, at1, pitch;  // where part 0 goes in a.partial (bytes), and parts 1, 2, ...
    __device__ __forceinline__ int at(int s) const { return s == 0 ? at0 : at1 + (s - 1) * pitch; }
};

// A tile of 16 QT rows (the query heads of a kv head, and tokens); 64 keys a
// wave at a time.  Scores are k q^T: lane (g, c) = (lane / 16, lane % 16)
// holds row c's scores of the 16 keys of block g, and those are what the
// product v^T p takes from that lane: p never leaves its registers.  Codes go
// from global memory to matrix operands without LDS: lane (g, c) reads 16
// bytes of key 16 (c / 4) + 4 T + c % 4 for tile T of the scores, and 16 keys
// of block g of column c for v.  A block lies in one page, so a lane's 16
// scores and weights share one scale each.
//
//   score = q.code * (k_max / 127 * scale * log2 e), weight = exp2(score - m),
//   out = sum(weight * v_max / 127 * code) / sum(weight)
//
// by way of p (cache_attend.hpp), m and D each wave's own, kept at every step.
constexpr float kLift = 15.0f;  // p is at most 2^15
// Scores past this, whose steps are 2^-8 and more, are rounded before m is
// taken from them: p must not pass 2^15 by such steps.
constexpr float kLarge = 65536.0f;
template <class E, int DP, int QT>
__device__ __forceinline__ void attend_share(const CacheView& c, int64_t layer, const AttendArgs& a, const Tile& t,
                                             const Share& sh) {
    typedef typename E::T T;
    typedef typename MmaOf<E>::M M;
    typedef typename M::V V8;
    constexpr int D = 32 * DP, DC = DP / 2, DT = 2 * DP, RT = 16 * QT, OP = D + 4;
    constexpr bool ODD = DP % 2 != 0;
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = sh.kv, c1 = sh.c1, parts = sh.parts;

    // the rows, clamped (the doubles are not stored), as operands
    const int d = c.head_dim;
    V8 q[QT][DP];
    int lo[QT], hi[QT];
    int lo_all = 0, hi_all = 0x7FFFFFFF;  // keys that every row sees
#pragma unroll
    for (int n = 0; n < QT; n++) {
        const int row = t.r0 + min(16 * n + col, t.rows - 1);
        const int token = row / a.group, head = kv * a.group + row % a.group;
        const int pos = t.length - t.count + token;
        lo[n] = key_begin(a, pos);
        hi[n] = key_end(a, t.length, pos);
        const T* src = (const T*)a.q + (int64_t)(t.row0 + token) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
        for (int s = 0; s < DP; s++) {
            const int at = ODD && s == DP - 1 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            V8 x;
            if (a.wide && at + 8 <= d) {
                x = *(const V8*)(src + at);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = at + j < d ? src[at + j] : (T)0.0f;
            }
            q[n][s] = a.scale < 0.0f ? -x : x;  // (the scores' order is that of the products)
        }
    }
    {
        // begin and end rise with the row
        const int first = t.length - t.count + t.r0 / a.group;
        const int last = t.length - t.count + (t.r0 + t.rows - 1) / a.group;
        lo_all = key_begin(a, last);
        hi_all = key_end(a, t.length, first);
    }

    const int32_t* table = c.tables + (int64_t)t.seq * c.table_pages;
    const int mask = c.page_tokens - 1, last_page = (t.end - 1) >> c.page_shift;
    const uint32_t page_codes = (uint32_t)c.page_codes();  // (at most 65535 * 128 * 256)
    const int64_t slab0 = c.slab(layer, 0), head_codes = (int64_t)kv * c.page_tokens * c.pitch;
    const int8_t* kbase = c.k_codes + slab0 * page_codes + head_codes;
    const int8_t* vbase = c.v_codes + slab0 * page_codes + head_codes;
    const float* kmax = c.k_max + slab0 * c.kv_heads + kv;
    const float* vmax = c.v_max + slab0 * c.kv_heads + kv;
    const int kb = col >> 2;  // the block of the keys whose k this lane reads

    u32x4 k16[4][DC > 0 ? DC : 1], v16[DT];
    u32x2 k8[4];
    int page_k = 0, page_v = 0;  // table entries of the next chunk
    float ks = 0.0f, vs = 0.0f;  // largest k and v of block g, of the chunk in registers
    bool bad = false;
    auto look = [&](int x) {
        x = min(x, c1 - 1);
        page_k = table[min((64 * x + 16 * kb) >> c.page_shift, last_page)];
        page_v = table[min((64 * x + 16 * g) >> c.page_shift, last_page)];
    };
    auto load_k = [&](int x) {
        const unsigned page = (unsigned)page_k < (unsigned)c.pages ? page_k : 0;
        const int8_t* p = kbase + (uint64_t)page * page_codes + (((64 * x + 16 * kb) & mask) + (col & 3)) * c.pitch;
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int s = 0; s < DC; s++) k16[i][s] = stream<QT == 1>((const u32x4*)(p + 4 * i * c.pitch + 64 * s + 16 * g));
            if (ODD) k8[i] = stream<QT == 1>((const u32x2*)(p + 4 * i * c.pitch + 64 * DC + 8 * g));
        }
    };
    auto load_v = [&](int x, int entry) {
        bad = (unsigned)entry >= (unsigned)c.pages;
        const unsigned page = bad ? 0 : entry;
        if (bad) cache_report(c, kCacheBadPage, entry, 0);
        ks = kmax[(int64_t)page * c.kv_heads];
        vs = vmax[(int64_t)page * c.kv_heads];
        const int8_t* p = vbase + (uint64_t)page * page_codes + ((64 * x + 16 * g) & mask) + col * c.page_tokens;
#pragma unroll
        for (int i = 0; i < DT; i++) v16[i] = stream<QT == 1>((const u32x4*)(p + 16 * i * c.page_tokens));
    };

    float m[QT], D_max[QT], l[QT];
    f32x4 o[QT][DT];
#pragma unroll
    for (int n = 0; n < QT; n++) {
        m[n] = D_max[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[n][i] = f32x4{0, 0, 0, 0};
    }

    const int step = sh.step;
    int x = sh.c0 + sh.first + wave;
    if (x < c1) {
        look(x);
        load_k(x);
        const int entry = page_v;
        look(x + step);
        load_v(x, entry);
    }
    for (; x < c1; x += step) {
        f32x4 s[QT][4];
#pragma unroll
        for (int j = 0; j < DP; j++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                V8 k;
                if (ODD && j == DP - 1) k = M::codes(k8[i][0], k8[i][1]);
                else k = M::codes(k16[i][j >> 1][2 * (j & 1)], k16[i][j >> 1][2 * (j & 1) + 1]);
#pragma unroll
                for (int n = 0; n < QT; n++) s[n][i] = M::mma(k, q[n][j], j ? s[n][i] : f32x4{0, 0, 0, 0});
            }
            __builtin_amdgcn_sched_barrier(0);  // (conversions that run far ahead would take all registers)
        }
        const bool more = x + step < c1;
        if (more) load_k(x + step);

        const float kscale = ks * fabsf(a.scale);
        const BlockKind kind = block_kind(bad, vs);
        const bool odd = __any(kind != kBlockUsual);
        const bool whole = 64 * x >= lo_all && 64 * x + 63 < hi_all && !odd;
        const float lead = lead_of(vs);
        half8 p[QT][2];
#pragma unroll
        for (int n = 0; n < QT; n++) {
            float e[16], top = -INFINITY, factor = kscale;
#pragma unroll
            for (int k = 0; k < 16; k++) e[k] = s[n][k >> 2][k & 3];
            const int from = bad ? 16 : lo[n] - (64 * x + 16 * g), to = hi[n] - (64 * x + 16 * g);
            if (!whole) {
                // (the scale first: it may be zero or NaN, which a key that is not seen must not meet)
#pragma unroll
                for (int k = 0; k < 16; k++) e[k] = k >= from && k < to ? e[k] * kscale : -INFINITY;
                factor = 1.0f;
            }
#pragma unroll
            for (int k = 0; k < 16; k++) top = fmaxf(top, e[k]);
            top = rounded(top * factor);
            const float m2 = fmaxf(m[n], max_quarters(top));
            float base = or_zero(m2);
            const float keep = __builtin_amdgcn_exp2f(m[n] - base);
            const float was = D_max[n] + (m[n] - base);
            const float D2 = fmaxf(was, max_quarters(top - base + lead));
            if (__any(D2 > was)) {
                const float shrink = __builtin_amdgcn_exp2f(was - or_zero(D2));
#pragma unroll
                for (int i = 0; i < DT; i++) o[n][i] *= shrink;
            }
            m[n] = m2;
            D_max[n] = D2;
            if (__any(fabsf(base) > kLarge)) {
#pragma unroll
                for (int k = 0; k < 16; k++) e[k] = rounded(e[k] * factor) - base;
                factor = 1.0f;
                base = 0.0f;
            }
            const float scale = fmaxf(lead, D2 - kFar) - or_zero(D2) + kLift, shift = scale - base;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                e[k] = __builtin_amdgcn_exp2f(e[k] * factor + shift);
                sum += e[k];
                p[n][k >> 3][k & 7] = (_Float16)e[k];
            }
            if (odd && (kind == kBlockPoison || kind == kBlockEmpty)) {
                const _Float16 all = kind == kBlockPoison ? (_Float16)NAN : (_Float16)0.0f;
#pragma unroll
                for (int k = 0; k < 16; k++)
                    if (k >= from && k < to) p[n][k >> 3][k & 7] = all;
            }
            l[n] = l[n] * keep + sum * __builtin_amdgcn_exp2f(-scale);
        }
#pragma unroll
        for (int i = 0; i < DT; i++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const half8 v = codes_f16(v16[i][2 * u], v16[i][2 * u + 1]);
#pragma unroll
                for (int n = 0; n < QT; n++) o[n][i] = MmaF16::mma(v, p[n][u], o[n][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (more) {
            // loads return in order: table entries ahead of the codes, so that
            // the next k need not wait for this v
            const int entry = page_v;
            look(x + 2 * step);
            load_v(x + step, entry);
        }
    }

    // the waves' results joined
    __shared__ float so[kWaves * RT * OP];
    __shared__ float sm[kWaves][RT], sD[kWaves][RT], sl[kWaves][RT];
#pragma unroll
    for (int n = 0; n < QT; n++) {
        l[n] = sum_quarters(l[n]);
        if (g == 0) {
            sm[wave][16 * n + col] = m[n];
            sD[wave][16 * n + col] = D_max[n];
            sl[wave][16 * n + col] = l[n];
        }
#pragma unroll
        for (int i = 0; i < DT; i++) *(f32x4*)&so[(wave * RT + 16 * n + col) * OP + 16 * i + 4 * g] = o[n][i];
    }
    __syncthreads();

    // 4 columns a thread: of the output, or of this part
    const Parts parts_mem(a);
    for (int i = threadIdx.x; i < t.rows * (D / 4); i += kThreads) {
        const int row = i / (D / 4), k = 4 * (i % (D / 4));
        float big = sm[0][row], lead = -INFINITY;
#pragma unroll
        for (int w = 1; w < kWaves; w++) big = fmaxf(big, sm[w][row]);
        const float base = or_zero(big);
#pragma unroll
        for (int w = 0; w < kWaves; w++) lead = fmaxf(lead, sD[w][row] + (sm[w][row] - base));
        float sum = 0.0f;
        f32x4 y = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            sum += __builtin_amdgcn_exp2f(sm[w][row] - base) * sl[w][row];
            y += *(const f32x4*)&so[(w * RT + row) * OP + k] *
                 __builtin_amdgcn_exp2f(sD[w][row] + (sm[w][row] - base) - or_zero(lead));
        }
        const Unit unit(or_zero(lead) - kLift, sum);
        if (parts > 1) {
            const int at = sh.at(sh.part) + row * (OP * 4);
            parts_mem.store(at + 4 * k, sum == 0.0f ? f32x4{0, 0, 0, 0} : unit(y));
            if (k == 0) parts_mem.store(at + 4 * D, f32x2{big, sum});
        } else {
            store_out<T>(a, t, kv, d, row, k, unit(y), big, sum);
        }
    }
    if (parts == 1) return;
    if (!last_part(sh.ticket, parts)) return;

    __shared__ float weight[kMaxSplits * RT];
    join_parts<T, RT, D, kThreads, kMaxSplits>(a, t, kv, d, parts_mem, [&](int s) { return sh.at(s); }, parts, so, weight);
}

// A workgroup a tile and part: parts of `rounds` steps or more.
template <class E, int DP, int QT>
__global__ __launch_bounds__(kThreads, DP * QT <= 6 ? 2 : 1) void attend_few_kernel(CacheView c, int64_t layer,
                                                                                  RaggedRows r, AttendArgs a) {
    constexpr int RT = 16 * QT, BYTES = RT * (32 * DP + 4) * 4;
    const Tile t = my_tile(c, r, a, blockIdx.x, RT);
    if (t.rows == 0) return;
    Share sh;
    sh.kv = blockIdx.y;
    sh.c0 = t.begin >> 6;
    sh.c1 = t.end > t.begin ? (t.end + 63) >> 6 : sh.c0;
    const int want = (sh.c1 - sh.c0 + kWaves * a.rounds - 1) / (kWaves * a.rounds);
    sh.parts = min(max(want, 1), a.splits);
    sh.part = blockIdx.z;
    if (sh.part >= sh.parts) return;
    sh.first = kWaves * sh.part;
    sh.step = kWaves * sh.parts;
    const int64_t tile = (int64_t)blockIdx.x * gridDim.y + sh.kv;
    sh.ticket = a.tickets + (sh.parts > 1 ? tile : 0);
    sh.at0 = sh.parts > 1 ? (int)(tile * a.splits) * BYTES : 0;
    sh.at1 = sh.at0 + BYTES;
    sh.pitch = BYTES;
    attend_share<E, DP, QT>(c, layer, a, t, sh);
}

// The same work cut evenly: one workgroup a place on the card, each with as
// many steps as the others of the sequences' steps laid end to end, whatever
// their lengths (64 sequences of up to 8192: 149 us by tiles, 131 so).  At
// most 64 sequences, one a lane, so that every workgroup can lay them out by
// itself.
template <class E, int DP, int QT>
__global__ __launch_bounds__(kThreads, DP * QT <= 6 ? 2 : 1) void attend_even_kernel(CacheView c, int64_t layer,
                                                                                   RaggedRows r, AttendArgs a) {
    constexpr int RT = 16 * QT, BYTES = RT * (32 * DP + 4) * 4;
    const int lane = threadIdx.x & 63, j = min(lane, r.n - 1);
    const int o0 = clamp_row(r.offsets[j], r.tokens), o1 = clamp_row(r.offsets[j + 1], r.tokens);
    // (tickets are counted for offsets that ascend)
    if (__any(o1 < o0)) {
        if (o1 < o0 && lane < r.n && blockIdx.x == 0 && threadIdx.x < 64) cache_report(c, kCacheBadOffsets, j, 0);
        return;
    }
    const int seq = r.seqs ? r.seqs[j] : j;
    const bool good = (unsigned)seq < (unsigned)c.seqs;
    const int length = good ? c.clamp_length(c.lengths[seq]) : 0;
    // a tile's steps of 64 kWaves keys (1 for one that sees nothing: its rows are zeros)
    int tiles = 0, steps = 1, c_lo = 0;
    if (lane < r.n && o1 > o0) {
        if (!good && blockIdx.x == 0 && threadIdx.x < 64) cache_report(c, kCacheBadSeq, seq, 0);
        tiles = tile_count(o0, o1, a.group, RT);
        c_lo = key_begin(a, length - (o1 - o0)) >> 6;
        steps = max(1, (((length + 63) >> 6) - c_lo + kWaves - 1) / kWaves);
    }
    int64_t below = (int64_t)tiles * steps;
    int tiles_below = tiles, most = steps;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const int64_t y = __shfl_up((long long)below, x);
        const int z = __shfl_up(tiles_below, x);
        if (lane >= x) {
            below += y;
            tiles_below += z;
        }
        most = max(most, __shfl_xor(most, x));
    }
    // (kept in LDS: the registers are for the keys)
    __shared__ int64_t s_below[64];
    __shared__ int s_from[64], s_count[64], s_seq[64], s_length[64], s_lo[64], s_steps[64], s_tiles[64];
    __shared__ int64_t s_total;
    __shared__ int s_all, s_most;
    if (threadIdx.x < 64) {
        s_below[lane] = tiles > 0 ? below - (int64_t)tiles * steps : INT64_MAX;
        s_from[lane] = o0;
        s_count[lane] = o1 - o0;
        s_seq[lane] = good ? seq : 0;
        s_length[lane] = length;
        s_lo[lane] = c_lo;
        s_steps[lane] = steps;
        s_tiles[lane] = tiles_below - tiles;
        if (lane == 63) {
            s_total = below;  // of a kv head
            s_all = tiles_below;
            s_most = most;
        }
    }
    __syncthreads();
    auto uniform = [](int64_t x) {
        const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 | lo);
    };
    if (!tiles_fit(s_all, c.kv_heads, a.ntickets)) return;
    const int64_t total = uniform(s_total), all = total * c.kv_heads;
    // each workgroup's steps: no tile in more parts than can be joined
    const int64_t quota = uniform(max((all + gridDim.x - 1) / gridDim.x, (int64_t)(s_most / (kMaxSplits - 2) + 1)));
    int64_t at = blockIdx.x * quota;
    const int64_t end = min(at + quota, all);
    while (at < end) {
        const int kv = __builtin_amdgcn_readfirstlane((int)(at / total));
        const int64_t rest = at - kv * total;
        const int i = 63 - __clzll(__ballot(s_below[lane] <= rest) | 1ull);
        const int n = __builtin_amdgcn_readfirstlane(s_steps[i]);
        const int64_t in = rest - uniform(s_below[i]);
        const int ordinal = __builtin_amdgcn_readfirstlane((int)(in / n));
        const int s0 = (int)(in - (int64_t)ordinal * n);
        const int s1 = (int)min((int64_t)n, s0 + (end - at));
        const int64_t from = at - s0;  // the tile's first step
        Tile t{};
        t.row0 = __builtin_amdgcn_readfirstlane(s_from[i]);
        t.count = __builtin_amdgcn_readfirstlane(s_count[i]);
        t.seq = __builtin_amdgcn_readfirstlane(s_seq[i]);
        t.length = __builtin_amdgcn_readfirstlane(s_length[i]);
        t.r0 = ordinal * RT;
        t.rows = (int)min((int64_t)RT, (int64_t)t.count * a.group - t.r0);
        t.end = key_end(a, t.length, t.length - t.count + (t.r0 + t.rows - 1) / a.group);
        t.begin = key_begin(a, t.length - t.count + t.r0 / a.group);
        Share sh;
        sh.kv = kv;
        const int lo = __builtin_amdgcn_readfirstlane(s_lo[i]);
        sh.c0 = lo + kWaves * s0;
        sh.c1 = min(lo + kWaves * s1, t.end > t.begin ? (t.end + 63) >> 6 : 0);
        sh.first = 0;
        sh.step = kWaves;
        const int64_t w0 = uniform(from / quota), w1 = uniform((from + n - 1) / quota);
        sh.part = (int)(blockIdx.x - w0);
        sh.parts = (int)(w1 - w0 + 1);
        sh.ticket = a.tickets + ((int64_t)kv * s_all + __builtin_amdgcn_readfirstlane(s_tiles[i]) + ordinal);
        // a workgroup leaves at most two parts: that of the tile it begins with,
        // and that of the one it begins
        sh.at0 = (int)(2 * w0 + (from > w0 * quota ? 1 : 0)) * BYTES;
        sh.at1 = (int)(2 * (w0 + 1)) * BYTES;
        sh.pitch = 2 * BYTES;
        attend_share<E, DP, QT>(c, layer, a, t, sh);
        at += s1 - s0;
        __syncthreads();  // (this tile's results have left LDS)
    }
}

template <class E, int DP, int QT>
hipError_t launch_few(const CacheView& c, int64_t layer, const RaggedRows& r, AttendArgs a, hipStream_t s) {
    constexpr int RT = 16 * QT, OP = 32 * DP + 4;
    const int64_t slots = tile_slots(r.tokens, r.n, a.group, RT), tiles = slots * c.kv_heads;
    // about: keys that a tile sees in steps of 64, tiles that hold rows
    const int64_t each = (r.tokens + r.n - 1) / r.n;
    const int64_t keys = a.window > 0 && a.window + each < a.longest ? a.window + each : a.longest;
    const int64_t chunks = (keys + 63) / 64;
    int64_t live = r.n * ((each * a.group + RT - 1) / RT) * c.kv_heads;
    if (live > tiles) live = tiles;
    // Two workgroups fit a compute unit (of heads wider than 128 or 32 rows,
    // one).  One sequence: as many as that, all with the same work (262145
    // keys of 8 heads of 128: 104 us, with twice as many 113).  Several, of
    // lengths that the host does not know: twice as many, so that what the
    // longest leave is small.  (That holds for windows too, where all steps are
    // alike: 16 of 5 tokens of 6 heads of 96 a kv head, the last 4096 keys: 40.1
    // us, with half as many 41.5.)
    constexpr int RESIDENT = DP * QT <= 6 ? 2 : 1;
    int64_t splits = ((r.n == 1 ? 1 : 2) * RESIDENT * a.cus + live - 1) / live;
    if (splits > (chunks + kWaves - 1) / kWaves) splits = (chunks + kWaves - 1) / kWaves;
    // joining costs as much as two steps (300 keys: 8.6 us alone, 9.9 in two
    // parts; 1000: 9.8 in two, 8.8 in four)
    if (chunks <= 2 * kWaves) splits = 1;
    const int64_t fit = a.partial_bytes / (tiles * RT * OP * 4);
    if (splits > fit) splits = fit;
    if (splits > kMaxSplits) splits = kMaxSplits;
    if (splits < 1 || tiles > a.ntickets) splits = 1;
    a.splits = (int)splits;
    // Several sequences, of lengths that may differ, and enough steps for every
    // place on the card (6 of heads of 128, 12 of 64, as their bytes go): cut
    // evenly.  64 sequences of up to 8192, 8 heads of 128: 131 us against 149;
    // 12: 41 against 44, and 8 (4 steps) 35.1 against 34.5; 20 of 16 heads of
    // 64 (13 steps): 54 against 58, and 32 of up to 4000 (11) 45.8 against 44.3.
    // Windows (64 sequences, 4096 keys: 104 against 115; 1024: 41 against 44, not
    // taken) and tiles of 32 rows (32 of 8 tokens, up to 4000 keys: 75 against
    // 100; 8 of 7, not taken: 37.4 against 36.2) lie on the same line within 7%.
    constexpr int PLACES = DP <= 2 && QT == 1 ? 3 : RESIDENT;
    const int64_t places = (int64_t)PLACES * a.cus;
    if (r.n > 1 && r.n <= 64 && tiles <= a.ntickets &&
        live * ((chunks + kWaves - 1) / kWaves) * DP >= 22 * places && 2 * places * RT * OP * 4 <= a.partial_bytes) {
        attend_even_kernel<E, DP, QT><<<(unsigned)places, kThreads, 0, s>>>(c, layer, r, a);
        return hipGetLastError();
    }
    const int64_t rounds = (chunks + kWaves * splits - 1) / (kWaves * splits);
    // wide heads have more to join (8 sequences of up to 8000, 2 heads of 256: 33
    // us with steps of 1, 25 of 2, 28 of 3; one sequence: 20, 22, 25)
    constexpr int LEAST = DP <= 4 ? 1 : 3;
    a.rounds = rounds < LEAST ? LEAST : (int)rounds;
    attend_few_kernel<E, DP, QT><<<dim3((unsigned)slots, c.kv_heads, (unsigned)splits), kThreads, 0, s>>>(c, layer, r, a);
    return hipGetLastError();
}

template <class E, int QT>
hipError_t launch_width(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a, hipStream_t s) {
    switch (c.pitch / 32) {
        case 1: return launch_few<E, 1, QT>(c, layer, r, a, s);
        case 2: return launch_few<E, 2, QT>(c, layer, r, a, s);
        case 3: return launch_few<E, 3, QT>(c, layer, r, a, s);
        case 4: return launch_few<E, 4, QT>(c, layer, r, a, s);
        case 5: return launch_few<E, 5, QT>(c, layer, r, a, s);
        case 6: return launch_few<E, 6, QT>(c, layer, r, a, s);
        case 7: return launch_few<E, 7, QT>(c, layer, r, a, s);
        default: return launch_few<E, 8, QT>(c, layer, r, a, s);
    }
}

template <class E>
hipError_t launch_rows(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a, hipStream_t s) {
    const int64_t rows = ((int64_t)r.tokens * a.group + r.n - 1) / r.n;  // a sequence's, about
    if (rows <= 16) return launch_width<E, 1>(c, layer, r, a, s);
    // (8 sequences of up to 16000, 64 rows each: 85 us in two tiles here, 89
    // staged once there; 32 of up to 8000, 40 rows each: 124 either way)
    if (rows <= 32) return launch_width<E, 2>(c, layer, r, a, s);
    return launch_attend_many(c, layer, r, a, s);
}

}  // namespace

hipError_t launch_cache_attention(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                                  hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F16) return launch_rows<F16>(c, layer, r, a, s);
    return launch_rows<Bf16>(c, layer, r, a, s);
}

}  // namespace manta
