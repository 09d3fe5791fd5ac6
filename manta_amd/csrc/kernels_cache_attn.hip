// kernels_cache_attn.hip -- softmax(scale q k^T) v over the 8-bit cache, few
// rows at a time: a sequence's newest token, or a handful of them.
//
// Bytes bound: every code is read once for all query heads of its kv head
// (2 * head_dim bytes a key), and nothing else is large.
#include "cache_attend.hpp"

namespace manta {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxSplits = 128;

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
//   out = R / 127 * sum(weight * (v_max / R) * code) / sum(weight)
//
// with m the running maximum and R at least the largest v_max so far: weight *
// (v_max / R) is at most 1 and is rounded to f16 (half a step, 2^-11, as the
// operand of an f32 sum; codes are exact).  The pages' own scales would leave
// f16's range, and the codes times them would be rounded once more.
template <class E, int DP, int QT>
__global__ __launch_bounds__(kThreads, DP * QT <= 6 ? 2 : 1) void attend_few_kernel(CacheView c, int64_t layer, RaggedRows r, AttendArgs a) {
    typedef typename E::T T;
    typedef typename MmaOf<E>::M M;
    typedef typename M::V V8;
    constexpr int D = 32 * DP, DC = DP / 2, DT = 2 * DP, RT = 16 * QT, OP = D + 4;
    constexpr bool ODD = DP % 2 != 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int kv = blockIdx.y, split = blockIdx.z;
    const Tile t = my_tile(c, r, a, blockIdx.x, RT);
    if (t.rows == 0) return;
    const int c0 = t.begin >> 6, c1 = t.end > t.begin ? (t.end + 63) >> 6 : c0;
    // workgroups that share the keys, `rounds` steps of theirs or more for each
    const int want = (c1 - c0 + kWaves * a.rounds - 1) / (kWaves * a.rounds);
    const int parts = min(max(want, 1), a.splits);
    if (split >= parts) return;

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
            q[n][s] = x;
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
    const int64_t page_codes = c.page_codes(), slab0 = c.slab(layer, 0), head_codes = (int64_t)kv * c.page_tokens * c.pitch;
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
        const int page = (unsigned)page_k < (unsigned)c.pages ? page_k : 0;
        const int8_t* p = kbase + page * page_codes + (((64 * x + 16 * kb) & mask) + (col & 3)) * c.pitch;
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int s = 0; s < DC; s++) k16[i][s] = *(const u32x4*)(p + 4 * i * c.pitch + 64 * s + 16 * g);
            if (ODD) k8[i] = *(const u32x2*)(p + 4 * i * c.pitch + 64 * DC + 8 * g);
        }
    };
    auto load_v = [&](int x) {
        bad = (unsigned)page_v >= (unsigned)c.pages;
        const int page = bad ? 0 : page_v;
        if (bad) cache_report(c, kCacheBadPage, page_v, 0);
        ks = kmax[(int64_t)page * c.kv_heads];
        vs = vmax[(int64_t)page * c.kv_heads];
        const int8_t* p = vbase + page * page_codes + ((64 * x + 16 * g) & mask) + col * c.page_tokens;
#pragma unroll
        for (int i = 0; i < DT; i++) v16[i] = *(const u32x4*)(p + 16 * i * c.page_tokens);
    };

    float m[QT], l[QT], R = 0.0f;
    f32x4 o[QT][DT];
#pragma unroll
    for (int n = 0; n < QT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[n][i] = f32x4{0, 0, 0, 0};
    }

    const int step = kWaves * parts;
    int x = c0 + wave + kWaves * split;
    if (x < c1) {
        look(x);
        load_k(x);
        load_v(x);
        look(x + step);
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

        const float kscale = ks * a.scale;
        const bool any_bad = __any(bad);
        const bool whole = 64 * x >= lo_all && 64 * x + 63 < hi_all && !any_bad;
        const float R2 = fmaxf(R, max_quarters(finite_or_zero(bad ? 0.0f : vs)));
        const float w = R2 > 0.0f ? vs / R2 : vs;
        const float shrink = R2 > R ? R / R2 : 1.0f;
        R = R2;
        half8 p[QT][2];
#pragma unroll
        for (int n = 0; n < QT; n++) {
            float e[16], top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                e[k] = s[n][k >> 2][k & 3] * kscale;
                if (!whole) {
                    const int key = 64 * x + 16 * g + k;
                    if (key < lo[n] || key >= hi[n] || bad) e[k] = -INFINITY;
                }
                top = fmaxf(top, e[k]);
            }
            const float m2 = fmaxf(m[n], max_quarters(top));
            const float base = m2 == -INFINITY ? 0.0f : m2;
            const float keep = __builtin_amdgcn_exp2f(m[n] - base);
            if (__any(m2 > m[n] || shrink != 1.0f)) {
#pragma unroll
                for (int i = 0; i < DT; i++) o[n][i] *= keep * shrink;
            }
            m[n] = m2;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                e[k] = __builtin_amdgcn_exp2f(e[k] - base);
                sum += e[k];
                float f = e[k] * w;
                if (!whole) {
                    // nothing of a page that the row does not see, not even its NaN
                    const int key = 64 * x + 16 * g + k;
                    if (key < lo[n] || key >= hi[n] || bad) f = 0.0f;
                }
                p[n][k >> 3][k & 7] = (_Float16)f;
            }
            l[n] = l[n] * keep + sum;
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
            load_v(x + step);
            look(x + 2 * step);
        }
    }

    // the waves' results joined, one after the other
    __shared__ float so[RT * OP];
    __shared__ float sm[kWaves][RT], sl[kWaves][RT], sR[kWaves];
    __shared__ float top_m[RT], top_l[RT];
    __shared__ int last;
#pragma unroll
    for (int n = 0; n < QT; n++) {
        l[n] = sum_quarters(l[n]);
        if (g == 0) {
            sm[wave][16 * n + col] = m[n];
            sl[wave][16 * n + col] = l[n];
        }
    }
    if (lane == 0) sR[wave] = R;
    __syncthreads();
    float R2 = sR[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) R2 = fmaxf(R2, sR[w]);
    if (threadIdx.x < RT) {
        float big = sm[0][threadIdx.x], sum = 0.0f;
        for (int w = 1; w < kWaves; w++) big = fmaxf(big, sm[w][threadIdx.x]);
        const float base = big == -INFINITY ? 0.0f : big;
        for (int w = 0; w < kWaves; w++) sum += sl[w][threadIdx.x] * __builtin_amdgcn_exp2f(sm[w][threadIdx.x] - base);
        top_m[threadIdx.x] = big;
        top_l[threadIdx.x] = sum;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; w++) {
        if (w == wave) {
#pragma unroll
            for (int n = 0; n < QT; n++) {
                const float big = top_m[16 * n + col];
                const float f = __builtin_amdgcn_exp2f(m[n] - (big == -INFINITY ? 0.0f : big)) * (R2 > 0.0f ? R / R2 : 1.0f);
#pragma unroll
                for (int i = 0; i < DT; i++) {
                    f32x4* at = (f32x4*)&so[(16 * n + col) * OP + 16 * i + 4 * g];
                    const f32x4 y = o[n][i] * f;
                    *at = w == 0 ? y : *at + y;
                }
            }
        }
        __syncthreads();
    }

    const int64_t tile = (int64_t)blockIdx.x * gridDim.y + kv;
    const float unit = R2 / 127.0f;
    if (parts > 1) {
        float* part = a.partial + (tile * a.splits + split) * RT * OP;
        for (int i = threadIdx.x; i < t.rows * D; i += kThreads) {
            const int row = i / D, k = i % D;
            const float sum = top_l[row];
            part_store(part + row * OP + k, sum == 0.0f ? 0.0f : so[row * OP + k] / sum * unit);
        }
        if (threadIdx.x < t.rows) {
            part_store(part + threadIdx.x * OP + D, top_m[threadIdx.x]);
            part_store(part + threadIdx.x * OP + D + 1, top_l[threadIdx.x]);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0)
            last = __hip_atomic_fetch_add(&a.tickets[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                   (uint32_t)(parts - 1);
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0)
            __hip_atomic_store(&a.tickets[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // the parts in their order, whichever workgroup came last
        __shared__ float weight[kMaxSplits * RT];
        part = a.partial + tile * a.splits * RT * OP;
        if (threadIdx.x < t.rows) {
            float big = -INFINITY, sum = 0.0f;
            for (int s = 0; s < parts; s++) big = fmaxf(big, part_load(part + (s * RT + threadIdx.x) * OP + D));
            const float base = big == -INFINITY ? 0.0f : big;
            for (int s = 0; s < parts; s++) {
                const float* e = part + (s * RT + threadIdx.x) * OP + D;
                const float w = part_load(e + 1) * __builtin_amdgcn_exp2f(part_load(e) - base);
                weight[s * RT + threadIdx.x] = w;
                sum += w;
            }
            top_m[threadIdx.x] = big;
            top_l[threadIdx.x] = sum;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < t.rows * D; i += kThreads) {
            const int row = i / D, k = i % D;
            float sum = 0.0f;
            for (int s = 0; s < parts; s++) sum += weight[s * RT + row] * part_load(part + (s * RT + row) * OP + k);
            so[row * OP + k] = sum;
        }
        __syncthreads();
    }
    const float factor = parts > 1 ? 1.0f : unit;
    constexpr int WIDE = 8;
    const int pieces = (d + WIDE - 1) / WIDE;
    for (int i = threadIdx.x; i < t.rows * pieces; i += kThreads) {
        const int row = i / pieces, at = WIDE * (i % pieces);
        const int rr = t.r0 + row, token = rr / a.group, head = kv * a.group + rr % a.group;
        const int pos = t.length - t.count + token;
        const bool none = key_begin(a, pos) >= key_end(a, t.length, pos);
        T* dst = (T*)a.out + (int64_t)(t.row0 + token) * a.o_token + (int64_t)head * a.o_head + at;
        const float sum = top_l[row];
        V8 y;
#pragma unroll
        for (int j = 0; j < WIDE; j++) {
            const float v = so[row * OP + at + j] / sum * factor;
            y[j] = E::store(none ? 0.0f : v);
        }
        if (a.wide && at + WIDE <= d) {
            *(V8*)dst = y;
        } else {
            for (int j = 0; j < WIDE; j++)
                if (at + j < d) dst[j] = y[j];
        }
        if (a.lse && at == 0)
            a.lse[(int64_t)(t.row0 + token) * a.heads + head] =
                none ? -INFINITY : (top_m[row] + __builtin_amdgcn_logf(sum)) * 0.693147180559945f;
    }
}

template <class E, int DP, int QT>
hipError_t launch_few(const CacheView& c, int64_t layer, const RaggedRows& r, AttendArgs a, hipStream_t s) {
    constexpr int RT = 16 * QT, OP = 32 * DP + 4;
    const int64_t slots = tile_slots(r.tokens, r.n, a.group, RT), tiles = slots * c.kv_heads;
    const int64_t chunks = ((int64_t)a.longest + 63) / 64;
    int64_t splits = (4 * a.cus + tiles - 1) / tiles;
    splits = splits < (chunks + kWaves - 1) / kWaves ? splits : (chunks + kWaves - 1) / kWaves;
    const int64_t fit = a.partial_bytes / (tiles * RT * OP * 4);
    if (splits > fit) splits = fit;
    if (splits > kMaxSplits) splits = kMaxSplits;
    if (splits < 1 || tiles > a.ntickets) splits = 1;
    a.splits = (int)splits;
    const int64_t rounds = (chunks + kWaves * splits - 1) / (kWaves * splits);
    a.rounds = rounds < 1 ? 1 : (int)rounds;
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
    return launch_width<E, 2>(c, layer, r, a, s);
}

}  // namespace

hipError_t launch_cache_attention(const CacheView& c, int64_t layer, const RaggedRows& r, const AttendArgs& a,
                                  hipStream_t s) {
    if (a.dtype == MANTA_ROCM_F16) return launch_rows<F16>(c, layer, r, a, s);
    return launch_rows<Bf16>(c, layer, r, a, s);
}

}  // namespace manta
