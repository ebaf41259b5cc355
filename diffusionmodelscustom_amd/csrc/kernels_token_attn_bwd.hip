// Backward pass of danra_token_attention_* (token_attn.h has the formulas and the layout), from q, k, v, out, dout and each row's
// maximum and sum, without the score matrix in memory and without atomics:
//   delta = rowsum(dout . out)
//   p = 2^(score2 - m - log2 l),  dP = dout v^T,  dS = p (dP - delta) (1 - tanh^2)
//   dv = p^T dout,  dk = scale dS^T q,  dq = scale dS k
// One kernel owns query rows and sums dq over the keys, one owns keys and sums dk and dv over the rows of all the heads that share
// them; both form S and dP again (seven products of the size of S instead of five, for sums in a fixed order).  All sums are float32.
// P and dS are rounded to the operand's type for their products: 2^-9 relative in bfloat16, of the size of the rounding of the inputs.
// Half precision has no exponents for that: there P is kept times 2^12 (at most 2^12), and dS times a power of two of its column
// that falls when a tile brings larger values (the accumulator is rescaled then), the largest values lying between 2^10 and 2^14.
#include "token_attn.h"

namespace danra {
namespace token {

namespace {

constexpr int kRun = 16;  // tiles of 32 rows that are worth a workgroup and a partial result of their own

// p = 2^(score2 - m - log2 l).  In float32 the two are subtracted one after the other: m is itself a score of the row, so the first
// difference is small where p counts, while m + log2 l rounds at the size of m (2^-20 at m = 16, which p would have as relative error).
// That is far below the rounding of a two-byte P: there it is one number.
template <typename T>
struct Power {
    float m, lg;
    __device__ __forceinline__ explicit Power(float2 s) : m(sizeof(T) == 2 ? s.x + s.y : s.x), lg(s.y) {}
    __device__ __forceinline__ float operator()(float score2) const {
        if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(score2 - m);
        else return __builtin_amdgcn_exp2f(score2 - m - lg);
    }
};

// the power of two that a column's dS carries in half precision
struct Fit {
    float s = 0x1p60f;
    // c: the tile's dS; acc: what has been summed with the old power.  Multiplies both by what they need.
    template <int DT>
    __device__ __forceinline__ void apply(f32x16& c, f32x16 (&acc)[DT]) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(c[e]));
        top = pair_max(top);
        if (__any(top * s > 16384.f)) {
            if (top * s > 16384.f) {
                const float now = __builtin_amdgcn_ldexpf(1.f, min(60, max(-110, 11 - __builtin_amdgcn_frexp_expf(top))));
                const float keep = now / s;
                s = now;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[d][e] *= keep;
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] *= s;
    }
};

// delta[b][hk][r]: 16 lanes a row
template <typename T>
__global__ __launch_bounds__(256) void k_token_attn_delta(const TokenAttnArgs a) {
    const int total = a.Lq * a.G;
    const long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= (long long)a.B * a.Hk * total) return;  // (whole groups of 16 lanes)
    const int bh = (int)(item / total), r = (int)(item - (long long)bh * total);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const Rows rows{a.G, a.magic};
    const int query = rows.query(r), head = hk * a.G + r - query * a.G;
    const T* o = static_cast<const T*>(a.out) + (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D;
    const T* g = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0] + (long long)query * a.g_stride[1] + (long long)head * a.g_stride[2];
    const T* rest = a.rest ? static_cast<const T*>(a.rest) + (o - static_cast<const T*>(a.out)) : nullptr;
    const int c = threadIdx.x & 15;
    float sum = 0.f;
    if (c * 8 < a.D) {
        typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const T4 x = reinterpret_cast<const T4*>(o + 8 * c)[h], y = reinterpret_cast<const T4*>(g + 8 * c)[h];
            T4 r = {};
            if (rest) r = reinterpret_cast<const T4*>(rest + 8 * c)[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fmaf((float)x[e] + (float)r[e], (float)y[e], sum);
        }
    }
#pragma unroll
    for (int n = 8; n; n >>= 1) sum += __shfl_xor(sum, n);
    if (c == 0) a.delta[item] = a.stats[item].x == INFINITY ? 0.f : sum;
}

template <typename T, int DK>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DK >= 64 ? 1 : 2) void k_token_attn_dq(const TokenAttnArgs a) {
    typedef Tile<T, DK> Tl;
    typedef Type<T> Ty;
    constexpr int KS = DK / 16, DT = (DK + 31) / 32, kKeys = 32, kTile = kKeys * Tl::kRowBytes;
    __shared__ __align__(16) char lds[2 * 2 * kTile];
    __shared__ int ids[2][kKeys];
    __shared__ int shared_range[4][3];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const Rows rows{a.G, a.magic};
    const int total = a.Lq * a.G;
    int tile, bh;
    place(a.B * a.Hk, tile, bh);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    if (a.causal) tile = (total + 127) / 128 - 1 - tile;
    const int row = tile * 128 + wave * 32 + col;

    const Mask mask = make_mask(a, b);
    const int query = rows.query(min(row, total - 1)), head = hk * a.G + (min(row, total - 1) - query * a.G);
    const float2 stats = row < total ? a.stats[(size_t)bh * total + row] : make_float2(INFINITY, 0.f);
    const float delta = row < total ? a.delta[(size_t)bh * total + row] : 0.f;
    const bool used = stats.x != INFINITY;  // (false: the row sees no key)
    const int limit = used ? max(mask.limit(query), 0) : 0;
    const int doc = a.q_docs ? a.q_docs[(size_t)b * a.Lq + query] : 0;
    const int where = query + mask.shift;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
    const Score score = make_score<T>(a);
    const Power<T> power(stats);

    const int wave_limit = wave_max(limit), lowest = wave_min(limit);
    int id_lo = 0, id_hi = 0;
    if (a.q_docs) {
        id_lo = wave_min(limit > 0 ? doc : 0x7fffffff);
        id_hi = wave_max(limit > 0 ? doc : -1);
    }
    const bool one_id = id_lo == id_hi;
    if (lane == 0) {
        shared_range[wave][0] = wave_limit;
        shared_range[wave][1] = id_lo;
        shared_range[wave][2] = id_hi;
    }
    __syncthreads();
    int list_limit = wave_limit, list_lo = id_lo, list_hi = id_hi;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        list_limit = max(list_limit, shared_range[w][0]);
        list_lo = min(list_lo, shared_range[w][1]);
        list_hi = max(list_hi, shared_range[w][2]);
    }

    typename Ty::Frag qf[KS], gf[KS];
    {
        const T* q = static_cast<const T*>(a.q) + (long long)b * a.q_stride[0] + (long long)query * a.q_stride[1] + (long long)head * a.q_stride[2];
        const T* g = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0] + (long long)query * a.g_stride[1] + (long long)head * a.g_stride[2];
        load_owner<T, DK>(qf, used ? q : nullptr, a.D, lane);
        load_owner<T, DK>(gf, used ? g : nullptr, a.D, lane);
    }
    const T* kbase = static_cast<const T*>(a.k) + (long long)b * a.k_stride[0] + (long long)hk * a.k_stride[2];
    const T* vbase = static_cast<const T*>(a.v) + (long long)b * a.v_stride[0] + (long long)hk * a.v_stride[2];
    const int* kdocs = a.k_docs ? a.k_docs + (size_t)b * a.Lk : nullptr;
    const int4* ranges = a.k_ranges ? a.k_ranges + (size_t)b * ((a.Lk + kKeys - 1) / kKeys) : nullptr;

    f32x16 dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = f32x16{};
    Fit fit;

    TileList list;
    list.start(ranges, list_lo, list_hi, 0, (list_limit + kKeys - 1) / kKeys, lane);
    Fetch<T, DK, kKeys, 256> fk, fv;
    int next_id = 0;
    auto fetch = [&](int t) {
        const int k0 = t * kKeys;
        auto usable = [&](int r) { return k0 + r < mask.kv_len && !(kdocs && kdocs[k0 + r] < 0); };
        fk.load([&](int r) { return usable(r) ? kbase + (long long)(k0 + r) * a.k_stride[1] : nullptr; }, a.D, tid);
        fv.load([&](int r) { return usable(r) ? vbase + (long long)(k0 + r) * a.v_stride[1] : nullptr; }, a.D, tid);
        if (kdocs && tid < kKeys) next_id = k0 + tid < mask.kv_len ? kdocs[k0 + tid] : -1;
    };
    auto put = [&](int buf) {
        char* to = lds + buf * 2 * kTile;
        fk.store(to, tid);
        fv.store(to + kTile, tid);
        if (kdocs && tid < kKeys) ids[buf][tid] = next_id;
    };

    int t = list.next(lane), buf = 0;
    if (t >= 0) {
        fetch(t);
        put(0);
        __syncthreads();
    }
    while (t >= 0) {
        const int after = list.next(lane);
        if (after >= 0) fetch(after);
        const int k0 = t * kKeys;
        if (k0 < wave_limit) {
            const char* kt = lds + buf * 2 * kTile;
            const char* vt = kt + kTile;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                s = Ty::mfma(Tl::row(kt, col, 16 * c + 8 * half), qf[c], s);
                dp = Ty::mfma(Tl::row(vt, col, 16 * c + 8 * half), gf[c], dp);
            }
            const bool whole = k0 + kKeys <= lowest;
            bool same = true;
            if (kdocs) {
                const int4 g = ranges[t];
                same = one_id && g.z && g.x == id_lo;
            }
            // dp becomes (dP - delta) times the slope of the cap, s the score
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] -= delta;
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = bend<T>(s[e], score);
                    s[e] = score.out * x;
                    dp[e] *= bend_slope<T>(x);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= score.in;
            }
            const int j0 = k0 + 4 * half;
            if (a.slopes) {
                const float from = (float)(where - j0);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(from - (float)(8 * (e >> 2) + (e & 3))), s[e]);
            }
            unsigned seen = 0xffffu;
            if (!whole) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) seen |= j0 + 8 * (e >> 2) + (e & 3) < limit ? 1u << e : 0u;
            }
            if (!same) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 d = *reinterpret_cast<const int4*>(&ids[buf][4 * half + 8 * g]);
                    seen &= ~((d.x != doc ? 1u << (4 * g) : 0u) | (d.y != doc ? 2u << (4 * g) : 0u) | (d.z != doc ? 4u << (4 * g) : 0u) |
                              (d.w != doc ? 8u << (4 * g) : 0u));
                }
            }
            if (whole && same) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = power(s[e]) * dp[e];
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = seen >> e & 1 ? power(s[e]) * dp[e] : 0.f;
            }
            if constexpr (Ty::kNarrow) fit.apply<DT>(s, dq);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const typename Ty::Frag ds = round_frag<T>(s, h);
#pragma unroll
                for (int d = 0; d < DT; ++d) dq[d] = Ty::mfma(Tl::column(kt, 16 * h, 32 * d, lane), ds, dq[d]);
            }
        }
        if (after >= 0) {
            put(buf ^ 1);
            __syncthreads();
        }
        buf ^= 1;
        t = after;
    }

    if (row < total) {
        const float by = Ty::kNarrow ? a.scale / fit.s : a.scale;
        T* to = static_cast<T*>(a.dq) + (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * half;
                if (c < a.D) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    T4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = (T)(used ? dq[d][4 * g + e] * by : 0.f);
                    *reinterpret_cast<T4*>(to + c) = x;
                }
            }
    }
}

// rows of a streamed tile
struct RowFacts {
    float m[32], lg[32], delta[32], slope[32];  // (m, lg: as in Power)
    int limit[32], doc[32], where[32];
};

template <typename T, int DK>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DK >= 32) || DK > 64 ? 1 : 2) void k_token_attn_dkdv(const TokenAttnArgs a) {
    typedef Tile<T, DK> Tl;
    typedef Type<T> Ty;
    constexpr int KS = DK / 16, DT = (DK + 31) / 32, kTile = kRows * Tl::kRowBytes;
    constexpr float kShift = Ty::kNarrow ? 12.f : 0.f;
    __shared__ __align__(16) char lds[2 * 2 * kTile];
    __shared__ __align__(16) RowFacts facts[2];
    __shared__ int shared_range[4][2];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const Rows rows{a.G, a.magic};
    const int total = a.Lq * a.G;
    int tile, bh;
    place(a.B * a.Hk, tile, bh);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int key0 = tile * 128 + wave * 32, key = key0 + col;

    const Mask mask = make_mask(a, b);
    const Score score = make_score<T>(a);
    const int doc = a.k_docs && key < a.Lk ? a.k_docs[(size_t)b * a.Lk + key] : 0;
    const bool used = key < mask.kv_len && doc >= 0;  // (false: no row may see the key)
    int id_lo = 0, id_hi = 0;
    if (a.k_docs) {
        id_lo = wave_min(used ? doc : 0x7fffffff);
        id_hi = wave_max(used ? doc : -1);
    }
    const bool one_id = id_lo == id_hi;
    if (lane == 0) {
        shared_range[wave][0] = id_lo;
        shared_range[wave][1] = id_hi;
    }
    __syncthreads();
    int list_lo = id_lo, list_hi = id_hi;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        list_lo = min(list_lo, shared_range[w][0]);
        list_hi = max(list_hi, shared_range[w][1]);
    }

    typename Ty::Frag kf[KS], vf[KS];
    {
        const T* k = static_cast<const T*>(a.k) + (long long)b * a.k_stride[0] + (long long)key * a.k_stride[1] + (long long)hk * a.k_stride[2];
        const T* v = static_cast<const T*>(a.v) + (long long)b * a.v_stride[0] + (long long)key * a.v_stride[1] + (long long)hk * a.v_stride[2];
        load_owner<T, DK>(kf, used ? k : nullptr, a.D, lane);
        load_owner<T, DK>(vf, used ? v : nullptr, a.D, lane);
    }
    const T* qbase = static_cast<const T*>(a.q) + (long long)b * a.q_stride[0];
    const T* gbase = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0];
    const int* qdocs = a.q_docs ? a.q_docs + (size_t)b * a.Lq : nullptr;
    const int tiles = (total + kRows - 1) / kRows;
    const int4* ranges = a.q_ranges ? a.q_ranges + (size_t)b * tiles : nullptr;
    const float2* stats = a.stats + (size_t)bh * total;
    const float* delta = a.delta + (size_t)bh * total;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dk[t] = dv[t] = f32x16{};
    Fit fit;

    // the first row that sees any key from k on (the limits grow with the row)
    auto first_row = [&](int k) { return !a.causal || k < mask.prefix ? 0 : max(0, k - mask.shift) * a.G; };
    const int from = tile * 128 < mask.kv_len ? min(first_row(tile * 128) / kRows, tiles) : tiles;
    const int wave_from = key0 < mask.kv_len ? first_row(key0) : total;
    TileList list;
    list.start(ranges, list_lo, list_hi, from, tiles, lane);
    // the row tiles of these keys, in row_splits runs of at least kRun
    int run = 0x7fffffff, active = 1;
    if (a.row_splits > 1) {
        const int count = list.count(lane);
        run = max((count + a.row_splits - 1) / a.row_splits, kRun);
        active = max((count + run - 1) / run, 1);
        if ((int)blockIdx.y >= active) return;
        if (blockIdx.y) list.skip(blockIdx.y * run, lane);
        else if (tid == 0) a.grad_active[bh * ((a.Lk + 127) / 128) + tile] = active;
    }
    Fetch<T, DK, kRows, 256> fq, fg;
    float2 next_stats = make_float2(INFINITY, 0.f);
    float next_delta = 0.f, next_slope = 0.f;
    int next_limit = 0, next_doc = -1, next_where = 0;
    auto fetch = [&](int t) {
        const int r0 = t * kRows;
        auto address = [&](const T* base, const long long* stride, int r) -> const T* {
            if (r0 + r >= total || stats[r0 + r].x == INFINITY) return nullptr;  // a row that sees no key: whatever it holds counts as zero
            const int query = rows.query(r0 + r), head = hk * a.G + (r0 + r - query * a.G);
            return base + (long long)query * stride[1] + (long long)head * stride[2];
        };
        fq.load([&](int r) { return address(qbase, a.q_stride, r); }, a.D, tid);
        fg.load([&](int r) { return address(gbase, a.g_stride, r); }, a.D, tid);
        if (tid < kRows) {
            const int r = r0 + tid;
            const bool in = r < total;
            const int query = rows.query(min(r, total - 1)), head = hk * a.G + (min(r, total - 1) - query * a.G);
            next_stats = in ? stats[r] : make_float2(INFINITY, 0.f);
            next_delta = in ? delta[r] : 0.f;
            next_slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
            next_limit = in ? mask.limit(query) : 0;
            next_doc = qdocs ? qdocs[query] : 0;
            next_where = query + mask.shift;
        }
    };
    auto put = [&](int buf) {
        char* to = lds + buf * 2 * kTile;
        fq.store(to, tid);
        fg.store(to + kTile, tid);
        if (tid < kRows) {
            const Power<T> power(next_stats);
            facts[buf].m[tid] = power.m - kShift;
            if (sizeof(T) == 4) facts[buf].lg[tid] = power.lg;
            facts[buf].delta[tid] = next_delta;
            facts[buf].slope[tid] = next_slope;
            facts[buf].limit[tid] = next_limit;
            facts[buf].doc[tid] = next_doc;
            facts[buf].where[tid] = next_where;
        }
    };

    int t = list.next(lane), buf = 0;
    if (t >= 0) {
        fetch(t);
        put(0);
        __syncthreads();
    }
    while (t >= 0) {
        const int after = --run > 0 ? list.next(lane) : -1;
        if (after >= 0) fetch(after);
        const int r0 = t * kRows;
        if (r0 + kRows > wave_from) {
            const char* qt = lds + buf * 2 * kTile;
            const char* gt = qt + kTile;
            const RowFacts& f = facts[buf];
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                s = Ty::mfma(Tl::row(qt, col, 16 * c + 8 * half), kf[c], s);
                dp = Ty::mfma(Tl::row(gt, col, 16 * c + 8 * half), vf[c], dp);
            }
            // (the first row of the tile has its lowest limit)
            const bool whole = key0 + 32 <= mask.limit(rows.query(min(r0, total - 1)));
            bool same = true;
            if (qdocs) {
                const int4 g = ranges[t];
                same = one_id && g.z && g.x == id_lo;
            }
            f32x16 p;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = 8 * g + 4 * half;
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(&f.delta[at]);
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(&f.m[at]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dp[4 * g + e] -= d4[e];
                    p[4 * g + e] = -l4[e];
                }
            }
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = bend<T>(s[e], score);
                    s[e] = score.out * x;
                    dp[e] *= bend_slope<T>(x);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= score.in;
            }
            if (a.slopes) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int at = 8 * g + 4 * half;
                    const f32x4 m4 = *reinterpret_cast<const f32x4*>(&f.slope[at]);
                    const int4 w4 = *reinterpret_cast<const int4*>(&f.where[at]);
                    s[4 * g + 0] = fmaf(-m4[0], fabsf((float)(w4.x - key)), s[4 * g + 0]);
                    s[4 * g + 1] = fmaf(-m4[1], fabsf((float)(w4.y - key)), s[4 * g + 1]);
                    s[4 * g + 2] = fmaf(-m4[2], fabsf((float)(w4.z - key)), s[4 * g + 2]);
                    s[4 * g + 3] = fmaf(-m4[3], fabsf((float)(w4.w - key)), s[4 * g + 3]);
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] += s[e];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(&f.lg[8 * g + 4 * half]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[4 * g + e] -= l4[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(p[e]);
            if (!whole) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 m4 = *reinterpret_cast<const int4*>(&f.limit[8 * g + 4 * half]);
                    p[4 * g + 0] = key < m4.x ? p[4 * g + 0] : 0.f;
                    p[4 * g + 1] = key < m4.y ? p[4 * g + 1] : 0.f;
                    p[4 * g + 2] = key < m4.z ? p[4 * g + 2] : 0.f;
                    p[4 * g + 3] = key < m4.w ? p[4 * g + 3] : 0.f;
                }
            }
            if (!same) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 m4 = *reinterpret_cast<const int4*>(&f.doc[8 * g + 4 * half]);
                    p[4 * g + 0] = doc == m4.x ? p[4 * g + 0] : 0.f;
                    p[4 * g + 1] = doc == m4.y ? p[4 * g + 1] : 0.f;
                    p[4 * g + 2] = doc == m4.z ? p[4 * g + 2] : 0.f;
                    p[4 * g + 3] = doc == m4.w ? p[4 * g + 3] : 0.f;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const typename Ty::Frag pf = round_frag<T>(p, h);
#pragma unroll
                for (int d = 0; d < DT; ++d) dv[d] = Ty::mfma(Tl::column(gt, 16 * h, 32 * d, lane), pf, dv[d]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] *= dp[e];
            if constexpr (Ty::kNarrow) fit.apply<DT>(p, dk);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const typename Ty::Frag ds = round_frag<T>(p, h);
#pragma unroll
                for (int d = 0; d < DT; ++d) dk[d] = Ty::mfma(Tl::column(qt, 16 * h, 32 * d, lane), ds, dk[d]);
            }
        }
        if (after >= 0) {
            put(buf ^ 1);
            __syncthreads();
        }
        buf ^= 1;
        t = after;
    }

    if (active > 1) {
        if (key < a.Lk) {
            const float by = Ty::kNarrow ? 0x1p-12f / fit.s : 1.f, byv = Ty::kNarrow ? 0x1p-12f : 1.f;
            float* to = a.grad_part + ((((size_t)blockIdx.y * a.B + b) * a.Lk + key) * a.Hk + hk) * 2 * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = 32 * d + 8 * g + 4 * half;
                    if (c < a.D) {
                        f32x4 x, y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[e] = used ? dk[d][4 * g + e] * by : 0.f;
                            y[e] = used ? dv[d][4 * g + e] * byv : 0.f;
                        }
                        *reinterpret_cast<f32x4*>(to + c) = x;
                        *reinterpret_cast<f32x4*>(to + a.D + c) = y;
                    }
                }
        }
        return;
    }
    if (key < a.Lk) {
        const float by = Ty::kNarrow ? a.scale * 0x1p-12f / fit.s : a.scale;
        const float byv = Ty::kNarrow ? 0x1p-12f : 1.f;
        const size_t at = (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D;
        T *tk = static_cast<T*>(a.dk) + at, *tv = static_cast<T*>(a.dv) + at;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * half;
                if (c < a.D) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    T4 x, y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = (T)(used ? dk[d][4 * g + e] * by : 0.f);
                        y[e] = (T)(used ? dv[d][4 * g + e] * byv : 0.f);
                    }
                    *reinterpret_cast<T4*>(tk + c) = x;
                    *reinterpret_cast<T4*>(tv + c) = y;
                }
            }
    }
}

// dk and dv of the keys whose rows were split: the splits' sums in order; a thread per key and four channels of dk or dv
template <typename T>
__global__ __launch_bounds__(256) void k_token_attn_sum(const TokenAttnArgs a) {
    const int quads = a.D >> 1;  // of dk, then of dv
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x, at = item / quads;
    if (at >= (long long)a.B * a.Lk * a.Hk) return;
    const int c = 4 * (int)(item - at * quads);
    const int hk = (int)(at % a.Hk);
    const long long place = at / a.Hk;
    const int b = (int)(place / a.Lk), key = (int)(place - (long long)b * a.Lk);
    const int active = a.grad_active[(b * a.Hk + hk) * ((a.Lk + 127) / 128) + key / 128];
    if (active < 2) return;
    const size_t step = (size_t)a.B * a.Lk * a.Hk * 2 * a.D;
    const float* from = a.grad_part + (size_t)at * 2 * a.D + c;
    f32x4 sum = *reinterpret_cast<const f32x4*>(from);
    for (int s = 1; s < active; ++s) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(from + s * step);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += x[e];
    }
    const bool values = c >= a.D;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (T)(values ? sum[e] : sum[e] * a.scale);
    *reinterpret_cast<T4*>(static_cast<T*>(values ? a.dv : a.dk) + (size_t)at * a.D + (values ? c - a.D : c)) = x;
}

template <typename T, int DK>
hipError_t bwd(const TokenAttnArgs& a, hipStream_t stream) {
    const int total = a.Lq * a.G, heads = a.B * a.Hk;
    if (total > 0) {
        const long long items = (long long)heads * total;
        DANRA_LAUNCH_KERNEL((k_token_attn_delta<T>), dim3((unsigned)((items + 15) / 16)), dim3(256), 0, stream, a);
    }
    if (a.Lk > 0 && a.dk) {
        DANRA_LAUNCH_KERNEL((k_token_attn_dkdv<T, DK>), dim3((unsigned)((a.Lk + 127) / 128) * heads, a.row_splits), dim3(256), 0, stream, a);
        if (a.row_splits > 1) {
            const long long items = (long long)heads * a.Lk * (a.D / 2);
            DANRA_LAUNCH_KERNEL((k_token_attn_sum<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, a);
        }
    }
    if (total > 0 && a.dq)
        DANRA_LAUNCH_KERNEL((k_token_attn_dq<T, DK>), dim3((unsigned)((total + 127) / 128) * heads), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <typename T>
hipError_t bwd_type(const TokenAttnArgs& a, hipStream_t stream) {
    if (a.D <= 16) return bwd<T, 16>(a, stream);
    if (a.D <= 32) return bwd<T, 32>(a, stream);
    if (a.D <= 64) return bwd<T, 64>(a, stream);
    if (a.D <= 96) return bwd<T, 96>(a, stream);
    return bwd<T, 128>(a, stream);
}

}  // namespace
}  // namespace token

void plan_token_attn_bwd(TokenAttnArgs& a) {
    // Keys are owned 128 to a workgroup, and its rows - those of all the heads that share the keys, and with a causal mask all later
    // ones - follow one another: few keys or shared heads leave CUs idle, and the first keys run longest.  So the rows are
    // split until there are about four workgroups per CU, into runs of at least kRun tiles.
    const long long groups = (a.Lk + 127LL) / 128 * a.B * a.Hk, tiles = ((long long)a.Lq * a.G + 31) / 32;
    long long s = groups > 0 ? (1024 + groups - 1) / groups : 1;
    if (s > tiles / token::kRun) s = tiles / token::kRun;
    a.row_splits = s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

size_t token_attn_bwd_workspace(TokenAttnArgs& a, char* base) {
    token::Parts parts{base};
    parts.take(a.delta, (size_t)a.B * a.Hk * a.Lq * a.G);
    if (a.row_splits > 1) {
        parts.take(a.grad_part, (size_t)a.row_splits * a.B * a.Lk * a.Hk * 2 * a.D);
        parts.take(a.grad_active, (size_t)a.B * a.Hk * ((a.Lk + 127) / 128));
    }
    if (a.k_docs) {
        parts.take(a.k_ranges, (size_t)a.B * ((a.Lk + 31) / 32));
        parts.take(a.q_ranges, (size_t)a.B * (((size_t)a.Lq * a.G + 31) / 32));
    }
    return parts.bytes;
}

hipError_t launch_token_attn_bwd(const TokenAttnArgs& a, hipStream_t stream) {
    if (a.k_docs && a.Lk > 0 && a.Lq > 0) {
        const int k_tiles = (a.Lk + 31) / 32, q_tiles = (a.Lq * a.G + 31) / 32;
        if (hipError_t e = token::launch_ranges(a.k_docs, a.k_ranges, a.Lk, 1, 32, k_tiles, a.B, stream); e != hipSuccess) return e;
        if (hipError_t e = token::launch_ranges(a.q_docs, a.q_ranges, a.Lq, a.G, 32, q_tiles, a.B, stream); e != hipSuccess) return e;
    }
    switch (a.type) {
        case TOKEN_F32: return token::bwd_type<float>(a, stream);
        case TOKEN_BF16: return token::bwd_type<__bf16>(a, stream);
        default: return token::bwd_type<_Float16>(a, stream);
    }
}

}  // namespace danra
