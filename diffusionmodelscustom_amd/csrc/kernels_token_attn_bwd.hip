// Backward pass of danra_token_attention_* (token_attn.h has the formulas and the layout), from q, k, v, out, dout and each row's
// maximum and sum, without the score matrix in memory and without atomics:
//   delta = rowsum(dout . out)
//   p = 2^(score2 - m - log2 l),  dP = dout v^T,  dS = p (dP - delta) (1 - tanh^2)
//   dv = p^T dout,  dk = scale dS^T q,  dq = scale dS k
// One kernel owns query rows and sums dq over the keys, one owns keys and sums dk and dv over the rows of all the heads that share
// them; both form S and dP again (seven products of the size of S instead of five, for sums in a fixed order).  All sums are float32.
// P is rounded to the operand's type for its product: 2^-9 relative in bfloat16, of the size of the rounding of the inputs.  dS goes into its
// products in two parts, rounded value and remainder: its terms have both signs and cancel in the sums, and with one part dq and dk were up to 1.55
// times as far off as one rounding of the exact result is; with two at most 1.25 (dq of 16 heads of 4096 tokens, D = 128, 204 -> 261 us, dk and dv
// 331 -> 397; packed documents 96 -> 111 and 235 -> 263).
// Half precision has no exponents for that: there P is kept times 2^12 (at most 2^12), and dS times a power of two of its column
// that falls when a tile brings larger values (the accumulator is rescaled then), the largest values lying between 2^10 and 2^14.
//
// Measured (bfloat16, D = 128, 16 heads of 4096 tokens): dk and dv 381 us, dq 255 us: 902 and 1078 TFLOP/s of the five and four
// products that they form (dS in two parts); at D = 64 205 and 150 us.  There the matrix unit is busy 34 and 44 % of the time and the vector unit
// 30 and 33 %, with 1.5 and 1.4 waves on a SIMD: a wave's products, its sixteen or so vector instructions a score and its reading of a
// fragment for every product out of LDS follow one another, and a second wave is not enough to fill the gaps.  Packed documents (dk and dv
// matrix unit 10 %, vector unit 16 %, 0.9 waves) wait: workgroups with few tiles leave their CU to the long ones.
#include "token_attn.h"

namespace danra {
namespace token {

namespace {

// rows (dk, dv) and keys (dq) of a streamed tile: two of the matrix instruction's, so that what a tile costs besides them counts half, but one
// where the registers are full (dq of 16 heads of 4096 tokens in bfloat16, D = 128: 255 us with one, 290 with two, which spill; D = 64: 160 and 150)
constexpr int rows_of(bool f32, int D) { return f32 && D > 64 ? 32 : 64; }
constexpr int keys_of(bool f32, int D) { return D > (f32 ? 32 : 64) ? 32 : 64; }
int rows_of(const TokenAttnArgs& a) { return rows_of(a.type == TOKEN_F32, a.D); }
int keys_of(const TokenAttnArgs& a) { return keys_of(a.type == TOKEN_F32, a.D); }
// tiles of rows that are worth a workgroup and a partial result of their own (packed documents, whose runs differ, bfloat16, D = 128, with the
// join: 16 279 us, 8 285, 24 280)
__host__ __device__ constexpr int run_of(bool docs) { return docs ? 16 : 8; }

// p = 2^(score2 - m - log2 l).  In float32 the two are subtracted one after the other: m is itself a score of the row, so the first
// difference is small where p counts, while m + log2 l rounds at the size of m (2^-20 at m = 16, which p would have as relative error).
// That is far below the rounding of a two-byte P: there it is one number, and lg is not used.  kShift: P is kept times 2^kShift.
template <typename T>
__device__ constexpr float shift_of() { return Type<T>::kNarrow ? 12.f : 0.f; }

// the power of two that a column's dS carries in half precision
struct Fit {
    float s = 0x1p60f;
    // c: the tile's dS; acc: what has been summed with the old power.  Multiplies both by what they need.
    template <int DT>
    __device__ __forceinline__ void apply(f32x16& c, f32x16 (&acc)[DT]) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(fabsf(c[e]), fabsf(c[e + 1])));
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

// What the two kernels below need of each row: facts [3][B Hk][rows, up to whole tiles]: m (+ log2 l - kShift in two-byte types; infinity
// for a row that sees no key and for the places behind the last row), delta, log2 l; and of each tile of rows whether it has any
// such row.  A workgroup per tile, 16 lanes a row.
template <typename T, int kStream>
__global__ __launch_bounds__(256) void k_token_attn_delta(const TokenAttnArgs a) {
    const int total = a.Lq * a.G, tiles = (total + kStream - 1) / kStream;
    const int bh = blockIdx.x / tiles, tile = blockIdx.x - bh * tiles;
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const Rows rows{a.G, a.magic};
    const int c = threadIdx.x & 15;
    bool dead = false;
#pragma unroll
    for (int n = 0; n < kStream / 16; ++n) {
        const int r = tile * kStream + n * 16 + (threadIdx.x >> 4);
        float sum = 0.f;
        float2 stats = make_float2(INFINITY, 0.f);
        if (r < total) {
            stats = a.stats[(size_t)bh * total + r];
            const int query = rows.query(r), head = hk * a.G + r - query * a.G;
            const size_t at = (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D;
            const T* o = static_cast<const T*>(a.out) + at;
            const T* g = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0] + (long long)query * a.g_stride[1] + (long long)head * a.g_stride[2];
            const T* rest = a.rest ? static_cast<const T*>(a.rest) + at : nullptr;
            if (c * 8 < a.D) {
                typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const T4 x = reinterpret_cast<const T4*>(o + 8 * c)[h], y = reinterpret_cast<const T4*>(g + 8 * c)[h];
                    T4 z = {};
                    if (rest) z = reinterpret_cast<const T4*>(rest + 8 * c)[h];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum = fmaf((float)x[e] + (float)z[e], (float)y[e], sum);
                }
            }
        }
#pragma unroll
        for (int k = 8; k; k >>= 1) sum += __shfl_xor(sum, k);
        const bool none = stats.x == INFINITY;
        dead |= none;
        if (c == 0) {
            const size_t n_facts = (size_t)a.B * a.Hk * tiles * kStream, at = (size_t)bh * tiles * kStream + r;
            a.facts[at] = sizeof(T) == 2 ? stats.x + stats.y - shift_of<T>() : stats.x;
            a.facts[n_facts + at] = none ? 0.f : sum;
            if (sizeof(T) == 4) a.facts[2 * n_facts + at] = stats.y;
        }
    }
    dead = __syncthreads_or(dead);
    if (threadIdx.x == 0) a.row_flags[blockIdx.x] = dead;
}

template <typename T, int DK, Cap CAP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DK >= 64 ? 1 : 2) void k_token_attn_dq(const TokenAttnArgs a) {
    typedef Tile<T, DK> Tl;
    typedef Type<T> Ty;
    constexpr int kStream = rows_of(sizeof(T) == 4, DK);
    constexpr int KS = DK / 16, DT = (DK + 31) / 32, kKeys = keys_of(sizeof(T) == 4, DK), kTile = kKeys * Tl::kRowBytes;
    __shared__ __align__(16) char lds[2 * 2 * kTile];
    __shared__ __align__(16) int ids[2][64];
    __shared__ int shared_range[4][3];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const Rows rows{a.G, a.magic};
    const int total = a.Lq * a.G, row_tiles = (total + kStream - 1) / kStream;
    int tile, bh;
    place(a.B * a.Hk, tile, bh);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    if (a.causal) tile = (total + 127) / 128 - 1 - tile;
    const int row = tile * 128 + wave * 32 + col;

    const Mask mask = make_mask(a, b);
    const int query = rows.query(min(row, total - 1)), head = hk * a.G + (min(row, total - 1) - query * a.G);
    const size_t n_facts = (size_t)a.B * a.Hk * row_tiles * kStream, fact = (size_t)bh * row_tiles * kStream + min(row, total - 1);
    // (kShift is for dv's P only: here it is taken out again)
    const float m = row < total ? a.facts[fact] + shift_of<T>() : INFINITY;
    const float delta = row < total ? a.facts[n_facts + fact] : 0.f, lg = sizeof(T) == 4 && row < total ? a.facts[2 * n_facts + fact] : 0.f;
    const bool used = m != INFINITY;  // (false: the row sees no key)
    const int limit = used ? max(mask.limit(query), 0) : 0;
    const int doc = a.q_docs ? a.q_docs[(size_t)b * a.Lq + query] : 0;
    const int where = query + mask.shift;
    const Score score = make_score<CAP>(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2e / score.out : 0.f;

    const int wave_limit = __builtin_amdgcn_readfirstlane(wave_max(limit)), lowest = __builtin_amdgcn_readfirstlane(wave_min(limit));
    int id_lo = 0, id_hi = 0;
    if (a.q_docs) {
        id_lo = wave_min(limit > 0 ? doc : 0x7fffffff);
        id_hi = wave_max(limit > 0 ? doc : -1);
    }
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
    list_limit = __builtin_amdgcn_readfirstlane(list_limit);

    typename Ty::Frag qf[KS], gf[KS];
    {
        const T* q = static_cast<const T*>(a.q) + (long long)b * a.q_stride[0] + (long long)query * a.q_stride[1] + (long long)head * a.q_stride[2];
        const T* g = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0] + (long long)query * a.g_stride[1] + (long long)head * a.g_stride[2];
        load_owner<T, DK>(qf, used ? q : nullptr, a.D, lane);
        owner_sign<T>(qf, a.scale);
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
    list.start(ranges, nullptr, list_lo, list_hi, id_lo, id_hi, 0, (list_limit + kKeys - 1) / kKeys, lane);
    Rowwise<T, DK, kKeys, 4> keys, values;
    const unsigned k_step = (unsigned)a.k_stride[1] * (unsigned)sizeof(T), v_step = (unsigned)a.v_stride[1] * (unsigned)sizeof(T);
    keys.prepare(k_step, a.D, wave, lane);
    values.prepare(v_step, a.D, wave, lane);
    auto stage = [&](const Visit& x, int buf) {
        const int k0 = x.t * kKeys, count = mask.kv_len - k0;
        char* to = lds + buf * 2 * kTile;
        auto dead = [&](int r) { return r < count && kdocs[k0 + r] < 0; };
        keys.load(kbase + (long long)k0 * a.k_stride[1], count, k_step, a.D, to, wave, lane, x.dead, dead);
        values.load(vbase + (long long)k0 * a.v_stride[1], count, v_step, a.D, to + kTile, wave, lane, x.dead, dead);
        if (kdocs && wave == 0) load_lds4(buffer(kdocs + k0, 4u * min(count, kKeys)), 4u * lane, (char*)ids[buf]);
    };

    auto process = [&](bool whole, const Visit& x, int buf, int n) {
        const char* kt = lds + buf * 2 * kTile;
        const char* vt = kt + kTile;
        const int k0 = x.t * kKeys + 32 * n;
        f32x16 s = {}, dp = {};
        typename Ty::Frag kf[KS], vf[KS];
#pragma unroll
        for (int c = 0; c < KS; ++c) kf[c] = Tl::row(kt, 32 * n + col, 16 * c + 8 * half);
#pragma unroll
        for (int c = 0; c < KS; ++c) vf[c] = Tl::row(vt, 32 * n + col, 16 * c + 8 * half);
        __builtin_amdgcn_sched_barrier(0);  // (left alone, each fragment is read when it is needed, and waited for)
#pragma unroll
        for (int c = 0; c < KS; ++c) s = Ty::mfma(kf[c], qf[c], s);
#pragma unroll
        for (int c = 0; c < KS; ++c) dp = Ty::mfma(vf[c], gf[c], dp);
        typename Ty::Frag columns[2][DT];  // of the keys, for the product behind: read while the scores are worked on
#pragma unroll
        for (int d = 0; d < DT; ++d) columns[0][d] = Tl::column(kt, 32 * n, 32 * d, lane);
        __builtin_amdgcn_sched_barrier(0);
        // s becomes the bent product with its bias, then dS; dp becomes (dP - delta) times the cap's derivative
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = bend<CAP>(s[e], score);
            dp[e] -= delta;
            if constexpr (CAP != kNoCap) dp[e] *= bend_slope<CAP>(s[e]);
        }
        const int j0 = k0 + 4 * half;
        if (a.slopes) {
            const float from = (float)(where - j0);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(from - (float)(8 * (e >> 2) + (e & 3))), s[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float power = sizeof(T) == 2 ? fmaf(s[e], score.out, -m) : fmaf(s[e], score.out, -m) - lg;
            s[e] = __builtin_amdgcn_exp2f(power) * dp[e];
        }
        if (!whole) {
            const int left = limit - j0;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) < left ? s[e] : 0.f;
        }
        if (!x.same) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int4 d = *reinterpret_cast<const int4*>(&ids[buf][32 * n + 4 * half + 8 * g]);
                s[4 * g + 0] = d.x == doc ? s[4 * g + 0] : 0.f;
                s[4 * g + 1] = d.y == doc ? s[4 * g + 1] : 0.f;
                s[4 * g + 2] = d.z == doc ? s[4 * g + 2] : 0.f;
                s[4 * g + 3] = d.w == doc ? s[4 * g + 3] : 0.f;
            }
        }
        if constexpr (Ty::kNarrow) fit.apply<DT>(s, dq);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h == 0) {
#pragma unroll
                for (int d = 0; d < DT; ++d) columns[1][d] = Tl::column(kt, 32 * n + 16, 32 * d, lane);
                __builtin_amdgcn_sched_barrier(0);
            }
            const typename Ty::Frag ds = round_frag<T>(s, h);
#pragma unroll
            for (int d = 0; d < DT; ++d) dq[d] = Ty::mfma(columns[h][d], ds, dq[d]);
            // The rounding's remainder as well: a query's gradient takes the rounding of its row of dS and, through rowsum(dout . out), that
            // of its row of P; with one part it was 1.5 times as far off as one rounding of the exact value is, with two 1.1 times.
            if constexpr (sizeof(T) == 2) {
                const typename Ty::Frag rest = rest_frag<T>(s, ds, h);
#pragma unroll
                for (int d = 0; d < DT; ++d) dq[d] = Ty::mfma(columns[h][d], rest, dq[d]);
            }
        }
    };

    auto work = [&](const Visit& x, auto buf) {
#pragma unroll
        for (int n = 0; n < kKeys / 32; ++n) {
            const int k0 = x.t * kKeys + 32 * n;
            if (x.wanted && k0 < wave_limit) process(k0 + 32 <= lowest, x, buf(), n);
        }
    };
    two_buffers([&]() { return list.next(lane); }, stage, work);

    if (row < total) {
        const float by = a.scale * bend_factor<CAP>() / (Ty::kNarrow ? fit.s : 1.f);
        T* to = static_cast<T*>(a.dq) + (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * half;
                if (c < a.D) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    T4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = (T)(used ? dq[d][4 * g + e] * by : 0.f);
                    *reinterpret_cast<T4*>(to + c) = y;
                }
            }
    }
}

// rows of a streamed tile
struct RowFacts {
    float m[64], delta[64], lg[64], slope[64];
    float where[64];  // the row's place, from the workgroup's first key
    int doc[64], limit[64];
};

// A wave owns 32 keys.  Where the keys' fragments and both accumulators fit the registers that two waves of a SIMD share (D <= 64 in a
// two-byte type) four waves with 128 keys go through every row tile.  Beyond (WIDE) the fragments of keys and values stay in LDS, and eight
// waves share the 128 keys: each takes one half of every row tile, and the two sums are added at the end.  (With all of it in the
// registers of one wave per SIMD, dk/dv of 4096 tokens x 16 heads at D = 128 takes 455 us instead of 381, of packed documents 275 instead of 264.)
constexpr bool wide_of(bool f32, int DK) { return !f32 && DK > 64; }

template <typename T, int DK, Cap CAP>
__global__ __launch_bounds__(wide_of(sizeof(T) == 4, DK) ? 512 : 256, sizeof(T) == 4 && DK >= 32 ? 1 : 2) void k_token_attn_dkdv(const TokenAttnArgs a) {
    constexpr bool WIDE = wide_of(sizeof(T) == 4, DK);
    constexpr int kWaves = WIDE ? 8 : 4;
    typedef Tile<T, DK> Tl;
    typedef Type<T> Ty;
    constexpr int kStream = rows_of(sizeof(T) == 4, DK);
    typedef Stage<T, DK, kStream, kWaves> St;
    constexpr int KS = DK / 16, DT = (DK + 31) / 32, kTile = kStream * Tl::kRowBytes;
    constexpr int kOwn = 32 * Tl::kRowBytes;                                             // a wave's keys, or values
    constexpr int kLds = 2 * 2 * kTile + (WIDE ? 2 * 4 * kOwn : 0), kJoin = WIDE ? 4 * 2 * DT * 16 * 64 * 4 : 0;
    __shared__ __align__(16) char lds[kLds > kJoin ? kLds : kJoin];
    __shared__ __align__(16) RowFacts facts[2];
    __shared__ int shared_range[4][2];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const Rows rows{a.G, a.magic};
    const int total = a.Lq * a.G, tiles = (total + kStream - 1) / kStream;
    int tile, bh;
    place(a.B * a.Hk, tile, bh);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int mine = wave & 3, part = wave >> 2;  // (part: 0 unless WIDE)
    const int key0 = tile * 128 + mine * 32, key = key0 + col;

    const Mask mask = make_mask(a, b);
    const Score score = make_score<CAP>(a);
    const float bias = -kLog2e / score.out, place_of_key = (float)(mine * 32 + col);
    const int doc = a.k_docs && key < a.Lk ? a.k_docs[(size_t)b * a.Lk + key] : 0;
    const bool used = key < mask.kv_len && doc >= 0;  // (false: no row may see the key)
    int id_lo = 0, id_hi = 0;
    if (a.k_docs) {
        id_lo = wave_min(used ? doc : 0x7fffffff);
        id_hi = wave_max(used ? doc : -1);
    }
    if (lane == 0 && part == 0) {
        shared_range[mine][0] = id_lo;
        shared_range[mine][1] = id_hi;
    }
    __syncthreads();
    int list_lo = id_lo, list_hi = id_hi;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        list_lo = min(list_lo, shared_range[w][0]);
        list_hi = max(list_hi, shared_range[w][1]);
    }

    // the first row that sees any key from k on (the limits grow with the row)
    auto first_row = [&](int k) { return !a.causal || k < mask.prefix ? 0 : max(0, k - mask.shift) * a.G; };
    const int from = tile * 128 < mask.kv_len ? min(first_row(tile * 128) / kStream, tiles) : tiles;
    const int wave_from = key0 < mask.kv_len ? first_row(key0) : total;
    TileList list;
    list.start(a.q_ranges ? a.q_ranges + (size_t)b * tiles : nullptr, a.row_flags + (size_t)bh * tiles, list_lo, list_hi, id_lo, id_hi, from,
               tiles, lane);
    // the row tiles of these keys, in row_splits runs of at least run_of
    int run = 0x7fffffff, active = 1;
    if (a.row_splits > 1) {
        const int count = list.count(lane);
        run = max((count + a.row_splits - 1) / a.row_splits, run_of(a.q_docs));
        active = max((count + run - 1) / run, 1);
        if ((int)blockIdx.y >= active) return;
        if (blockIdx.y) list.skip(blockIdx.y * run, lane);
        else if (tid == 0) a.grad_active[bh * ((a.Lk + 127) / 128) + tile] = active;
    }

    typename Ty::Frag kf[WIDE ? 1 : KS], vf[WIDE ? 1 : KS];
    char* const own_k = lds + 2 * 2 * kTile + mine * 2 * kOwn;
    char* const own_v = own_k + kOwn;
    {
        const T* k = static_cast<const T*>(a.k) + (long long)b * a.k_stride[0] + (long long)key * a.k_stride[1] + (long long)hk * a.k_stride[2];
        const T* v = static_cast<const T*>(a.v) + (long long)b * a.v_stride[0] + (long long)key * a.v_stride[1] + (long long)hk * a.v_stride[2];
        if constexpr (WIDE) {  // (the first barrier stands in front of their first use)
            typename Ty::Frag f[KS];
            load_owner<T, DK>(f, used ? (part ? v : k) : nullptr, a.D, lane);
            if (!part) owner_sign<T>(f, a.scale);
#pragma unroll
            for (int c = 0; c < KS; ++c) Tl::set_row(part ? own_v : own_k, col, 16 * c + 8 * half, f[c]);
        } else {
            load_owner<T, DK>(kf, used ? k : nullptr, a.D, lane);
            owner_sign<T>(kf, a.scale);
            load_owner<T, DK>(vf, used ? v : nullptr, a.D, lane);
        }
    }
    const T* qbase = static_cast<const T*>(a.q) + (long long)b * a.q_stride[0] + (long long)hk * a.G * a.q_stride[2];
    const T* gbase = static_cast<const T*>(a.dout) + (long long)b * a.g_stride[0] + (long long)hk * a.G * a.g_stride[2];
    const int* qdocs = a.q_docs ? a.q_docs + (size_t)b * a.Lq : nullptr;
    const size_t n_facts = (size_t)a.B * a.Hk * tiles * kStream;
    const float* row_facts = a.facts + (size_t)bh * tiles * kStream;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dk[t] = dv[t] = f32x16{};
    Fit fit;

    // bytes between a row's queries and heads (the host has checked that the kStream rows of a tile lie within 2^31)
    const unsigned q_step = (unsigned)a.q_stride[1] * (unsigned)sizeof(T), q_head = (unsigned)a.q_stride[2] * (unsigned)sizeof(T);
    const unsigned g_step = (unsigned)a.g_stride[1] * (unsigned)sizeof(T), g_head = (unsigned)a.g_stride[2] * (unsigned)sizeof(T);
    unsigned column[St::kEach];
#pragma unroll
    for (int n = 0; n < St::kEach; ++n) column[n] = St::column(n, wave, lane, a.D);
    auto stage = [&](const Visit& x, int buf) {
        const int r0 = x.t * kStream, i0 = __builtin_amdgcn_readfirstlane(rows.query(r0));
        const Buffer q = buffer(qbase + (long long)i0 * a.q_stride[1], 0x7fffffffu), g = buffer(gbase + (long long)i0 * a.g_stride[1], 0x7fffffffu);
        char* to = lds + buf * 2 * kTile;
        unsigned q_at[St::kEach], g_at[St::kEach];
#pragma unroll
        for (int n = 0; n < St::kEach; ++n) {
            const int r = r0 + St::row(n, wave, lane), i = rows.query(r), h = r - i * a.G;
            q_at[n] = g_at[n] = column[n];
            // a row that sees no key, or none at all, reads as zero whatever lies there
            if (column[n] != kNowhere) {
                q_at[n] += (unsigned)(i - i0) * q_step + (unsigned)h * q_head;
                g_at[n] += (unsigned)(i - i0) * g_step + (unsigned)h * g_head;
            }
            if (x.dead && row_facts[r] == INFINITY) q_at[n] = g_at[n] = kNowhere;
        }
        St::load(q, q_at, to, wave);
        St::load(g, g_at, to + kTile, wave);
        RowFacts& f = facts[buf];
        const int r = min(r0 + lane, total - 1), i = rows.query(r), h = hk * a.G + r - i * a.G;
        if (wave == 0) {
            load_lds4(buffer(row_facts + r0, 4 * kStream), 4u * lane, (char*)f.m);
            if (sizeof(T) == 4) load_lds4(buffer(row_facts + 2 * n_facts + r0, 4 * kStream), 4u * lane, (char*)f.lg);
        }
        if (wave == 1) load_lds4(buffer(row_facts + n_facts + r0, 4 * kStream), 4u * lane, (char*)f.delta);
        if (wave == 2) {
            if (qdocs) load_lds4(buffer(qdocs + i0, 0x7fffffffu), 4u * (i - i0), (char*)f.doc);
            f.limit[lane] = mask.limit(i);
        }
        if (wave == 3 && a.slopes) {
            load_lds4(buffer(a.slopes, 0x7fffffffu), 4u * h, (char*)f.slope);
            f.where[lane] = (float)(i + mask.shift - tile * 128);
        }
    };

    auto process = [&](bool whole, const Visit& x, int buf, int n) {
        const char* qt = lds + buf * 2 * kTile;
        const char* gt = qt + kTile;
        const RowFacts& f = facts[buf];
        f32x16 s = {}, dp = {};
        if constexpr (WIDE) {
            constexpr int kAhead = 2, kGroups = KS / kAhead;
            typename Ty::Frag left[2][kAhead], right[2][kAhead];
            auto read_rows = [&](int g) {  // the groups of q and the keys, then those of dout and the values
#pragma unroll
                for (int c = 0; c < kAhead; ++c) {
                    const int d = 16 * (g % kGroups * kAhead + c) + 8 * half;
                    left[g & 1][c] = Tl::row(g < kGroups ? qt : gt, 32 * n + col, d);
                    right[g & 1][c] = Tl::row(g < kGroups ? own_k : own_v, col, d);
                }
            };
            read_rows(0);
#pragma unroll
            for (int g = 0; g < 2 * kGroups; ++g) {
                if (g + 1 < 2 * kGroups) read_rows(g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < kAhead; ++c) {
                    if (g < kGroups) s = Ty::mfma(left[g & 1][c], right[g & 1][c], s);
                    else dp = Ty::mfma(left[g & 1][c], right[g & 1][c], dp);
                }
            }
        } else {
            typename Ty::Frag qf[KS], gf[KS];
#pragma unroll
            for (int c = 0; c < KS; ++c) qf[c] = Tl::row(qt, 32 * n + col, 16 * c + 8 * half);
#pragma unroll
            for (int c = 0; c < KS; ++c) gf[c] = Tl::row(gt, 32 * n + col, 16 * c + 8 * half);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < KS; ++c) s = Ty::mfma(qf[c], kf[c], s);
#pragma unroll
            for (int c = 0; c < KS; ++c) dp = Ty::mfma(gf[c], vf[c], dp);
        }
        // of dout and q, for the products behind: each group is read one product ahead, the first while the scores are worked on
        typename Ty::Frag columns[2][DT];
        auto read_columns = [&](int g) {
#pragma unroll
            for (int d = 0; d < DT; ++d) columns[g & 1][d] = Tl::column(g < 2 ? gt : qt, 32 * n + 16 * (g & 1), 32 * d, lane);
            __builtin_amdgcn_sched_barrier(0);
        };
        read_columns(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 d4 = *reinterpret_cast<const f32x4*>(&f.delta[32 * n + 8 * g + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * g + e] = bend<CAP>(s[4 * g + e], score);
                dp[4 * g + e] -= d4[e];
                if constexpr (CAP != kNoCap) dp[4 * g + e] *= bend_slope<CAP>(s[4 * g + e]);
            }
        }
        if (a.slopes) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 m4 = *reinterpret_cast<const f32x4*>(&f.slope[32 * n + 8 * g + 4 * half]);
                const f32x4 w4 = *reinterpret_cast<const f32x4*>(&f.where[32 * n + 8 * g + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(m4[e] * bias, fabsf(w4[e] - place_of_key), s[4 * g + e]);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 m4 = *reinterpret_cast<const f32x4*>(&f.m[32 * n + 8 * g + 4 * half]);
            f32x4 l4 = {};
            if constexpr (sizeof(T) == 4) l4 = *reinterpret_cast<const f32x4*>(&f.lg[32 * n + 8 * g + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float power = sizeof(T) == 2 ? fmaf(s[4 * g + e], score.out, -m4[e]) : fmaf(s[4 * g + e], score.out, -m4[e]) - l4[e];
                s[4 * g + e] = __builtin_amdgcn_exp2f(power);
            }
        }
        if (!whole) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int4 m4 = *reinterpret_cast<const int4*>(&f.limit[32 * n + 8 * g + 4 * half]);
                s[4 * g + 0] = key < m4.x ? s[4 * g + 0] : 0.f;
                s[4 * g + 1] = key < m4.y ? s[4 * g + 1] : 0.f;
                s[4 * g + 2] = key < m4.z ? s[4 * g + 2] : 0.f;
                s[4 * g + 3] = key < m4.w ? s[4 * g + 3] : 0.f;
            }
        }
        if (!x.same) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int4 m4 = *reinterpret_cast<const int4*>(&f.doc[32 * n + 8 * g + 4 * half]);
                s[4 * g + 0] = doc == m4.x ? s[4 * g + 0] : 0.f;
                s[4 * g + 1] = doc == m4.y ? s[4 * g + 1] : 0.f;
                s[4 * g + 2] = doc == m4.z ? s[4 * g + 2] : 0.f;
                s[4 * g + 3] = doc == m4.w ? s[4 * g + 3] : 0.f;
            }
        }
        typename Ty::Frag pf[2], ds[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) pf[h] = round_frag<T>(s, h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= dp[e];
        if constexpr (Ty::kNarrow) fit.apply<DT>(s, dk);
#pragma unroll
        for (int h = 0; h < 2; ++h) ds[h] = round_frag<T>(s, h);
        typename Ty::Frag rest[2];  // what the rounding of dS leaves, as for dq: dk with one part was up to 1.55 times as far off as one rounding is
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) rest[h] = rest_frag<T>(s, ds[h], h);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g < 3) read_columns(g + 1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (g < 2) dv[d] = Ty::mfma(columns[g & 1][d], pf[g & 1], dv[d]);
                else dk[d] = Ty::mfma(columns[g & 1][d], ds[g & 1], dk[d]);
            }
            if constexpr (sizeof(T) == 2) {
                if (g >= 2) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) dk[d] = Ty::mfma(columns[g & 1][d], rest[g & 1], dk[d]);
                }
            }
        }
    };

    auto work = [&](const Visit& x, auto buf) {
        auto rows_at = [&](int n) {
            const int r0 = x.t * kStream + 32 * n;
            // (the first of the rows has their lowest limit)
            if (x.wanted && r0 < total && r0 + 32 > __builtin_amdgcn_readfirstlane(wave_from))
                process(__builtin_amdgcn_readfirstlane(key0 + 32 <= mask.limit(rows.query(r0))), x, buf(), n);
        };
        if constexpr (WIDE) {
            rows_at(part);
        } else {
#pragma unroll
            for (int n = 0; n < kStream / 32; ++n) rows_at(n);
        }
    };
    two_buffers([&]() { return run-- > 0 ? list.next(lane) : Visit{-1, false, false, false}; }, stage, work);

    // dk is summed without the cap's constant factor, in half precision times fit.s 2^kShift, dv times 2^kShift
    const float unshift = Ty::kNarrow ? 0x1p-12f : 1.f, by = bend_factor<CAP>() * (Ty::kNarrow ? 0x1p-12f / fit.s : 1.f);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            dk[d][e] *= by;
            dv[d][e] *= unshift;
        }
    if constexpr (WIDE) {
        float* join = reinterpret_cast<float*>(lds) + mine * 2 * DT * 16 * 64;
        __syncthreads();
        if (part) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    join[(d * 16 + e) * 64 + lane] = dk[d][e];
                    join[((DT + d) * 16 + e) * 64 + lane] = dv[d][e];
                }
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dk[d][e] += join[(d * 16 + e) * 64 + lane];
                dv[d][e] += join[((DT + d) * 16 + e) * 64 + lane];
            }
    }
    if (active > 1) {
        if (key < a.Lk) {
            float* to = a.grad_part + ((((size_t)blockIdx.y * a.B + b) * a.Lk + key) * a.Hk + hk) * 2 * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = 32 * d + 8 * g + 4 * half;
                    if (c < a.D) {
                        f32x4 y, z;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y[e] = used ? dk[d][4 * g + e] : 0.f;
                            z[e] = used ? dv[d][4 * g + e] : 0.f;
                        }
                        *reinterpret_cast<f32x4*>(to + c) = y;
                        *reinterpret_cast<f32x4*>(to + a.D + c) = z;
                    }
                }
        }
        return;
    }
    if (key < a.Lk) {
        const size_t at = (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D;
        T *tk = static_cast<T*>(a.dk) + at, *tv = static_cast<T*>(a.dv) + at;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * half;
                if (c < a.D) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    T4 y, z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = (T)(used ? dk[d][4 * g + e] * a.scale : 0.f);
                        z[e] = (T)(used ? dv[d][4 * g + e] : 0.f);
                    }
                    *reinterpret_cast<T4*>(tk + c) = y;
                    *reinterpret_cast<T4*>(tv + c) = z;
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

template <typename T, int DK, Cap CAP>
hipError_t bwd(const TokenAttnArgs& a, hipStream_t stream) {
    const int total = a.Lq * a.G, heads = a.B * a.Hk;
    constexpr int kStream = rows_of(sizeof(T) == 4, DK);
    if (total > 0) DANRA_LAUNCH_KERNEL((k_token_attn_delta<T, kStream>), dim3((unsigned)((total + kStream - 1) / kStream) * heads), dim3(256), 0, stream, a);
    if (a.Lk > 0 && a.dk) {
        DANRA_LAUNCH_KERNEL((k_token_attn_dkdv<T, DK, CAP>), dim3((unsigned)((a.Lk + 127) / 128) * heads, a.row_splits),
                            dim3(wide_of(sizeof(T) == 4, DK) ? 512 : 256), 0, stream, a);
        if (a.row_splits > 1) {
            const long long items = (long long)heads * a.Lk * (a.D / 2);
            DANRA_LAUNCH_KERNEL((k_token_attn_sum<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, a);
        }
    }
    if (total > 0 && a.dq)
        DANRA_LAUNCH_KERNEL((k_token_attn_dq<T, DK, CAP>), dim3((unsigned)((total + 127) / 128) * heads), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <typename T, int DK>
hipError_t bwd(const TokenAttnArgs& a, hipStream_t stream) {
    switch (cap_of(a)) {
        case kNoCap: return bwd<T, DK, kNoCap>(a, stream);
        case kQuick:
            if constexpr (sizeof(T) == 2) return bwd<T, DK, kQuick>(a, stream);
        default: return bwd<T, DK, kExact>(a, stream);
    }
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

int token_attn_bwd_rows(const TokenAttnArgs& a) { return token::rows_of(a); }

void plan_token_attn_bwd(TokenAttnArgs& a) {
    // Keys are owned 128 to a workgroup, and its rows - those of all the heads that share the keys, and with a causal mask all later
    // ones - follow one another: few keys or shared heads leave CUs idle, and the first keys run longest.  So the rows are
    // split until there are about two workgroups per CU (bfloat16, D = 128, 4096 tokens: 16 heads 381 us unsplit, 401 + 25 for the join in two;
    // 16 heads over 4 361 + 13 in four, 389 + 22 in eight), with documents, whose keys have few rows or many, about four, in runs that are worth
    // it (264 + 15; with eight per CU 256 + 15).
    const long long groups = (a.Lk + 127LL) / 128 * a.B * a.Hk, tiles = ((long long)a.Lq * a.G + token::rows_of(a) - 1) / token::rows_of(a);
    long long s = groups > 0 ? ((a.q_docs ? 1024 : 512) + groups - 1) / groups : 1;
    if (s > tiles / token::run_of(a.q_docs)) s = tiles / token::run_of(a.q_docs);
    a.row_splits = s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

size_t token_attn_bwd_workspace(TokenAttnArgs& a, char* base) {
    token::Parts parts{base};
    const int per = token::rows_of(a);
    const size_t tiles = ((size_t)a.Lq * a.G + per - 1) / per * a.B * a.Hk;
    parts.take(a.facts, tiles * per * (a.type == TOKEN_F32 ? 3 : 2));
    parts.take(a.row_flags, tiles);
    if (a.row_splits > 1) {
        parts.take(a.grad_part, (size_t)a.row_splits * a.B * a.Lk * a.Hk * 2 * a.D);
        parts.take(a.grad_active, (size_t)a.B * a.Hk * ((a.Lk + 127) / 128));
    }
    if (a.k_docs) {
        parts.take(a.k_ranges, (size_t)a.B * ((a.Lk + 31) / 32));
        parts.take(a.q_ranges, (size_t)a.B * (((size_t)a.Lq * a.G + per - 1) / per));
    }
    return parts.bytes;
}

hipError_t launch_token_attn_bwd(const TokenAttnArgs& a, hipStream_t stream) {
    if (a.k_docs && a.Lk > 0 && a.Lq > 0) {
        const int per = token::rows_of(a), keys = token::keys_of(a), k_tiles = (a.Lk + keys - 1) / keys, q_tiles = (a.Lq * a.G + per - 1) / per;
        if (hipError_t e = token::launch_ranges(a.k_docs, a.k_ranges, a.Lk, 1, keys, k_tiles, a.B, stream); e != hipSuccess) return e;
        if (hipError_t e = token::launch_ranges(a.q_docs, a.q_ranges, a.Lq, a.G, per, q_tiles, a.B, stream); e != hipSuccess) return e;
    }
    switch (a.type) {
        case TOKEN_F32: return token::bwd_type<float>(a, stream);
        case TOKEN_BF16: return token::bwd_type<__bf16>(a, stream);
        default: return token::bwd_type<_Float16>(a, stream);
    }
}

}  // namespace danra
