// softmax attention with capped scores, a distance bias and positional / document masks, forward (token_attn.h has the formulas and
// the layout).  One pass over the keys with the running maximum m and sum l of each row:
//   S^T = K Q^T (rows: keys, columns: query rows), p = 2^(S - m), O^T += V^T P^T, and O^T and l are multiplied by 2^(m - m') where a
//   row's maximum grows by more than 8 (below that the powers stay under 2^8 and nothing is rescaled).
// O, m and l are float32; P is rounded to the operand's type (2^-9 relative in bfloat16, of the size of the rounding of V itself).  The sum
// that O is divided by is taken of the ROUNDED values, two to an instruction: a row with one large p then keeps only the part (1 - p) of
// that p's rounding, in the result and in the rowsum(dout . out) that the backward pass forms from it (packed documents, scores of a spread
// of 3, in units of one rounding of the exact result: out, dq and dk 1.26, 1.21 and 1.18 off with the sum of the unrounded values, 1.13, 1.08
// and 1.07 so; the forward pass of 16 heads of 4096 tokens, D = 128, 162 and 164 us).  What the
// backward pass forms P with again is the sum of the unrounded ones.
//
// Two forms.  With many rows, the four waves of a workgroup hold 32 rows each and share every tile of keys through LDS.  With few
// (a token of each sequence: the G heads of a key head make the rows), the waves hold the SAME 32 rows and divide the keys, each
// streaming tiles of its own through a part of LDS of its own, and the keys are further split over workgroups until they fill the
// chip; a second kernel joins the splits.
//
// Measured (bfloat16, D = 128): 16 heads of 4096 tokens without a mask 153 - 164 us, 840 - 900 TFLOP/s (matrix unit 40 %, vector unit 42 % of
// the time); a capped causal prompt of 8192 tokens 383 us, 718 TFLOP/s: there the exponentials and the cap (two exponentials and a
// reciprocal a score, at a quarter of the rate) and the other instructions of a score take the vector unit 54 % of the time, the products
// the matrix unit 33 %, and the two waves of a SIMD take turns.  Packed documents, prefixes: 1.3 and 1.0 waves on a SIMD, as workgroups with few
// tiles end early.  One token of 16 sequences over up to 16384 keys: 163 us, 4.9 TB/s, what a copy reaches; bound by reading the cache.  A third
// wave per SIMD in half the registers spills and takes twice as long.
#include "token_attn.h"

namespace danra {
namespace token {

namespace {

constexpr float kGrow = 8.f;

template <typename T, int DK, bool SPLIT>
struct FwdShape {
    static constexpr int kSub = SPLIT ? 1 : (sizeof(T) == 2 ? 2 : 1);  // subtiles of 32 keys
    static constexpr int kKeys = 32 * kSub;
    static constexpr int kWaves = SPLIT ? 1 : 4;                       // that bring a tile together
    static constexpr int kTile = kKeys * Tile<T, DK>::kRowBytes;
    static constexpr int kBufs = SPLIT && kTile > 8192 ? 1 : 2;        // of keys and values: two, where four waves' fit into the LDS
    static constexpr int kLds = (SPLIT ? 4 : 1) * kBufs * 2 * kTile;
    static constexpr int kJoin = SPLIT ? 2 * 32 * 32 * ((DK + 31) / 32) * 4 : 0;  // two waves' O
};

// P is kept times 2^6 in fp16: at most 2^14, and small ones stay normal numbers
template <typename T>
__device__ constexpr float shift_of() { return Type<T>::kNarrow ? 6.f : 0.f; }

// An infinite maximum is the mark of a row that sees no key (l = 0) and of no other: a row with an infinite score, whose l is no number,
// has no number for a maximum either.
template <typename T>
__device__ __forceinline__ float2 stats_of(float m, float l) {
    return l == 0.f ? make_float2(INFINITY, 0.f) : make_float2(m == INFINITY ? __builtin_nanf("") : m, log2f(l) - shift_of<T>());
}

// four channels of a result row, and what their rounding leaves over: the backward pass forms rowsum(dout . out), which enters every
// score gradient of the row, from both
template <typename T>
__device__ __forceinline__ void write_out(const TokenAttnArgs& a, size_t at, const f32x4& o, float l) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T4 x, r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = l == 0.f ? 0.f : o[e] * inv;
        x[e] = (T)y;
        r[e] = (T)(y - (float)x[e]);
    }
    *reinterpret_cast<T4*>(static_cast<T*>(a.out) + at) = x;
    if (sizeof(T) == 2 && a.rest) *reinterpret_cast<T4*>(static_cast<T*>(a.rest) + at) = r;
}

// KEEP: a backward pass follows.
template <typename T, int DK, bool SPLIT, Cap CAP, bool KEEP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DK >= 64) || (SPLIT && DK > 64) ? 1 : 2) void k_token_attn_fwd(const TokenAttnArgs a) {
    typedef FwdShape<T, DK, SPLIT> Sh;
    typedef Tile<T, DK> Tl;
    typedef Type<T> Ty;
    constexpr int NS = Sh::kSub, KS = DK / 16, DT = (DK + 31) / 32;
    constexpr float kShift = shift_of<T>();
    __shared__ __align__(16) char lds[Sh::kLds > Sh::kJoin ? Sh::kLds : Sh::kJoin];
    __shared__ __align__(16) int ids[2][SPLIT ? 4 * 64 : 64];
    __shared__ float4 ml[4][32];
    __shared__ int shared_range[4][3];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const Rows rows{a.G, a.magic};
    const int total = a.Lq * a.G;
    int tile, bh;
    place(a.B * a.Hk, tile, bh);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int per = SPLIT ? 32 : 128;
    if (a.causal) tile = (total + per - 1) / per - 1 - tile;  // the longest rows first
    const int row = tile * per + (SPLIT ? 0 : wave * 32) + col;

    const Mask mask = make_mask(a, b);
    const int query = rows.query(min(row, total - 1)), head = hk * a.G + (min(row, total - 1) - query * a.G);
    int doc = 0, limit = row < total ? max(mask.limit(query), 0) : 0;
    if (a.q_docs) {
        doc = a.q_docs[(size_t)b * a.Lq + query];
        if (doc < 0) limit = 0;
    }
    const int where = query + mask.shift;
    const Score score = make_score<CAP>(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2e / score.out : 0.f;

    const int wave_limit = __builtin_amdgcn_readfirstlane(wave_max(limit)), lowest = __builtin_amdgcn_readfirstlane(wave_min(limit));
    int id_lo = 0, id_hi = 0;
    if (a.q_docs) {
        id_lo = wave_min(limit > 0 ? doc : 0x7fffffff);
        id_hi = wave_max(limit > 0 ? doc : -1);
    }
    int list_limit = wave_limit, list_lo = id_lo, list_hi = id_hi;
    if constexpr (!SPLIT) {
        if (lane == 0) {
            shared_range[wave][0] = wave_limit;
            shared_range[wave][1] = id_lo;
            shared_range[wave][2] = id_hi;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            list_limit = max(list_limit, shared_range[w][0]);
            list_lo = min(list_lo, shared_range[w][1]);
            list_hi = max(list_hi, shared_range[w][2]);
        }
    }
    list_limit = __builtin_amdgcn_readfirstlane(list_limit);

    typename Ty::Frag qf[KS];
    {
        const T* q = static_cast<const T*>(a.q) + (long long)b * a.q_stride[0] + (long long)query * a.q_stride[1] +
                     (long long)head * a.q_stride[2];
        load_owner<T, DK>(qf, limit > 0 ? q : nullptr, a.D, lane);
        owner_sign<T>(qf, a.scale);
    }
    const T* kbase = static_cast<const T*>(a.k) + (long long)b * a.k_stride[0] + (long long)hk * a.k_stride[2];
    const T* vbase = static_cast<const T*>(a.v) + (long long)b * a.v_stride[0] + (long long)hk * a.v_stride[2];
    const int* kdocs = a.k_docs ? a.k_docs + (size_t)b * a.Lk : nullptr;
    const int4* ranges = a.k_ranges ? a.k_ranges + (size_t)b * ((a.Lk + Sh::kKeys - 1) / Sh::kKeys) : nullptr;

    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    float m = -INFINITY, l = 0.f, l_true = 0.f;  // (l: of the rounded values; l_true: of the unrounded, KEEP)
    // Whether the row sees a key, for rows whose l stays 0, which those have as well whose scores are all -infinity (a cap leaves none of them).
    // Without documents the limit tells.  With them it is found behind the loop where l is 0; but with the keys divided l is 0 in many a part,
    // and it is found in the loop, by the tiles of one document and, where they are mixed, by those with such a score (600 tokens: 9 us,
    // found behind the loop 13; by rows at D = 128 finding it in the loop spills).
    bool sees = CAP == kNoCap && !a.k_docs && limit > 0;

    int first = 0, last = (list_limit + Sh::kKeys - 1) / Sh::kKeys;
    if constexpr (SPLIT) {
        const int each = (last + a.splits - 1) / a.splits;
        first = blockIdx.y * each;
        last = min(last, first + each);
    }
    TileList list;
    list.start(ranges, nullptr, list_lo, list_hi, id_lo, id_hi, first, last, lane);
    const int stager = SPLIT ? 0 : wave;
    char* const own = SPLIT ? lds + wave * Sh::kBufs * 2 * Sh::kTile : lds;
    Rowwise<T, DK, Sh::kKeys, Sh::kWaves> keys, values;
    const unsigned k_step = (unsigned)a.k_stride[1] * (unsigned)sizeof(T), v_step = (unsigned)a.v_stride[1] * (unsigned)sizeof(T);
    keys.prepare(k_step, a.D, stager, lane);
    values.prepare(v_step, a.D, stager, lane);

    auto stage = [&](const Visit& x, int buf) {
        const int k0 = x.t * Sh::kKeys, count = mask.kv_len - k0;
        char* to = own + buf * 2 * Sh::kTile;
        auto dead = [&](int r) { return r < count && kdocs[k0 + r] < 0; };
        keys.load(kbase + (long long)k0 * a.k_stride[1], count, k_step, a.D, to, stager, lane, x.dead, dead);
        values.load(vbase + (long long)k0 * a.v_stride[1], count, v_step, a.D, to + Sh::kTile, stager, lane, x.dead, dead);
        // (ids past the sequence's end read as 0: those keys lie past every row's limit)
        if (kdocs && stager == 0) load_lds4(buffer(kdocs + k0, 4u * min(count, Sh::kKeys)), 4u * lane, (char*)&ids[buf][SPLIT ? wave * 64 : 0]);
    };
    auto advance = [&]() {  // the next tile of this wave (SPLIT: every fourth one) or workgroup
        Visit x = list.next(lane);
        if constexpr (SPLIT) {
            for (int n = 0; n < 3 && x.t >= 0; ++n) x = list.next(lane);
        }
        return x;
    };
    auto settle = [&]() {  // what was brought may be read, what was read may be overwritten
        if constexpr (SPLIT) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // this wave's own loads and reads
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            settle_loads();
            __syncthreads();
        }
    };

    // one tile from LDS; `whole`: no row's limit lies inside it.  (One body with the masks behind uniform branches: two bodies left the
    // accumulators in different registers, 50 to 140 moves a tile.)
    auto process = [&](bool whole, const Visit& x, int buf) {
        const char* kt = own + buf * 2 * Sh::kTile;
        const char* vt = kt + Sh::kTile;
        const int k0 = x.t * Sh::kKeys;
        f32x16 s[NS];
        typename Ty::Frag vf[2][DT];
        // fragments are read kAhead products ahead, in groups that the scheduler may not take apart: left alone, it reads each where it is
        // needed and waits for it
        constexpr int kAhead = KS < 4 ? KS : KS % 4 ? 3 : 4, kGroups = NS * KS / kAhead;
        static_assert(KS % kAhead == 0, "whole groups");
        typename Ty::Frag kf[2][kAhead];
        auto read_keys = [&](int g) {
#pragma unroll
            for (int c = 0; c < kAhead; ++c) {
                const int at = g * kAhead + c;
                kf[g & 1][c] = Tl::row(kt, 32 * (at / KS) + col, 16 * (at % KS) + 8 * half);
            }
        };
        read_keys(0);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g + 1 < kGroups) read_keys(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < kAhead; ++c) {
                const int at = g * kAhead + c;
                if (at % KS == 0) s[at / KS] = f32x16{};
                s[at / KS] = Ty::mfma(kf[g & 1][c], qf[at % KS], s[at / KS]);
            }
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < DT; ++d) vf[h][d] = Tl::column(vt, 16 * h, 32 * d, lane);
        }
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = bend<CAP>(s[n][e], score);
            const int j0 = k0 + 32 * n + 4 * half;
            if (a.slopes) {
                const float from = (float)(where - j0);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = fmaf(-slope, fabsf(from - (float)(8 * (e >> 2) + (e & 3))), s[n][e]);
            }
            if constexpr (SPLIT && CAP == kNoCap) {
                if (a.k_docs && x.same) {
                    sees |= k0 < limit;
                } else if (a.k_docs && __any(m == -INFINITY && k0 < limit)) {
                    float low = __builtin_elementwise_minimum(s[n][0], s[n][1]);
#pragma unroll
                    for (int e = 2; e < 16; e += 2) low = __builtin_elementwise_minimum(low, __builtin_elementwise_minimum(s[n][e], s[n][e + 1]));
                    if (__any(low == -INFINITY)) {
                        const int* id = &ids[buf][(SPLIT ? wave * 64 : 32 * n) + 4 * half];
                        for (int e = 0; e < 16; ++e) {
                            const int at = 8 * (e >> 2) + (e & 3);
                            sees |= at < limit - j0 && id[at] == doc;
                        }
                    }
                }
            }
            if (!whole) {
                const int left = limit - j0;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = 8 * (e >> 2) + (e & 3) < left ? s[n][e] : -INFINITY;
            }
            if (!x.same) {
                const int* id = &ids[buf][(SPLIT ? wave * 64 : 32 * n) + 4 * half];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 d = *reinterpret_cast<const int4*>(id + 8 * g);
                    s[n][4 * g + 0] = d.x == doc ? s[n][4 * g + 0] : -INFINITY;
                    s[n][4 * g + 1] = d.y == doc ? s[n][4 * g + 1] : -INFINITY;
                    s[n][4 * g + 2] = d.z == doc ? s[n][4 * g + 2] : -INFINITY;
                    s[n][4 * g + 3] = d.w == doc ? s[n][4 * g + 3] : -INFINITY;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e += 2) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(s[n][e], s[n][e + 1]));
        }
        top = pair_max(top) * score.out;
        if (__any(top > m + kGrow)) {
            const float now = fmaxf(m, top);
            const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= keep;
            l_true *= keep;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= keep;
        }
        const float base = m == -INFINITY ? 0.f : m - kShift;
        constexpr bool kBoth = KEEP && sizeof(T) == 2;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[n][e] = __builtin_amdgcn_exp2f(fmaf(s[n][e], score.out, -base));
                if constexpr (kBoth || sizeof(T) == 4) sum[e & 3] += s[n][e];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const typename Ty::Frag p = round_frag<T>(s[n], h);
                if constexpr (sizeof(T) == 2) l = Ty::sum(p, l);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    if constexpr (sizeof(T) == 2) {
                        o[d] = Ty::mfma(vf[h][d], p, o[d]);
                        if (n + 1 < NS) vf[h][d] = Tl::column(vt, 32 * (n + 1) + 16 * h, 32 * d, lane);
                    } else {
                        o[d] = Ty::mfma(Tl::column(vt, 32 * n + 16 * h, 32 * d, lane), p, o[d]);
                    }
                }
            }
        }
        const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (sizeof(T) == 4) l += all;
        else if constexpr (kBoth) l_true += all;
    };

    auto work = [&](const Visit& x, auto buf) {
        const int k0 = x.t * Sh::kKeys;
        if (x.wanted && k0 < wave_limit) process(k0 + Sh::kKeys <= lowest, x, buf());
    };
    if constexpr (SPLIT) {
        Visit x = list.next(lane);
        for (int n = 0; n < wave && x.t >= 0; ++n) x = list.next(lane);
        int buf = 0;
        if (x.t >= 0) {
            stage(x, 0);
            settle();
        }
        while (x.t >= 0) {
            const Visit after = advance();
            if (Sh::kBufs == 2 && after.t >= 0) stage(after, buf ^ 1);
            work(x, [&]() { return buf; });
            if (after.t >= 0) {
                settle();
                if (Sh::kBufs == 1) {
                    stage(after, 0);
                    settle();
                }
            }
            buf ^= Sh::kBufs - 1;
            x = after;
        }
    } else {
        two_buffers(advance, stage, work);
    }
    l = pair_sum(l);
    l_true = sizeof(T) == 4 ? l : KEEP ? pair_sum(l_true) : 0.f;
    if constexpr (CAP == kNoCap && SPLIT) {
        sees = pair_max(sees ? 1.f : 0.f) > 0.f;
    } else if constexpr (CAP == kNoCap) {
        if (a.k_docs && __any(limit > 0 && l == 0.f)) {
            list.start(ranges, nullptr, list_lo, list_hi, id_lo, id_hi, first, last, lane);
            for (Visit x = list.next(lane); x.t >= 0; x = list.next(lane)) {
                const int k0 = x.t * Sh::kKeys, end = min(Sh::kKeys, wave_limit - k0), id = lane < end ? kdocs[k0 + lane] : -1;
                for (int j = 0; j < end; ++j) sees |= k0 + j < limit && __builtin_amdgcn_readlane(id, j) == doc;
            }
        }
    }

    if constexpr (SPLIT) {  // the four waves' sums, in a fixed order: (0 + 2) + (1 + 3)
        if (half == 0) ml[wave][col] = make_float4(m, l, l_true, sees ? 1.f : 0.f);
        __syncthreads();
        float all = -INFINITY, sum = 0.f, sum_true = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) all = fmaxf(all, ml[w][col].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 x = ml[w][col];
            const float by = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - all);
            sum += x.y * by;
            sum_true += x.z * by;
            sees |= x.w != 0.f;
        }
        const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - all);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= keep;
        float* join = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int step = 2; step >= 1; --step) {
            __syncthreads();
            if (wave >= step && wave < 2 * step) {
                float* to = join + (wave - step) * 32 * 32 * DT;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) to[(d * 16 + e) * 64 + lane] = o[d][e];
            }
            __syncthreads();
            if (wave < step) {
                const float* from = join + wave * 32 * 32 * DT;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] += from[(d * 16 + e) * 64 + lane];
            }
        }
        if (wave) return;
        m = all;
        l = sum;
        l_true = sum_true;
        if (a.splits > 1) {
            if (row < total) {
                const size_t at = ((size_t)bh * a.splits + blockIdx.y) * total + row;
                if (half == 0) a.part_ml[at] = make_float4(m, l, l_true, sees ? 1.f : 0.f);
                float* to = a.part + at * a.D;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int c = 32 * d + 8 * g + 4 * half;
                        if (c < a.D) *reinterpret_cast<f32x4*>(to + c) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                    }
            }
            return;
        }
    }

    if (sees && l == 0.f) l = l_true = __builtin_nanf("");  // 0 / 0, and not a row without keys
    if (row < total) {
        if (a.stats && half == 0) a.stats[(size_t)bh * total + row] = stats_of<T>(m, l_true);
        const size_t at = (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * half;
                if (c < a.D) write_out<T>(a, at + c, f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]}, l);
            }
    }
}

// out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s: a thread per row and four channels, the splits in order.  With few rows it is bound by
// the trips to memory, so kJoin splits are asked for at a time.
constexpr int kJoin = 8;
template <typename T>
__global__ __launch_bounds__(256) void k_token_attn_join(const TokenAttnArgs a) {
    const int total = a.Lq * a.G, quads = a.D >> 2;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long at = item / quads;  // (batch and key head, row)
    if (at >= (long long)a.B * a.Hk * total) return;
    const int c = 4 * (int)(item - at * quads);
    const int bh = (int)(at / total), row = (int)(at - (long long)bh * total);
    const float4* ml = a.part_ml + (size_t)bh * a.splits * total + row;
    float m = -INFINITY, l = 0.f, l_true = 0.f;
    for (int s0 = 0; s0 < a.splits; s0 += kJoin) {
        float x[kJoin];
#pragma unroll
        for (int u = 0; u < kJoin; ++u) x[u] = ml[(size_t)min(s0 + u, a.splits - 1) * total].x;
#pragma unroll
        for (int u = 0; u < kJoin; ++u) m = fmaxf(m, x[u]);
    }
    bool sees = false;
    f32x4 o = {0, 0, 0, 0};
    const float* parts = a.part + ((size_t)bh * a.splits * total + row) * a.D + c;
    for (int s0 = 0; s0 < a.splits; s0 += kJoin) {
        float4 x[kJoin];
        f32x4 part[kJoin];
#pragma unroll
        for (int u = 0; u < kJoin; ++u) {
            const size_t s = min(s0 + u, a.splits - 1);
            x[u] = ml[s * total];
            part[u] = *reinterpret_cast<const f32x4*>(parts + s * total * a.D);
        }
#pragma unroll
        for (int u = 0; u < kJoin; ++u) {
            if (s0 + u >= a.splits) break;
            const float w = x[u].x == -INFINITY ? (x[u].y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(x[u].x - m);
            l += w * x[u].y;
            l_true += w * x[u].z;
            sees |= x[u].w != 0.f;
            if (w != 0.f) {  // (a split that saw nothing may hold 0 x infinity)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(w, part[u][e], o[e]);
            }
        }
    }
    if (sees && l == 0.f) l = l_true = __builtin_nanf("");
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const Rows rows{a.G, a.magic};
    const int query = rows.query(row), head = hk * a.G + row - query * a.G;
    if (a.stats && c == 0) a.stats[at] = stats_of<T>(m, l_true);
    write_out<T>(a, (((size_t)b * a.Lq + query) * (a.Hk * a.G) + head) * a.D + c, o, l);
}

template <typename T, int DK, Cap CAP, bool KEEP>
hipError_t fwd(const TokenAttnArgs& a, hipStream_t stream) {
    const int total = a.Lq * a.G, heads = a.B * a.Hk;
    if (a.by_keys) {
        const dim3 grid((unsigned)((total + 31) / 32) * heads, a.splits);
        DANRA_LAUNCH_KERNEL((k_token_attn_fwd<T, DK, true, CAP, KEEP>), grid, dim3(256), 0, stream, a);
        if (a.splits > 1) {
            const long long items = (long long)heads * total * (a.D / 4);
            DANRA_LAUNCH_KERNEL((k_token_attn_join<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, a);
        }
    } else {
        const dim3 grid((unsigned)((total + 127) / 128) * heads);
        DANRA_LAUNCH_KERNEL((k_token_attn_fwd<T, DK, false, CAP, KEEP>), grid, dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

template <typename T, int DK, bool KEEP>
hipError_t fwd(const TokenAttnArgs& a, hipStream_t stream) {
    switch (cap_of(a)) {
        case kNoCap: return fwd<T, DK, kNoCap, KEEP>(a, stream);
        case kQuick:
            if constexpr (sizeof(T) == 2) return fwd<T, DK, kQuick, KEEP>(a, stream);
        default: return fwd<T, DK, kExact, KEEP>(a, stream);
    }
}

template <typename T, int DK>
hipError_t fwd(const TokenAttnArgs& a, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (!a.stats) return fwd<T, DK, false>(a, stream);
    }
    return fwd<T, DK, true>(a, stream);
}

template <typename T>
hipError_t fwd_type(const TokenAttnArgs& a, hipStream_t stream) {
    if (a.D <= 16) return fwd<T, 16>(a, stream);
    if (a.D <= 32) return fwd<T, 32>(a, stream);
    if (a.D <= 64) return fwd<T, 64>(a, stream);
    if (a.D <= 96) return fwd<T, 96>(a, stream);
    return fwd<T, 128>(a, stream);
}

// keys of a tile: 64 where four waves share it in a two-byte type, else 32
int keys_of(const TokenAttnArgs& a) { return !a.by_keys && a.type != TOKEN_F32 ? 64 : 32; }

}  // namespace

// {lowest, highest, all equal, some negative} of the ids of each `per` consecutive places (negative ids left out; a place past the end
// counts as one);
// place p stands for id p / group: a wave per tile
__global__ __launch_bounds__(256) void k_token_ranges(const int* __restrict__ ids, int4* __restrict__ out, int length, int group, int per,
                                                      int tiles, int batch) {
    const int item = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (item >= tiles * batch) return;
    const int b = item / tiles, t = item - b * tiles;
    int lo = 0x7fffffff, hi = -1, none = 0;
    for (int p = lane; p < per; p += 64) {
        const int at = (t * per + p) / group;
        const int id = at < length ? ids[(size_t)b * length + at] : -1;
        if (id >= 0) {
            lo = min(lo, id);
            hi = max(hi, id);
        } else {
            none = 1;
        }
    }
    lo = wave_min(lo);
    hi = wave_max(hi);
    none = wave_max(none);
    if (lane == 0) out[item] = make_int4(lo, hi, lo == hi && !none, none);
}

hipError_t launch_ranges(const int* ids, int4* out, int length, int group, int per, int tiles, int batch, hipStream_t stream) {
    DANRA_LAUNCH_KERNEL(k_token_ranges, dim3((tiles * batch + 3) / 4), dim3(256), 0, stream, ids, out, length, group, per, tiles, batch);
    return hipGetLastError();
}

}  // namespace token

void plan_token_attn_fwd(TokenAttnArgs& a) {
    const long long total = (long long)a.Lq * a.G, heads = (long long)a.B * a.Hk;
    // The waves of a form by rows walk over all keys, however few they are: its time is that of one workgroup until the CUs are full.  The
    // form by keys takes the time of its work.  They meet at 320 groups of 32 rows (16 heads over 4096 keys, D = 128: 512 rows 64 us by
    // keys, 87 by rows; 640 rows 88 either way; 896 rows 115 and 91; single tokens of 512 key heads over 2048 keys 107 and 99).
    const long long groups = (total + 31) / 32 * heads;
    a.by_keys = groups < 320;
    // The keys are split until there are about two workgroups per CU, each with at least 512 of them, four tiles to a wave (4 sequences, 4 key
    // heads: 1024 keys 13 us and 4 for the join, with 1024 a split 19, with 256 11 + 4; 512 keys 13, with 256 11 + 4; 8192 keys 18 + 7, with 1024
    // 21 + 5, with 256 23 + 13).
    a.splits = 1;
    if (a.by_keys && total * heads > 0) {
        long long s = (512 + groups - 1) / groups;
        s = s < (a.Lk + 511) / 512 ? s : (a.Lk + 511) / 512;
        a.splits = s < 1 ? 1 : s > 128 ? 128 : (int)s;
    }
}

size_t token_attn_fwd_workspace(TokenAttnArgs& a, char* base) {
    token::Parts parts{base};
    if (a.splits > 1) {
        const size_t rows = (size_t)a.B * a.Hk * a.splits * a.Lq * a.G;
        parts.take(a.part, rows * a.D);
        parts.take(a.part_ml, rows);
    }
    if (a.k_docs) parts.take(a.k_ranges, (size_t)a.B * ((a.Lk + 31) / 32));
    return parts.bytes;
}

hipError_t launch_token_attn_fwd(const TokenAttnArgs& a, hipStream_t stream) {
    if (a.k_docs && a.Lk > 0) {
        const int per = token::keys_of(a), tiles = (a.Lk + per - 1) / per;
        if (hipError_t e = token::launch_ranges(a.k_docs, a.k_ranges, a.Lk, 1, per, tiles, a.B, stream); e != hipSuccess) return e;
    }
    switch (a.type) {
        case TOKEN_F32: return token::fwd_type<float>(a, stream);
        case TOKEN_BF16: return token::fwd_type<__bf16>(a, stream);
        default: return token::fwd_type<_Float16>(a, stream);
    }
}

}  // namespace danra
