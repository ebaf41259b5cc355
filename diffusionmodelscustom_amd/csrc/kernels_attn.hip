// Self-attention cores on gfx950.
//
// k_flash_hd16: head_dim 16 (every 64-channel level: L = 256 / 1024 / 4096 tokens).  Flash-style:
// no L x L matrix ever leaves the registers.  The matrix cores compute S^T = K Q^T, so that a lane holds
// 16 scores of ONE query (q = lane & 15) and the row maximum / sum are lane-local plus two cross-lane
// exchanges; the same accumulator registers are then the B operand of O^T = V^T P^T without passing
// through LDS.  Online softmax in the exp2 domain.  Both products run as split-operand fp16 products with
// fp32 accumulation (22 significant bits per operand, see PVH / QKH below) and fall back to the fp32
// instructions (v_mfma_f32_16x16x4_f32) when an operand leaves the fp16 range.
//
// k_attn_reg: the deeper levels (L <= 256 tokens, head_dim 32 / 64 / 128): one wave per 16-query tile, all
// score tiles in registers, exact two-pass softmax, operands read straight from memory.
//
// k_flash_wide: the flash scheme for head_dim 32 / 64 and L a multiple of 128 (networks with 2 heads or 1 head).
//
// k_attn_small: fallback for any other shape (plain VALU, keys walked in LDS chunks with online softmax).
#include <type_traits>

#include "danra_kernels.h"
#include "split_f16.h"

namespace danra {

typedef float f32x4 __attribute__((ext_vector_type(4)));


// QT = 16-query tiles per wave (template parameter of k_flash_hd16)
static constexpr int KVT = 64;  // keys per LDS tile
static constexpr int KROW = 20; // padded LDS row (floats) of a 16-float K/V row: conflict-free b32 column reads
static constexpr float RESCALE_LOG2 = 24.f;  // move the softmax reference when a score exceeds it by 2^24

// Becomes one v_max3_f32: this file is compiled with -fno-honor-nans, otherwise fmaxf adds a
// canonicalising v_max per operand that comes out of an MFMA.  (Not inline asm: the compiler does not
// insert the MFMA-result wait states in front of an asm statement.)
__device__ __forceinline__ float max3f(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// ABL: timing ablations for tune_flash (results are wrong unless 0): 1 = no exp2, 2 = no V reads from LDS,
// 4 = no staging/barrier after the first tile, 8 = no QK^T MFMAs, 16 = no PV MFMAs.
//
// PVH: O^T += V^T P^T on the fp16 matrix cores with both operands split in two fp16 halves:
// V^T P^T ~ Vhi Phi + Vhi Plo + Vlo Phi, three v_mfma_f32_16x16x32_f16 (one per 32 keys, fp32 accumulation)
// instead of eight fp32 products; the dropped Vlo Plo term is 2^-22 of the product.
//   P = hi + lo with hi = fp16(P), lo = fp16(P - hi).  P lies in [0, 2^15] (the reference moves at 2^15 in this
//      form) against a row sum >= 1: a probability above 2^-3 keeps 22 significant bits, a smaller one is off by at
//      most 2^-25 (lo is then an fp16 subnormal; the matrix cores and the conversions honour subnormals).
//   V = hi + 2^-11 lo with lo = fp16(2^11 (V - hi)); the Vlo Phi products have an accumulator of their own that is
//      scaled once, at the end.  |V| in 2^-14 ... 2^15 keeps 22 bits, smaller values are off by at most 2^-36.
// V tiles are taken this way only while every |V| staged so far is below 2^15 and every 16 keys x 16 columns
// staged by one wave hold a value of at least 2^-10 (so that the absolute bound is small against the largest
// value): the staging threads raise a workgroup flag otherwise (also for NaN/Inf), and from that tile on the
// workgroup multiplies in fp32 as before.
// (Tried and dropped: a reference 2^11 lower, which would keep Plo out of the subnormals as well.  That kernel gave
// run-to-run varying results in the second query tile of a wave on strongly peaked rows; the cause was not found.)
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
//
// QKH: S^T = K Q^T on the fp16 matrix cores as well.  Both operands are split as x = h + 2^-11 l, h = fp16(x),
// l = fp16(2^11 (x - h)) (Q after its multiplication by hd^-1/2 log2 e); the three products that matter are two
// 32-deep instructions per 16 keys and query tile that read the SAME K fragment, with NO arithmetic in the loop (K is
// split by the staging threads, Q once per kernel):  [Kh | Kl] [Qh | 2^-11 Qh]^T  +  [Kh | Kl] [2^-11 Ql | 0]^T  =
// Kh Qh + 2^-11 (Kl Qh + Kh Ql).  Every 2^-11 factor sits on the Q side, so a key row of the LDS tile is just its 32
// halves (64 bytes: a quarter of the tile's reads and half of its bytes against a tile that also carries 2^-11 Kh).
// The 2^-11 copies may be fp16 subnormals (quantum 2^-24), which bounds the absolute score error by
// 16 * 2^-23 max|K| on top of 2^-22 sum|k q'| for the dropped Kl Ql term.  The softmax reference still
// enters as the C operand of the first product.  The range flag covers |K| and |Q'| < 2^15 as it does V.
// Row layout: four groups of [h 4 | l 4] halves (columns 4g .. 4g + 3 of both parts are the eight k-slots of lane group g),
// so a staging thread writes its four columns as one 16-byte store and the fragment reads of a wave are 1 KB in a line.
static constexpr int KHROW = 32;  // halves per key row of the fp16 K tile
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
// KT64: 64-key sub-tiles per staged tile (one barrier per 64 * KT64 keys; 2 measured equal to 1 within the run-to-run
// spread, in tune_flash and in the network, so the library uses 1)
//
// PRE: K and V arrive already split, in the order of the LDS tiles, from the kernels that produce them (the QKV
// projections of the network, or launch_presplit_kv): K and V then point at those copies, staging a tile is a straight
// 8 KB copy with no arithmetic, and the range test has been made by the producer: pre.flags holds, per (image, head) and
// group of 16 keys, whether K (word 0) or V (word 1) of that group left the range of the split.  Only for such a group
// does the producer also write the fp32 values (pre.k32 / pre.v32, the [key][16] layout of the other form): a tile with
// a flagged group, and every tile of a wave whose own queries leave the fp16 range, is multiplied with the fp32
// instructions, per group from the fp32 values where they exist and from the sum of the halves (22 bits) elsewhere.
struct FlashPre {
    const float* k32;
    const float* v32;
    const int* flags;
};
// TOK: Q, K and V are read where a fused QKV projection leaves them - rows of one (image, head) lay.rs floats apart, the
// (image, head) pair at b * lay.img + head * lay.hs - instead of [n_bh][L][16] (the training step's in_proj output
// [B][L][3][heads * 16] is then used in place: rs = 3 heads 16, img = L rs, hs = 16, and K, V = Q + heads 16, + 2 heads 16).
template <int QT, int ABL = 0, bool PVH = true, bool QKH = PVH, int KT64 = 1, bool PRE = false, bool TOK = false>
__global__ __launch_bounds__(256) void k_flash_hd16(const float* __restrict__ Q, const float* __restrict__ K,
                                                    const float* __restrict__ V, float* __restrict__ O,
                                                    float* __restrict__ LSE2, int L, int heads, int n_bh,
                                                    float scale_log2e, const FlashPre pre, const QkvLayout lay) {
    static_assert(!PRE || (PVH && QKH && KT64 == 1), "pre-split operands: the fp16 form, 64 keys per tile");
    static_assert(!(PRE && TOK), "pre-split operands have their own layout");
    // fp32 tiles only in the all-fp32 form; the fp32 fallback of the fp16 forms (rare) reads global memory instead
    constexpr bool F32_TILES = !(PVH && QKH);
    __shared__ __attribute__((aligned(16))) float Ks[F32_TILES ? 2 : 1][F32_TILES ? KT64 * KVT * KROW : 4];
    __shared__ __attribute__((aligned(16))) float Vs[F32_TILES ? 2 : 1][F32_TILES ? KT64 * KVT * KROW : 4];
    // fp16 halves of the V tile in the A-operand order of the 32-deep product: [buffer][hi, lo][32-key half]
    // [d][g][slot], slot 4j + r <-> key 16j + 4g + r of the half (the order in which a lane holds its 8 scores)
    __shared__ __attribute__((aligned(16))) _Float16 Vh[PVH ? 2 : 1][2][2 * KT64][PVH ? 16 * 4 * 8 : 8];
    __shared__ __attribute__((aligned(16))) _Float16 Kh[QKH ? 2 : 1][QKH ? KT64 * KVT * KHROW : 8];
    // range flags, one per staging buffer: set (never cleared) by the threads that stage a tile into that buffer and read
    // at the top of the iteration that consumes it.  With a single flag a wave that runs ahead could raise it for tile
    // kt + 2 while a slower wave still decides about tile kt + 1, and which products that wave then used would depend on
    // timing; a buffer's flag is only written again behind the barrier that ends the iteration that read it.
    __shared__ int vbig_s[2];
    __shared__ int grp_s[PRE ? 2 : 1][8];   // PRE: the producer's flags of the staged tile: [16-key group][K, V]
    static_assert(PVH == QKH, "both products run on the fp16 matrix cores, or neither");
    constexpr float RESCALE = PVH ? 15.f : RESCALE_LOG2;  // log2 of the largest probability relative to the reference
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Workgroups are dealt round-robin over the 8 XCDs (id % 8 labels the XCD group).  The linear id is
    // decoded as (bh / 8, query block, bh % 8), so every query block of one (image, head) pair runs on the
    // same XCD and its K/V rows are fetched into one L2 instead of eight.  (Speed only.)
    const int nq = L / (4 * QT * 16);
    int bh, qblk;
    if (n_bh % 8 == 0) {
        const int id = blockIdx.x;
        bh = (id / (8 * nq)) * 8 + (id & 7);
        qblk = (id >> 3) % nq;
    } else {
        bh = blockIdx.x / nq;
        qblk = blockIdx.x - bh * nq;
    }
    const int q0 = qblk * (4 * QT * 16) + wave * (QT * 16);
    const int lq = lane & 15;  // query column / key row / d column, depending on the operand
    const int g = lane >> 4;   // k-slot of the MFMA

    const int RS = TOK ? lay.rs : 16;   // floats between two rows of an operand
    const size_t base = TOK ? (size_t)(bh / heads) * lay.img + (size_t)(bh % heads) * lay.hs : (size_t)bh * L * 16;
    const float* Qb = Q + base;
    const float* Kb = K + base;
    const float* Vb = V + base;

    // Q fragments: B operand of S^T = K Q^T: lane (q, g) holds Q[q][4g + r] for MFMA step r.
    // Q is pre-multiplied by hd^-1/2 * log2(e): scores come out of the matrix cores in the exp2 domain.
    auto load_qf = [&](int t) {
        float4 f = *reinterpret_cast<const float4*>(Qb + (size_t)(q0 + t * 16 + lq) * RS + 4 * g);
        f.x *= scale_log2e;
        f.y *= scale_log2e;
        f.z *= scale_log2e;
        f.w *= scale_log2e;
        return f;
    };
    float4 qf[F32_TILES ? QT : 1];  // kept in registers only in the all-fp32 form
    if (F32_TILES) {
#pragma unroll
        for (int t = 0; t < QT; ++t) qf[t] = load_qf(t);
    }

    // fp16 form of the Q fragments: lane (q, g) holds columns 4g ... 4g + 3.  First product: [Qh | 2^-11 Qh] against the
    // key row's [Kh | Kl]; second product: [2^-11 Ql | 0] = [fp16(x - h) | 0] against the same row (see QKH above)
    f16x8 qb1[QT], qb2[QT];
    bool q_bounded = true;
    if (QKH) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const float4 qa = *reinterpret_cast<const float4*>(Qb + (size_t)(q0 + t * 16 + lq) * RS + 4 * g);
            const float qq[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = qq[i] * scale_log2e;
                const _Float16 hi = (_Float16)x;
                qb1[t][i] = hi;
                qb1[t][4 + i] = (_Float16)((float)hi * 0.00048828125f);
                qb2[t][i] = (_Float16)(x - (float)hi);
                qb2[t][4 + i] = (_Float16)0.f;
                q_bounded = q_bounded && (fabsf(x) < 32768.f);
            }
        }
    }

    // Online softmax with a lazily updated reference: the reference is subtracted from the scores by feeding
    // its negative to the QK^T products as their C operand, so the common case needs no per-score
    // arithmetic before exp2.  The reference moves only on the first tile (to that tile's row maximum)
    // and when a score exceeds it by more than 2^RESCALE_LOG2 (fp32 has the headroom: probabilities
    // are then at most 2^24 relative to the reference and sums over 4096 keys stay far below 2^127).
    // negm[t] = -reference in all four registers: it is the C operand of the first QK^T product of every score
    // tile (no per-tile accumulator initialisation); lrun[t] keeps the row sum as two partial sums so that the
    // probabilities are added two at a time (packed fp32 adds).
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    f32x4 ot[QT], ot2[QT], negm[QT];  // ot2: 2^11 x the Vlo Phi terms of the fp16-halves products
    f32x2 lrun[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        ot[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        ot2[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        negm[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        lrun[t] = f32x2{0.f, 0.f};
    }

    // staging: 64 keys x 16 floats per operand.  K (and both operands of the all-fp32 form): one float4 per thread,
    // key srow, columns sc4 .. sc4 + 3.  V of the fp16 form: four floats per thread, ONE column vd of the four keys
    // that are neighbours in a lane's slot order (16 vj + 4 vg + r of half vhalf, r = 0..3: see Vh), so that their
    // halves leave as two 8-byte LDS writes (lanes l, l+1, .. walk vg then vd: conflict-free) instead of eight 2-byte
    // ones that collide four ways.
    const int srow = tid >> 2, sc4 = (tid & 3) * 4;
    const int vd = lane >> 2, vg = lane & 3, vj = wave & 1, vhalf = wave >> 1;
    const int vkey = 32 * vhalf + 16 * vj + 4 * vg;  // first of this thread's four keys within a tile
    constexpr int TK = KT64 * KVT;  // keys per staged tile
    float4 kreg[KT64], vreg[KT64];
    int flag_reg = 0;
    auto load_kv = [&](int tile) {
        if constexpr (PRE) {  // 4 KB of K rows and 4 KB of V fragments, both in the order of their LDS tiles
            kreg[0] = *reinterpret_cast<const float4*>(Kb + (size_t)tile * 1024 + tid * 4);
            vreg[0] = *reinterpret_cast<const float4*>(Vb + (size_t)tile * 1024 + tid * 4);
            if (tid < 8) flag_reg = pre.flags[((size_t)bh * (L / 16) + 4 * tile) * 2 + tid];
            return;
        }
#pragma unroll
        for (int u = 0; u < KT64; ++u) {
            kreg[u] = *reinterpret_cast<const float4*>(Kb + (size_t)(tile * TK + KVT * u + srow) * RS + sc4);
            if (PVH) {
                const float* vp = Vb + (size_t)(tile * TK + KVT * u + vkey) * RS + vd;
                vreg[u] = make_float4(vp[0], vp[RS], vp[2 * RS], vp[3 * RS]);
            } else {
                vreg[u] = *reinterpret_cast<const float4*>(Vb + (size_t)(tile * TK + KVT * u + srow) * RS + sc4);
            }
        }
    };
    load_kv(0);
    // x = h + 2^-11 l: h = fp16(x) rounded towards zero, l = fp16(2^11 (x - h)) (the difference is exact in fp32);
    // six instructions per pair of values
    auto split_scaled = [&](float x0, float x1, unsigned& h, unsigned& l) { split_scaled_pair_f16(x0, x1, h, l); };
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    auto stage = [&](int buf) {
        if constexpr (PRE) {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(&Kh[buf][0]) + tid * 4) = kreg[0];
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(&Vh[buf][0][0][0]) + tid * 4) = vreg[0];
            if (wave == 0) {
                const bool any = __any(tid < 8 && flag_reg != 0) != 0;
                if (tid < 8) grp_s[buf][tid] = flag_reg;
                if (tid == 0) vbig_s[buf] = any ? 1 : 0;
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < KT64; ++u) {
            const float4 kr = kreg[u], vr = vreg[u];
            if (F32_TILES) {
                *reinterpret_cast<float4*>(&Ks[buf][(KVT * u + srow) * KROW + sc4]) = kr;
                *reinterpret_cast<float4*>(&Vs[buf][(KVT * u + srow) * KROW + sc4]) = vr;
            }
            if (QKH) {
                unsigned h[2], l[2];
                split_scaled(kr.x, kr.y, h[0], l[0]);
                split_scaled(kr.z, kr.w, h[1], l[1]);
                typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
                *reinterpret_cast<u32x4*>(&Kh[buf][(KVT * u + srow) * KHROW + 2 * sc4]) = u32x4{h[0], h[1], l[0], l[1]};
                const float kmax = fmaxf(max3f(fabsf(kr.x), fabsf(kr.y), fabsf(kr.z)), fabsf(kr.w));
                if (!(kmax < 32768.f)) vbig_s[buf] = 1;
            }
            if (PVH) {
                unsigned h[2], l[2];
                split_scaled(vr.x, vr.y, h[0], l[0]);
                split_scaled(vr.z, vr.w, h[1], l[1]);
                const int at = (vd * 4 + vg) * 8 + 4 * vj;
                *reinterpret_cast<u32x2*>(&Vh[buf][0][2 * u + vhalf][at]) = u32x2{h[0], h[1]};
                *reinterpret_cast<u32x2*>(&Vh[buf][1][2 * u + vhalf][at]) = u32x2{l[0], l[1]};
                const float vmax = fmaxf(max3f(fabsf(vr.x), fabsf(vr.y), fabsf(vr.z)), fabsf(vr.w));
                // (a wave stages 16 keys x 16 columns.)  Never cleared: the tiles from this one on are multiplied in fp32
                if (!(vmax < 32768.f) || __all(vmax < 0.0009765625f)) vbig_s[buf] = 1;
            }
        }
    };
    if (PVH) {
        if (tid < 2) vbig_s[tid] = 0;
        __syncthreads();
    }
    stage(0);
    __syncthreads();

    const int ntiles = L / TK;
    // fp32 products: always in the all-fp32 form; in the fp16 form from the first tile on for a wave whose own queries
    // leave the fp16 range, and for every wave from the first flagged K / V tile on
    const bool q_big = PVH ? (__any(!q_bounded) != 0) : true;
    bool vbig = q_big;
    for (int kt = 0; kt < ntiles; ++kt) {
        const int buf = (ABL & 4) ? 0 : (kt & 1);
        if constexpr (PRE) vbig = q_big || (__builtin_amdgcn_readfirstlane(vbig_s[buf]) != 0);   // this tile only
        else vbig = vbig || (__builtin_amdgcn_readfirstlane(vbig_s[buf]) != 0);  // from the first flagged tile on
        {   // unconditional prefetch (the last tile re-reads itself): a load under a condition is waited for on the spot
            const int nxt = min(kt + 1, ntiles - 1);
            load_kv(nxt);
        }
        // The 64-key tile is consumed in two halves of 32 keys (QK^T -> softmax -> PV each), which keeps
        // the live score registers at 8 per query tile.  `fast`: both products on the fp16 matrix cores; decided once
        // per tile, so that the body is one long basic block in which the compiler can interleave the matrix
        // instructions of one query tile with the softmax arithmetic of the other.
        auto tile_body = [&](auto fast_tag) {
        constexpr bool FAST = decltype(fast_tag)::value;
#pragma unroll
        for (int hf = 0; hf < 2 * KT64; ++hf) {
            // ---- S^T tiles: s[t][j][r] = score(query q0+16t+lq, key 32hf + 16j + 4g + r) - reference
            f32x4 s[QT][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (QKH && FAST) {
                    const f16x8 ka = *reinterpret_cast<const f16x8*>(&Kh[buf][((2 * hf + j) * 16 + lq) * KHROW + 8 * g]);
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        f32x4 a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb1[t], negm[t], 0, 0, 0);
                        s[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb2[t], a, 0, 0, 0);
                    }
                    continue;
                }
                float4 kf;
                if constexpr (PRE) {
                    if (grp_s[buf][(2 * hf + j) * 2] != 0) {   // the producer left this group's fp32 values
                        kf = *reinterpret_cast<const float4*>(pre.k32 + ((size_t)bh * L + kt * TK + (2 * hf + j) * 16 + lq) * 16 + 4 * g);
                    } else {                                    // the sum of the halves
                        const f16x8 kk = *reinterpret_cast<const f16x8*>(&Kh[buf][((2 * hf + j) * 16 + lq) * KHROW + 8 * g]);
                        kf = make_float4((float)kk[0] + (float)kk[4] * 0.00048828125f, (float)kk[1] + (float)kk[5] * 0.00048828125f,
                                         (float)kk[2] + (float)kk[6] * 0.00048828125f, (float)kk[3] + (float)kk[7] * 0.00048828125f);
                    }
                } else {
                    kf = F32_TILES
                        ? *reinterpret_cast<const float4*>(&Ks[buf][((2 * hf + j) * 16 + lq) * KROW + 4 * g])
                        : *reinterpret_cast<const float4*>(Kb + (size_t)(kt * TK + (2 * hf + j) * 16 + lq) * RS + 4 * g);
                }
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    f32x4 a = negm[t];
                    const float4 qt = F32_TILES ? qf[t] : load_qf(t);
                    if (!(ABL & 8)) {
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.x, qt.x, negm[t], 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.y, qt.y, a, 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.z, qt.z, a, 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.w, qt.w, a, 0, 0, 0);
                    } else {
                        a[0] += kf.x * qt.x; a[1] += kf.y; a[2] += kf.z; a[3] += kf.w;
                    }
                    s[t][j] = a;
                }
            }
            // ---- online softmax (per query = per lane & 15; the four lanes g = 0..3 share a query)
            float mx[QT];
            const bool first = (kt == 0 && hf == 0);
            bool move = first;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float m0 = max3f(s[t][0][0], s[t][0][1], s[t][0][2]);
                const float m1 = max3f(s[t][0][3], s[t][1][0], s[t][1][1]);
                const float m2 = max3f(s[t][1][2], s[t][1][3], m0);
                mx[t] = fmaxf(m1, m2);  // lane-local maximum of (score - reference)
                move = move || (mx[t] > RESCALE);
            }
            if (__any(move)) {  // wave-uniform; first step, then only if a score runs away from the reference
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    float m = mx[t];
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));  // the four lanes that share a query agree on the shift
                    const float delta = first ? m : ((m > RESCALE) ? m : 0.f);
                    const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(-delta);
#pragma unroll
                    for (int r = 0; r < 4; ++r) negm[t][r] -= delta;
                    lrun[t] *= alpha;
#pragma unroll
                    for (int r = 0; r < 4; ++r) ot[t][r] *= alpha;
                    if (PVH) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) ot2[t][r] *= alpha;
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][j][r] -= delta;
                }
            }
#pragma unroll
            for (int t = 0; t < QT; ++t) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = (ABL & 1) ? s[t][j][0] * 0.5f : __builtin_amdgcn_exp2f(s[t][j][0]);
                    const float p1 = (ABL & 1) ? s[t][j][1] * 0.5f : __builtin_amdgcn_exp2f(s[t][j][1]);
                    const float p2 = (ABL & 1) ? s[t][j][2] * 0.5f : __builtin_amdgcn_exp2f(s[t][j][2]);
                    const float p3 = (ABL & 1) ? s[t][j][3] * 0.5f : __builtin_amdgcn_exp2f(s[t][j][3]);
                    s[t][j] = f32x4{p0, p1, p2, p3};
                    lrun[t] += f32x2{p0, p1};
                    lrun[t] += f32x2{p2, p3};
                }
            }
            // ---- O^T += V^T P^T : A = V^T, B = P (the S^T registers)
            if (PVH && FAST) {  // fp16 halves, 32 keys per product: lane (d, g) holds V[key 16j + 4g + r][d] in slot 4j + r
                const f16x8 vhi = *reinterpret_cast<const f16x8*>(&Vh[buf][0][hf][(lq * 4 + g) * 8]);
                const f16x8 vlo = *reinterpret_cast<const f16x8*>(&Vh[buf][1][hf][(lq * 4 + g) * 8]);
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    // P = hi + lo, hi rounded towards zero (P <= 2^15 never overflows it): four instructions per pair
                    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
                    u32x4 ph, pl;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        unsigned h0, l0, h1, l1;
                        split_pair_f16(s[t][j][0], s[t][j][1], h0, l0);
                        split_pair_f16(s[t][j][2], s[t][j][3], h1, l1);
                        ph[2 * j] = h0; ph[2 * j + 1] = h1;
                        pl[2 * j] = l0; pl[2 * j + 1] = l1;
                    }
                    const f16x8 phi = __builtin_bit_cast(f16x8, ph), plo = __builtin_bit_cast(f16x8, pl);
                    if (!(ABL & 16)) {
                        ot2[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vlo, phi, ot2[t], 0, 0, 0);
                        ot[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vhi, plo, ot[t], 0, 0, 0);
                        ot[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vhi, phi, ot[t], 0, 0, 0);
                    } else {
                        ot[t][0] += (float)(vlo[0] * phi[1] + vhi[2] * plo[3] + phi[4] + plo[5] + phi[6] * plo[7]);
                    }
                }
            } else
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // fp32: lane (d, g) holds V[key 4g + r][d] for step r
                float vf[4];
                if constexpr (PRE) {
                    if (grp_s[buf][(2 * hf + j) * 2 + 1] != 0) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            vf[r] = pre.v32[((size_t)bh * L + kt * TK + (2 * hf + j) * 16 + 4 * g + r) * 16 + lq];
                    } else {
                        const f16x4 vh4 = *reinterpret_cast<const f16x4*>(&Vh[buf][0][hf][(lq * 4 + g) * 8 + 4 * j]);
                        const f16x4 vl4 = *reinterpret_cast<const f16x4*>(&Vh[buf][1][hf][(lq * 4 + g) * 8 + 4 * j]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) vf[r] = (float)vh4[r] + (float)vl4[r] * 0.00048828125f;
                    }
                } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    vf[r] = (ABL & 2) ? scale_log2e + (float)r
                          : F32_TILES ? Vs[buf][((2 * hf + j) * 16 + 4 * g + r) * KROW + lq]
                                      : Vb[(size_t)(kt * TK + (2 * hf + j) * 16 + 4 * g + r) * RS + lq];
                }
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (!(ABL & 16)) ot[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r], s[t][j][r], ot[t], 0, 0, 0);
                        else ot[t][r] += vf[r] * s[t][j][r];
                    }
            }
        }
        };
        if (PVH && !vbig) tile_body(std::true_type{});
        else tile_body(std::false_type{});
        if (!(ABL & 4)) {
            stage(buf ^ 1);
            __syncthreads();
        }
    }

    // ---- normalise and store: lane (q, g) holds O[q][4g + r], r = 0..3
    const int b = bh / heads, head = bh - b * heads;
    const int C = heads * 16;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float l = lrun[t][0] + lrun[t][1];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const float inv = 1.0f / l;
        if (PVH) {
#pragma unroll
            for (int r = 0; r < 4; ++r) ot[t][r] += ot2[t][r] * 0.00048828125f;
        }
        float4 o = make_float4(ot[t][0] * inv, ot[t][1] * inv, ot[t][2] * inv, ot[t][3] * inv);
        *reinterpret_cast<float4*>(O + ((size_t)b * L + q0 + t * 16 + lq) * C + head * 16 + 4 * g) = o;
        // the row's log-sum-exp in the exp2 domain (reference + log2 of the sum), kept for the backward kernels
        if (LSE2 != nullptr && g == 0) LSE2[(size_t)bh * L + q0 + t * 16 + lq] = log2f(l) - negm[t][0];
    }
}

// ------------------------------------------------------------------------------------------------
// k_flash_wide<DT>: the same flash scheme for head_dim = 16*DT (32 or 64: networks built with 2 heads or 1 head
// at the 64-channel levels) and L a multiple of 128.  Per 16-key x 16-query score tile it issues 4*DT QK^T and
// 4*DT PV matrix instructions for the same four exponentials per lane, so the softmax arithmetic weighs 1/DT of
// what it does at head_dim 16.  Operand mapping: MFMA step s of QK^T consumes d = (HD/4)*g + s from both K and Q
// (lane (row, g) reads HD/4 consecutive floats of its row); PV walks the DT 16-wide slices of V.
template <int DT, int QT>  // QT = 16-query tiles per wave (a workgroup owns 64*QT queries)
__global__ __launch_bounds__(256) void k_flash_wide(const float* __restrict__ Q, const float* __restrict__ K,
                                                    const float* __restrict__ V, float* __restrict__ O, int L,
                                                    int heads, int n_bh, float scale_log2e) {
    constexpr int HD = 16 * DT;
    constexpr int HQ = 4 * DT;       // floats of a row per lane in QK^T
    constexpr int ROW = HD + 4;      // padded LDS row
    constexpr int PER = KVT * HD / 4 / 256;  // float4 per thread and operand of a 64-key tile
    extern __shared__ __attribute__((aligned(16))) float fw_s[];
    float* Ks = fw_s;                        // [2][KVT * ROW]
    float* Vs = fw_s + 2 * KVT * ROW;        // [2][KVT * ROW]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nq = L / (4 * QT * 16);
    int bh, qblk;
    if (n_bh % 8 == 0) {  // all query blocks of one (image, head) on one XCD, as in k_flash_hd16
        const int id = blockIdx.x;
        bh = (id / (8 * nq)) * 8 + (id & 7);
        qblk = (id >> 3) % nq;
    } else {
        bh = blockIdx.x / nq;
        qblk = blockIdx.x - bh * nq;
    }
    const int q0 = qblk * (4 * QT * 16) + wave * (QT * 16);
    const int lq = lane & 15;
    const int g = lane >> 4;
    const float* Qb = Q + (size_t)bh * L * HD;
    const float* Kb = K + (size_t)bh * L * HD;
    const float* Vb = V + (size_t)bh * L * HD;

    float qf[QT][HQ];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(Qb + (size_t)(q0 + t * 16 + lq) * HD + HQ * g + 4 * j);
            qf[t][4 * j] = v.x * scale_log2e; qf[t][4 * j + 1] = v.y * scale_log2e;
            qf[t][4 * j + 2] = v.z * scale_log2e; qf[t][4 * j + 3] = v.w * scale_log2e;
        }
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    f32x4 ot[QT][DT], negm[QT];
    f32x2 lrun[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) ot[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        negm[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        lrun[t] = f32x2{0.f, 0.f};
    }
    // staging: thread owns float4 number tid + 256*i of the tile (row = idx / (HD/4), column quad = idx % (HD/4))
    float4 kreg[PER], vreg[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int idx = tid + 256 * i;
        kreg[i] = reinterpret_cast<const float4*>(Kb)[idx];
        vreg[i] = reinterpret_cast<const float4*>(Vb)[idx];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int idx = tid + 256 * i, r = idx / (HD / 4), c4 = (idx - r * (HD / 4)) * 4;
        *reinterpret_cast<float4*>(Ks + r * ROW + c4) = kreg[i];
        *reinterpret_cast<float4*>(Vs + r * ROW + c4) = vreg[i];
    }
    __syncthreads();

    const int ntiles = L / KVT;
    for (int kt = 0; kt < ntiles; ++kt) {
        const int buf = kt & 1;
        const float* Kt = Ks + buf * KVT * ROW;
        const float* Vt = Vs + buf * KVT * ROW;
        {
            const int nxt = min(kt + 1, ntiles - 1);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int idx = tid + 256 * i;
                kreg[i] = reinterpret_cast<const float4*>(Kb + (size_t)nxt * KVT * HD)[idx];
                vreg[i] = reinterpret_cast<const float4*>(Vb + (size_t)nxt * KVT * HD)[idx];
            }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            f32x4 s[QT][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float kf[HQ];
#pragma unroll
                for (int u = 0; u < DT; ++u) {
                    const float4 v = *reinterpret_cast<const float4*>(Kt + ((2 * hf + j) * 16 + lq) * ROW + HQ * g + 4 * u);
                    kf[4 * u] = v.x; kf[4 * u + 1] = v.y; kf[4 * u + 2] = v.z; kf[4 * u + 3] = v.w;
                }
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    f32x4 a = negm[t];
#pragma unroll
                    for (int u = 0; u < HQ; ++u) a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[u], qf[t][u], a, 0, 0, 0);
                    s[t][j] = a;
                }
            }
            float mx[QT];
            const bool first = (kt == 0 && hf == 0);
            bool move = first;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float m0 = max3f(s[t][0][0], s[t][0][1], s[t][0][2]);
                const float m1 = max3f(s[t][0][3], s[t][1][0], s[t][1][1]);
                const float m2 = max3f(s[t][1][2], s[t][1][3], m0);
                mx[t] = fmaxf(m1, m2);
                move = move || (mx[t] > RESCALE_LOG2);
            }
            if (__any(move)) {
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    float m = mx[t];
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));
                    const float delta = first ? m : ((m > RESCALE_LOG2) ? m : 0.f);
                    const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(-delta);
#pragma unroll
                    for (int r = 0; r < 4; ++r) negm[t][r] -= delta;
                    lrun[t] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) ot[t][dt][r] *= alpha;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][j][r] -= delta;
                }
            }
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = __builtin_amdgcn_exp2f(s[t][j][0]);
                    const float p1 = __builtin_amdgcn_exp2f(s[t][j][1]);
                    const float p2 = __builtin_amdgcn_exp2f(s[t][j][2]);
                    const float p3 = __builtin_amdgcn_exp2f(s[t][j][3]);
                    s[t][j] = f32x4{p0, p1, p2, p3};
                    lrun[t] += f32x2{p0, p1};
                    lrun[t] += f32x2{p2, p3};
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    float vf[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) vf[r] = Vt[((2 * hf + j) * 16 + 4 * g + r) * ROW + 16 * dt + lq];
#pragma unroll
                    for (int t = 0; t < QT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            ot[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r], s[t][j][r], ot[t][dt], 0, 0, 0);
                }
        }
        {
            float* Kn = Ks + (buf ^ 1) * KVT * ROW;
            float* Vn = Vs + (buf ^ 1) * KVT * ROW;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int idx = tid + 256 * i, r = idx / (HD / 4), c4 = (idx - r * (HD / 4)) * 4;
                *reinterpret_cast<float4*>(Kn + r * ROW + c4) = kreg[i];
                *reinterpret_cast<float4*>(Vn + r * ROW + c4) = vreg[i];
            }
            __syncthreads();
        }
    }
    const int b = bh / heads, head = bh - b * heads;
    const int C = heads * HD;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float l = lrun[t][0] + lrun[t][1];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const float inv = 1.0f / l;
        float* dst = O + ((size_t)b * L + q0 + t * 16 + lq) * C + head * HD + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<float4*>(dst + 16 * dt) =
                make_float4(ot[t][dt][0] * inv, ot[t][dt][1] * inv, ot[t][dt][2] * inv, ot[t][dt][3] * inv);
    }
}

template <int DT, int QT>
static hipError_t launch_flash_wide_qt(const float* q, const float* k, const float* v, float* out, int B, int heads, int L,
                                       hipStream_t stream) {
    constexpr int HD = 16 * DT;
    const size_t lds = (size_t)4 * KVT * (HD + 4) * sizeof(float);
    if (lds > 48 * 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_flash_wide<DT, QT>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const float scale_log2e = (1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
    DANRA_LAUNCH_KERNEL((k_flash_wide<DT, QT>), dim3((L / (64 * QT)) * B * heads), dim3(256), lds, stream, q, k, v, out, L,
                       heads, B * heads, scale_log2e);
    return hipGetLastError();
}
// L must be a multiple of 64.  Workgroups of 128 queries when that still gives every CU two of them, else 64.
template <int DT>
static hipError_t launch_flash_wide(const float* q, const float* k, const float* v, float* out, int B, int heads, int L,
                                    hipStream_t stream) {
    if (L % 128 == 0 && (long)(L / 128) * B * heads >= 512) return launch_flash_wide_qt<DT, 2>(q, k, v, out, B, heads, L, stream);
    return launch_flash_wide_qt<DT, 1>(q, k, v, out, B, heads, L, stream);
}

// Very short sequences (L <= 16 tokens: the deepest levels) with a wide head (any head_dim): one workgroup per
// (image, head), one wave per query.  A lane owns head_dim/64 strided columns: the L dot products are reduced across
// the wave, the softmax over the L scores is wave-uniform, and each lane forms its own output columns.
template <int NC, int ML>  // head_dim <= 64 * NC, L <= ML <= 16
__global__ __launch_bounds__(64 * ML) void k_attn_tiny(const float* __restrict__ Q, const float* __restrict__ K,
                                                    const float* __restrict__ V, float* __restrict__ O, int L,
                                                    int hd, int heads, float scale) {
    const int lane = threadIdx.x & 63, qi = threadIdx.x >> 6;
    const int bh = blockIdx.x;
    if (qi >= L) return;
    const float* Qr = Q + ((size_t)bh * L + qi) * hd;
    const float* Kb = K + (size_t)bh * L * hd;
    const float* Vb = V + (size_t)bh * L * hd;
    // Every load is unconditional (indices clamped, contributions zeroed instead): a load under a condition becomes
    // a branch with its own wait, and the ~100 loads of a wave would then be served one after the other.
    int dcol[NC];
    float qv[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        dcol[c] = min(lane + 64 * c, hd - 1);
        const float v = Qr[dcol[c]];
        qv[c] = (lane + 64 * c < hd) ? v : 0.f;
    }
    float sc[ML];
#pragma unroll
    for (int j = 0; j < ML; ++j) {
        const float* krow = Kb + (size_t)min(j, L - 1) * hd;
        float a = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) a = fmaf(qv[c], krow[dcol[c]], a);
        sc[j] = a;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < ML; ++j) {
        float a = sc[j];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) a += __shfl_xor(a, off);
        sc[j] = (j < L) ? a * scale : -INFINITY;
        mx = fmaxf(mx, sc[j]);
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < ML; ++j) {
        sc[j] = (j < L) ? expf(sc[j] - mx) : 0.f;
        sum += sc[j];
    }
    const float inv = 1.0f / sum;
    const int b = bh / heads, head = bh - b * heads;
    float* dst = O + ((size_t)b * L + qi) * (heads * hd) + head * hd;
    float o[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = 0.f;
#pragma unroll
    for (int j = 0; j < ML; ++j) {  // sc[j] is 0 for j >= L
        const float* vrow = Vb + (size_t)min(j, L - 1) * hd;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] = fmaf(sc[j], vrow[dcol[c]], o[c]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
        if (lane + 64 * c < hd) dst[lane + 64 * c] = o[c] * inv;
}

// Register-resident attention for short sequences (L <= 256) and head_dim = 16*DT: one wave per
// (batch, head, 16-query tile), no LDS and no barrier.  Same operand trick as k_flash_hd16: the scores
// are formed transposed (S^T = K Q^T on v_mfma_f32_16x16x4_f32, keys as rows, queries as columns), so a
// lane's four accumulator registers of a key tile are exactly the B operand of O^T = V^T P^T.  All NKT
// score tiles stay in registers, which makes the softmax an exact two-pass one (no running rescale).
// Lane (c = lane & 15, kg = lane >> 4) holds the contiguous head_dim/4 slice kg of Q row c and of K row c:
// MFMA step s consumes d = (head_dim/4)*kg + s from both operands, and the 16 x head_dim K tile is read
// with fully coalesced 16-byte loads straight from memory.  Keys >= L are masked to -inf (their loads are
// clamped), queries >= L are computed and not stored.

template <int DT, int NKT>
__global__ __launch_bounds__(256) void k_attn_reg(const float* __restrict__ Q, const float* __restrict__ K,
                                                  const float* __restrict__ V, float* __restrict__ O, int L,
                                                  int heads, int n_bh, float scale_log2e) {
    constexpr int HD = 16 * DT;
    constexpr int HQ = 4 * DT;  // floats of a row per lane
    const int lane = threadIdx.x & 63;
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int qtiles = (L + 15) >> 4;
    const int task = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    const int bh = task / qtiles;
    const int qt = task - bh * qtiles;
    if (bh >= n_bh) return;
    const float* Qb = Q + (size_t)bh * L * HD;
    const float* Kb = K + (size_t)bh * L * HD;
    const float* Vb = V + (size_t)bh * L * HD;
    const int q0 = qt * 16;

    float q[HQ];
    {
        const float* src = Qb + (size_t)min(q0 + c, L - 1) * HD + HQ * kg;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(src + 4 * j);
            q[4 * j] = v.x * scale_log2e; q[4 * j + 1] = v.y * scale_log2e;
            q[4 * j + 2] = v.z * scale_log2e; q[4 * j + 3] = v.w * scale_log2e;
        }
    }
    // ---- S^T tiles: st[kt][r] = score(query q0 + c, key 16*kt + 4*kg + r), in the log2 domain
    f32x4 st[NKT];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
        float kf[HQ];
        const float* src = Kb + (size_t)min(kt * 16 + c, L - 1) * HD + HQ * kg;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(src + 4 * j);
            kf[4 * j] = v.x; kf[4 * j + 1] = v.y; kf[4 * j + 2] = v.z; kf[4 * j + 3] = v.w;
        }
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < HQ; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[s], q[s], acc, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (kt * 16 + 4 * kg + r >= L) acc[r] = -INFINITY;
            mx = fmaxf(mx, acc[r]);
        }
        st[kt] = acc;
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float e = __builtin_amdgcn_exp2f(st[kt][r] - mx);
            st[kt][r] = e;
            sum += e;
        }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    // ---- O^T tiles: ot[dt][r] = out(query q0 + c, d = 16*dt + 4*kg + r)
    f32x4 ot[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ot[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float* vrow = Vb + (size_t)min(kt * 16 + 4 * kg + r, L - 1) * HD + c;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                ot[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vrow[16 * dt], st[kt][r], ot[dt], 0, 0, 0);
        }
    if (q0 + c < L) {
        const float inv = 1.0f / sum;
        const int b = bh / heads, head = bh - b * heads;
        float* dst = O + ((size_t)b * L + q0 + c) * (heads * HD) + head * HD + 4 * kg;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<float4*>(dst + 16 * dt) =
                make_float4(ot[dt][0] * inv, ot[dt][1] * inv, ot[dt][2] * inv, ot[dt][3] * inv);
    }
}

template <int DT>
static hipError_t launch_attn_reg(const float* q, const float* k, const float* v, float* out, int B, int heads, int L,
                                  hipStream_t stream) {
    const int n_bh = B * heads;
    const int tasks = n_bh * ((L + 15) / 16);
    const int wpb = tasks > 1024 ? 4 : 1;  // one wave per workgroup spreads few tasks over all CUs
    const dim3 grid((tasks + wpb - 1) / wpb), block(64 * wpb);
    const float scale_log2e = (1.0f / sqrtf(16.0f * DT)) * 1.4426950408889634f;
    if (L <= 16) hipLaunchKernelGGL((k_attn_reg<DT, 1>), grid, block, 0, stream, q, k, v, out, L, heads, n_bh, scale_log2e);
    else if (L <= 64) hipLaunchKernelGGL((k_attn_reg<DT, 4>), grid, block, 0, stream, q, k, v, out, L, heads, n_bh, scale_log2e);
    else hipLaunchKernelGGL((k_attn_reg<DT, 16>), grid, block, 0, stream, q, k, v, out, L, heads, n_bh, scale_log2e);
    return hipGetLastError();
}

// Generic fallback for any other shape (any L, head_dim <= 64*NC <= 512): grid (B*heads, ceil(L/32)); a workgroup
// owns 32 queries (8 per wave, their running maximum / sum / output in registers) and walks the keys in chunks of
// AS_KC staged in LDS, with the usual online-softmax rescaling between chunks.  Plain VALU arithmetic: correctness
// first, this path is not on any benchmarked configuration.
constexpr int AS_QPW = 8;   // queries per wave
template <int NC, int AS_KC>  // NC: output columns per lane (head_dim <= 64*NC); AS_KC: keys per chunk (<= 64)
__global__ __launch_bounds__(256) void k_attn_small(const float* __restrict__ Q, const float* __restrict__ K,
                                                    const float* __restrict__ V, float* __restrict__ O, int L,
                                                    int hd, int heads, float scale) {
    extern __shared__ __attribute__((aligned(16))) float sm[];
    const int kst = hd + 1;
    float* Ks = sm;                          // [AS_KC][hd+1]
    float* Vs = Ks + AS_KC * kst;            // [AS_KC][hd]
    float* Ps = Vs + AS_KC * hd;             // [4 waves][AS_KC]
    float* Qs = Ps + 4 * AS_KC;              // [4 waves][AS_QPW][hd]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x;
    const float* Qb = Q + (size_t)bh * L * hd;
    const float* Kb = K + (size_t)bh * L * hd;
    const float* Vb = V + (size_t)bh * L * hd;
    const int q0 = blockIdx.y * (4 * AS_QPW) + wave * AS_QPW;
    float* Pw = Ps + wave * AS_KC;
    float* Qw = Qs + wave * AS_QPW * hd;
    for (int i = lane; i < AS_QPW * hd; i += 64) {
        const int qi = i / hd, d = i - qi * hd;
        Qw[i] = Qb[(size_t)min(q0 + qi, L - 1) * hd + d] * scale;
    }
    float m[AS_QPW], l[AS_QPW], o[AS_QPW][NC];  // lane holds output columns lane + 64*c
#pragma unroll
    for (int qi = 0; qi < AS_QPW; ++qi) {
        m[qi] = -INFINITY; l[qi] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[qi][c] = 0.f;
    }
    for (int k0 = 0; k0 < L; k0 += AS_KC) {
        const int nk = min(AS_KC, L - k0);
        __syncthreads();  // the previous chunk has been consumed (and Qw is written, the first time round)
        for (int i = tid; i < nk * hd; i += 256) {
            const int r = i / hd, c = i - r * hd;
            Ks[r * kst + c] = Kb[(size_t)k0 * hd + i];
            Vs[i] = Vb[(size_t)k0 * hd + i];
        }
        __syncthreads();
#pragma unroll
        for (int qi = 0; qi < AS_QPW; ++qi) {
            float sc = -INFINITY;
            if (lane < nk) {
                sc = 0.f;
                for (int d = 0; d < hd; ++d) sc = fmaf(Qw[qi * hd + d], Ks[lane * kst + d], sc);
            }
            float cm = sc;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) cm = fmaxf(cm, __shfl_xor(cm, off));
            const float mn = fmaxf(m[qi], cm);
            const float alpha = expf(m[qi] - mn);  // 0 the first time round (m = -inf)
            const float pe = (lane < nk) ? expf(sc - mn) : 0.f;
            float ps = pe;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) ps += __shfl_xor(ps, off);
            l[qi] = l[qi] * alpha + ps;
            m[qi] = mn;
            if (lane < AS_KC) Pw[lane] = pe;
            __builtin_amdgcn_wave_barrier();
            float a[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) a[c] = 0.f;
            for (int j = 0; j < nk; ++j) {
                const float pj = Pw[j];
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if (lane + 64 * c < hd) a[c] = fmaf(pj, Vs[j * hd + lane + 64 * c], a[c]);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) o[qi][c] = o[qi][c] * alpha + a[c];
            __builtin_amdgcn_wave_barrier();
        }
    }
    const int b = bh / heads, head = bh - b * heads;
    const int C = heads * hd;
#pragma unroll
    for (int qi = 0; qi < AS_QPW; ++qi) {
        const int q = q0 + qi;
        if (q >= L) continue;
        const float inv = 1.0f / l[qi];
        float* dst = O + ((size_t)b * L + q) * C + head * hd;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < hd) dst[lane + 64 * c] = o[qi][c] * inv;
    }
}

template <int NC, int KC>
static hipError_t launch_attn_small(const float* q, const float* k, const float* v, float* out, int B, int heads, int L,
                                    int hd, hipStream_t stream) {
    const size_t lds = ((size_t)KC * (hd + 1) + (size_t)KC * hd + 4 * KC + 4 * AS_QPW * (size_t)hd) * sizeof(float);
    if (lds > 48 * 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_small<NC, KC>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    dim3 grid(B * heads, (L + 4 * AS_QPW - 1) / (4 * AS_QPW));
    const float scale = 1.0f / sqrtf((float)hd);
    hipLaunchKernelGGL((k_attn_small<NC, KC>), grid, dim3(256), lds, stream, q, k, v, out, L, hd, heads, scale);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// A whole attention block up to its head outputs, for the short sequences of the deep levels: LayerNorm, the QKV
// projection of ONE head and that head's attention in one kernel, one workgroup per (image, head).  The three
// launches this replaces (LayerNorm-fused QKV GEMM, its head-split store, the register-resident attention) spend
// most of their 16-24 us in launch, fill and drain; here q, k and v of the head never leave LDS.
//   X    [B][L][C] tokens (the block's input, NHWC map)
//   Wf   in_proj [3C][C] with the LayerNorm affine folded in, split in fp16 halves at pack time (after a power-of-two
//        scale 1 / wscale) and laid out in FRAGMENT ORDER (launch_split_to_frag16): per 16-row tile and 32-deep step
//        the 64 lanes' 16-byte hi fragments, then their lo fragments, so that a fragment load of a wave is one
//        contiguous kilobyte (rows that lie a power of two apart would all fall on the same few memory channels);
//        row p*C + head*HD + d, p = q/k/v;  bin [3C] its bias
//   O    [B][L][C] head outputs, head h in columns h*HD .. (the operand of the output projection)
// Projection: a split-operand product like k_igemm's (W x ~ Wh xh + Wh xl + Wl xh on v_mfma_f32_16x16x32_f16, fp32
// accumulation): the waves normalise the token tiles, split them in fp16 halves and leave them in LDS; wave w of NW
// then owns column tiles w, w + NW, ... for every token tile, so each weight row is read from memory by one wave only, as
// 16-byte fragment loads that are issued before the tokens are touched (one trip to memory covers both).  Weights
// are the A operand, so a lane ends up with four consecutive output columns of one token (16-byte LDS stores).
// The normalised tokens are O(1) by construction (|x| < sqrt(C)), inside the range where the split keeps 22 bits; a
// row whose variance is far below the LayerNorm's epsilon is kept to an absolute 2^-25, which is what fp32 keeps of
// it next to the bias.  The attention part is k_attn_reg reading LDS: one wave per 16-query tile, scores in
// registers, exact two-pass softmax, fp32 matrix instructions.
template <int NT, int C, int HD, int NW>
__global__ __launch_bounds__(64 * NW) void k_attn_block_small(const float* __restrict__ X, const _Float16* __restrict__ Wf,
                                                          float wscale, const float* __restrict__ bin,
                                                          float* __restrict__ O, int heads, float scale_log2e) {
    constexpr int L = 16 * NT;
    constexpr int N3 = 3 * HD;
    constexpr int NTILES = N3 / 16;   // 16-column tiles of [q | k | v]
    constexpr int LDQ = N3 + 4;       // LDS row pitch in floats
    constexpr int DT = HD / 16;
    constexpr int HQ = HD / 4;
    constexpr int KS = C / 32;        // 32-deep steps of the projection
    constexpr int XP = 2 * C + 8;     // halves per token row in LDS: [C hi | C lo] + 16 bytes (rows land on different banks)
    constexpr int NIT = (NTILES + NW - 1) / NW;  // column tiles per wave
    constexpr int RING = NIT < (16 / KS > 1 ? 16 / KS : 1) ? NIT : (16 / KS > 1 ? 16 / KS : 1);  // weight tiles in flight per wave (8 * KS registers each)
    static_assert(NT <= NW && (NW == 4 || NW == 8), "one wave per token tile");
    static_assert(HD % 16 == 0 && C % 64 == 0, "tile sizes");
    __shared__ __attribute__((aligned(16))) float qkv[L * LDQ];
    __shared__ __attribute__((aligned(16))) _Float16 xs[L * XP];
    const int b = blockIdx.x / heads, head = blockIdx.x - b * heads;
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & (NW - 1);
    const int c = lane & 15, kg = lane >> 4;

    // ---- weights of this wave's first column tiles: loads only (tiles past the end re-read the last one, so that no
    // load sits behind a branch)
    auto wtile = [&](int nt) {  // halves; this lane's 16 bytes of column tile nt's first fragment
        const int n0 = min(nt, NTILES - 1) * 16;
        const int part = n0 / HD;
        const int T = (part * C + head * HD + (n0 - part * HD)) >> 4;  // 16-row tile of the whole [3C][C] matrix
        return Wf + (size_t)T * (KS * 1024) + lane * 8;
    };
    f16x8 wh[RING][KS], wl[RING][KS];
#pragma unroll
    for (int it = 0; it < RING; ++it) {
        const _Float16* wr = wtile(wave + NW * it);
#pragma unroll
        for (int s2 = 0; s2 < KS; ++s2) {
            wh[it][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024);
            wl[it][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024 + 512);
        }
    }
    __builtin_amdgcn_sched_barrier(0);  // (the scheduler would sink these loads to their uses to save registers)

    // ---- token tile `wave`: LayerNorm in registers (a row is spread over the four kg lanes of column c), split, to LDS.
    // Rows of more than 256 channels go through the registers in chunks of 128: mean and centred sum of squares per
    // chunk, combined by the pairwise update (equal chunk sizes), then a second trip (to L1) for the values themselves.
    if (wave < NT) {
        constexpr int CH = KS <= 8 ? KS : 4;  // steps per chunk (wide rows: 128 channels at a time, the weights hold most registers)
        constexpr int NCH = KS / CH;
        static_assert(KS % CH == 0, "whole chunks");
        const float* xr = X + ((size_t)b * L + wave * 16 + c) * C + 8 * kg;
        _Float16* dst = xs + (wave * 16 + c) * XP + 8 * kg;
        float xf[8 * CH];  // xf[8 s + e] = x[row][32 (s + chunk * CH) + 8 kg + e]
        auto load_chunk = [&](int ch) {
#pragma unroll
            for (int s2 = 0; s2 < CH; ++s2) {
                const float4 v0 = *reinterpret_cast<const float4*>(xr + 32 * (ch * CH + s2));
                const float4 v1 = *reinterpret_cast<const float4*>(xr + 32 * (ch * CH + s2) + 4);
                xf[8 * s2] = v0.x; xf[8 * s2 + 1] = v0.y; xf[8 * s2 + 2] = v0.z; xf[8 * s2 + 3] = v0.w;
                xf[8 * s2 + 4] = v1.x; xf[8 * s2 + 5] = v1.y; xf[8 * s2 + 6] = v1.z; xf[8 * s2 + 7] = v1.w;
            }
        };
        float mean = 0.f, m2 = 0.f;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
            load_chunk(ch);
            float sm = 0.f;
#pragma unroll
            for (int k = 0; k < 8 * CH; ++k) sm += xf[k];
            sm += __shfl_xor(sm, 16);
            sm += __shfl_xor(sm, 32);
            const float cmean = sm / (float)(32 * CH);
            float q2 = 0.f;
#pragma unroll
            for (int k = 0; k < 8 * CH; ++k) {
                const float d = xf[k] - cmean;
                q2 += d * d;
            }
            q2 += __shfl_xor(q2, 16);
            q2 += __shfl_xor(q2, 32);
            if (ch == 0) {
                mean = cmean;
                m2 = q2;
            } else {  // ch chunks so far + this one
                const float d = cmean - mean;
                m2 += q2 + d * d * ((float)(ch * 32 * CH) / (float)(ch + 1));
                mean += d / (float)(ch + 1);
            }
        }
        const float rstd = 1.0f / sqrtf(m2 / (float)C + 1e-5f);
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
            if (NCH > 1) load_chunk(ch);
#pragma unroll
            for (int s2 = 0; s2 < CH; ++s2) {
                unsigned hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    split_pair_f16((xf[8 * s2 + 2 * e] - mean) * rstd, (xf[8 * s2 + 2 * e + 1] - mean) * rstd, hi[e], lo[e]);
                *reinterpret_cast<uint4*>(dst + 32 * (ch * CH + s2)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(dst + 32 * (ch * CH + s2) + C) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    __syncthreads();

    // ---- projection of this wave's column tiles
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
        const int nt = wave + NW * it;  // wave-uniform
        if (nt < NTILES) {
            // a tile lies inside one of q, k, v (16 divides HD)
            const int part = (nt * 16) / HD;
            const float4 bv = *reinterpret_cast<const float4*>(bin + (size_t)part * C + head * HD + (nt * 16 - part * HD) + 4 * kg);
            const float sc = part == 0 ? scale_log2e : 1.0f;  // the scores are formed in the log2 domain
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                const _Float16* xrow = xs + (tt * 16 + c) * XP + 8 * kg;
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s2 = 0; s2 < KS; ++s2) {
                    const f16x8 xh = *reinterpret_cast<const f16x8*>(xrow + 32 * s2);
                    const f16x8 xl = *reinterpret_cast<const f16x8*>(xrow + 32 * s2 + C);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl[it % RING][s2], xh, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[it % RING][s2], xl, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[it % RING][s2], xh, acc, 0, 0, 0);
                }
                // acc[r] = out[token tt*16 + c][column nt*16 + 4 kg + r] * (1 / wscale)
                *reinterpret_cast<float4*>(qkv + (tt * 16 + c) * LDQ + nt * 16 + 4 * kg) =
                    make_float4((acc[0] * wscale + bv.x) * sc, (acc[1] * wscale + bv.y) * sc, (acc[2] * wscale + bv.z) * sc,
                                (acc[3] * wscale + bv.w) * sc);
            }
        }
        if (it + RING < NIT) {  // this tile's registers take the tile RING further on
            __builtin_amdgcn_sched_barrier(0);  // (... once the products above have read them: no second register set)
            const _Float16* wr = wtile(nt + NW * RING);
#pragma unroll
            for (int s2 = 0; s2 < KS; ++s2) {
                wh[it % RING][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024);
                wl[it % RING][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024 + 512);
            }
        }
    }
    __syncthreads();
    if (wave >= NT) return;

    // ---- attention of query tile `wave` (see k_attn_reg for the operand layout)
    const int q0 = wave * 16;
    float q[HQ];
    {
        const float* src = qkv + (q0 + c) * LDQ + HQ * kg;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(src + 4 * j);
            q[4 * j] = v.x; q[4 * j + 1] = v.y; q[4 * j + 2] = v.z; q[4 * j + 3] = v.w;
        }
    }
    f32x4 st[NT];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
        float kf[HQ];
        const float* src = qkv + (kt * 16 + c) * LDQ + HD + HQ * kg;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(src + 4 * j);
            kf[4 * j] = v.x; kf[4 * j + 1] = v.y; kf[4 * j + 2] = v.z; kf[4 * j + 3] = v.w;
        }
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s2 = 0; s2 < HQ; ++s2) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[s2], q[s2], acc, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[r]);
        st[kt] = acc;
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float e = __builtin_amdgcn_exp2f(st[kt][r] - mx);
            st[kt][r] = e;
            sum += e;
        }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    f32x4 ot[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ot[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float* vrow = qkv + (kt * 16 + 4 * kg + r) * LDQ + 2 * HD + c;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                ot[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vrow[16 * dt], st[kt][r], ot[dt], 0, 0, 0);
        }
    const float inv = 1.0f / sum;
    float* dst = O + ((size_t)b * L + q0 + c) * C + head * HD + 4 * kg;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4*>(dst + 16 * dt) = make_float4(ot[dt][0] * inv, ot[dt][1] * inv, ot[dt][2] * inv, ot[dt][3] * inv);
}

// The shapes the fused block kernel is built for: 64 tokens x 128 channels and 16 tokens x 256 channels with four heads -
// the 8x8 and 4x4 levels of a 64x64 input.  (A form for 4 tokens x 512 channels - four images per workgroup, the scores
// between tokens of different images masked out - streamed 786 KB of weights through each of only B/4 x heads
// workgroups: 20.4 us at 64 images, against 10.0 + 4.8 us for k_proj_small's QKV projection, which spreads the same
// weights over 768 waves, and k_attn_reg.)
bool attn_block_small_supported(int B, int L, int C, int heads) {
    (void)B;
    return heads == 4 && ((L == 64 && C == 128) || (L == 16 && C == 256));
}

hipError_t launch_attn_block_small(const float* x, const float* w_in_frag, float wscale, const float* b_in, float* o,
                                   int B, int L, int C, int heads, hipStream_t stream) {
    if (!attn_block_small_supported(B, L, C, heads) || !w_in_frag) return hipErrorInvalidValue;
    const float scale_log2e = (1.0f / sqrtf((float)(C / heads))) * 1.4426950408889634f;
    const _Float16* wh = reinterpret_cast<const _Float16*>(w_in_frag);
    if (L == 64)
        DANRA_LAUNCH_KERNEL((k_attn_block_small<4, 128, 32, 4>), dim3(B * heads), dim3(256), 0, stream, x, wh, wscale, b_in, o, heads, scale_log2e);
    else
        DANRA_LAUNCH_KERNEL((k_attn_block_small<1, 256, 64, 8>), dim3(B * heads), dim3(512), 0, stream, x, wh, wscale, b_in, o, heads, scale_log2e);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// Output projection of the short-sequence attention blocks: out = act(A W^T + bias + res) for a few hundred to a few
// thousand rows and K = N = 128 / 256 / 512.  Through k_igemm such a product is two to eight chunks of work inside
// 7-8 us of launch, pipeline fill and epilogue (plus a split-K reduction kernel at 256 rows).  Here a wave owns one
// 16-row tile and NCT of the 16-column tiles: its weight fragments (split fp16 halves in fragment order, see
// launch_split_to_frag16) and its rows are all in flight in one trip to memory, the rows are split in registers,
// and the 3 * NCT * K / 32 matrix instructions run back to back; residual and bias arrive meanwhile.  No LDS, no
// barrier, one wave per workgroup (a few hundred waves spread over all CUs: 5.6-6.2 us where k_igemm took 7.5-8.2 and,
// with its split-K reduction at 256 rows, 11.7; four waves per workgroup on a quarter of the CUs took 9.2).  A wave whose rows leave the range of the split (a value >= 2^15 or non-finite, or nothing but values below
// 2^-8 that are not all zero) multiplies with fp32 instructions from the fp32 matrix instead.
//   A [M][K], Wf = W [N][K] split and in fragment order (scale 1 / wscale), W the fp32 matrix, res [M][N] or null
// With ct_W != 0 the product is a kernel-2 stride-2 transposed convolution on a ct_H x ct_W map (N = 4 x channels,
// column = (dy, dx, channel)) and the rows are stored pixel-shuffled: out [B][2 ct_H][2 ct_W][N / 4].  That pays at
// K = 64 only (bound by its 16 MB store); with K >= 128 the 1024 waves of such a product each fetch 32-64 KB of weights
// again and k_igemm is as fast or faster (9.2-11.0 against 8.2-10.5 us).
// Exact (erf) GELU, as torch.nn.GELU() evaluates it.
__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f)); }

template <int KS, int NCT, bool LN = false, bool QKV = false>
__global__ __launch_bounds__(64) void k_proj_small(const float* __restrict__ A, const _Float16* __restrict__ Wf,
                                                    const float* __restrict__ W, float wscale,
                                                    const float* __restrict__ bias, const float* __restrict__ res,
                                                    float* __restrict__ out, int M, int N, int act, int qkv_L,
                                                    int qkv_hd, int ct_H, int ct_W, float* __restrict__ pre_ks,
                                                    float* __restrict__ pre_vs, int* __restrict__ pre_flags) {
    constexpr int K = 32 * KS;
    const int lane = threadIdx.x & 63, c = lane & 15, kg = lane >> 4;
    const int task = blockIdx.x;  // one wave per workgroup: a few hundred tasks spread over all CUs
    const int groups = N / (16 * NCT);  // column groups per row tile
    const int rt = task / groups, cg = task - rt * groups;
    if (rt * 16 >= M) return;
    const int row = min(rt * 16 + c, M - 1);  // (rows past M are computed from row M - 1 and not stored)
    // ---- loads: the weight fragments of this wave's column tiles, then its rows
    f16x8 wh[NCT][KS], wl[NCT][KS];
#pragma unroll
    for (int t = 0; t < NCT; ++t) {
        const _Float16* wr = Wf + (size_t)(cg * NCT + t) * (KS * 1024) + lane * 8;
#pragma unroll
        for (int s2 = 0; s2 < KS; ++s2) {
            wh[t][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024);
            wl[t][s2] = *reinterpret_cast<const f16x8*>(wr + s2 * 1024 + 512);
        }
    }
    float xf[8 * KS];  // xf[8 s + e] = A[row][32 s + 8 kg + e]
    {
        const float* ar = A + (size_t)row * K + 8 * kg;
#pragma unroll
        for (int s2 = 0; s2 < KS; ++s2) {
            const float4 v0 = *reinterpret_cast<const float4*>(ar + 32 * s2);
            const float4 v1 = *reinterpret_cast<const float4*>(ar + 32 * s2 + 4);
            xf[8 * s2] = v0.x; xf[8 * s2 + 1] = v0.y; xf[8 * s2 + 2] = v0.z; xf[8 * s2 + 3] = v0.w;
            xf[8 * s2 + 4] = v1.x; xf[8 * s2 + 5] = v1.y; xf[8 * s2 + 6] = v1.z; xf[8 * s2 + 7] = v1.w;
        }
    }
    // what the epilogue adds: lane (c, kg) ends up with columns n0 + 4 kg .. + 3 of row rt * 16 + c
    float4 bv[NCT], rv[NCT];
#pragma unroll
    for (int t = 0; t < NCT; ++t) {
        const int n = (cg * NCT + t) * 16 + 4 * kg;
        bv[t] = bias ? *reinterpret_cast<const float4*>(bias + n) : make_float4(0.f, 0.f, 0.f, 0.f);
        rv[t] = res ? *reinterpret_cast<const float4*>(res + (size_t)row * N + n) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __builtin_amdgcn_sched_barrier(0);  // (keeps every load above ahead of the first use)
    if (LN) {  // LayerNorm over the K channels of a row (its four kg lanes); the affine part is folded into W and bias
        float sm = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < 8 * KS; ++k2) sm += xf[k2];
        sm += __shfl_xor(sm, 16);
        sm += __shfl_xor(sm, 32);
        const float mean = sm / (float)K;
        float q2 = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < 8 * KS; ++k2) {
            const float d = xf[k2] - mean;
            q2 += d * d;
        }
        q2 += __shfl_xor(q2, 16);
        q2 += __shfl_xor(q2, 32);
        const float rstd = 1.0f / sqrtf(q2 / (float)K + 1e-5f);
#pragma unroll
        for (int k2 = 0; k2 < 8 * KS; ++k2) xf[k2] = (xf[k2] - mean) * rstd;
    }
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8 * KS; ++k) amax = fmaxf(amax, fabsf(xf[k]));
    // (normalised rows are O(1) by construction: inside the split's range, see k_attn_block_small)
    const bool bad = !LN && (!(amax < 32768.f) || (amax > 0.f && amax < 0.00390625f));
    f32x4 acc[NCT];
#pragma unroll
    for (int t = 0; t < NCT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float scale = wscale;
    const bool pre_v = QKV && pre_flags != nullptr && cg == 2;   // this wave forms V for the pre-split form: untransposed
    if (__any(bad)) {  // rare: fp32 instructions, the fp32 matrix straight from memory (k = 32 s + 8 kg + e on both sides)
        scale = 1.0f;
        for (int t = 0; t < NCT; ++t) {
            const float* wr = W + (size_t)((cg * NCT + t) * 16 + c) * K + 8 * kg;
#pragma unroll
            for (int s2 = 0; s2 < KS; ++s2) {
                const float4 w0 = *reinterpret_cast<const float4*>(wr + 32 * s2);
                const float4 w1 = *reinterpret_cast<const float4*>(wr + 32 * s2 + 4);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w0.x, xf[8 * s2], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w0.y, xf[8 * s2 + 1], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w0.z, xf[8 * s2 + 2], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w0.w, xf[8 * s2 + 3], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w1.x, xf[8 * s2 + 4], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w1.y, xf[8 * s2 + 5], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w1.z, xf[8 * s2 + 6], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w1.w, xf[8 * s2 + 7], acc[t], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int s2 = 0; s2 < KS; ++s2) {
            unsigned hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) split_pair_f16(xf[8 * s2 + 2 * e], xf[8 * s2 + 2 * e + 1], hi[e], lo[e]);
            const f16x8 xh = __builtin_bit_cast(f16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            const f16x8 xl = __builtin_bit_cast(f16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
            for (int t = 0; t < NCT; ++t) {
                if (QKV && pre_v) {   // rows as the A operand: the same products, term by term, untransposed
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, wl[t][s2], acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, wh[t][s2], acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, wh[t][s2], acc[t], 0, 0, 0);
                    continue;
                }
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl[t][s2], xh, acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[t][s2], xl, acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[t][s2], xh, acc[t], 0, 0, 0);
            }
        }
    }
    if constexpr (QKV) {
        // ---- K and V of a head_dim-16 block left pre-split for the attention core (launch_presplit_kv describes the
        // form): this wave holds 16 keys of one image; its column tiles are the heads
        if (pre_flags != nullptr && cg >= 1) {
            typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
            typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
            const int row0 = rt * 16, b = row0 / qkv_L, l0 = row0 - b * qkv_L, heads = NCT;
#pragma unroll
            for (int t = 0; t < NCT; ++t) {
                const int bh = b * heads + t;
                int* fl = pre_flags + ((size_t)bh * (qkv_L >> 4) + (l0 >> 4)) * 2;
                if (cg == 1) {   // K: lane (key c, kg) holds columns 4 kg .. + 3
                    const float4 v = make_float4(acc[t][0] * scale + bv[t].x, acc[t][1] * scale + bv[t].y, acc[t][2] * scale + bv[t].z,
                                                 acc[t][3] * scale + bv[t].w);
                    unsigned h2[2], l2[2];
                    split_scaled_pair_f16(v.x, v.y, h2[0], l2[0]);
                    split_scaled_pair_f16(v.z, v.w, h2[1], l2[1]);
                    *reinterpret_cast<u32x4*>(pre_ks + ((size_t)bh * qkv_L + l0 + c) * 16 + 4 * kg) = u32x4{h2[0], h2[1], l2[0], l2[1]};
                    const float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
                    const bool flagged = __any(!(m < 32768.f)) != 0;
                    if (lane == 0) fl[0] = flagged ? 1 : 0;
                    if (flagged)   // (rare) the group's fp32 values
                        *reinterpret_cast<float4*>(out + (size_t)M * (N / 3) + ((size_t)bh * qkv_L + l0 + c) * 16 + 4 * kg) = v;
                } else {         // V, formed untransposed: lane (column c, kg) holds keys 4 kg .. + 3
                    const float bc = bias ? bias[(cg * NCT + t) * 16 + c] : 0.f;
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = acc[t][r] * scale + bc;
                    unsigned h2[2], l2[2];
                    split_scaled_pair_f16(v[0], v[1], h2[0], l2[0]);
                    split_scaled_pair_f16(v[2], v[3], h2[1], l2[1]);
                    // slot 4 j + r of group g = kg, column d = c, in the 32-key half this group of 16 belongs to
                    float* vt = pre_vs + ((size_t)bh * qkv_L + (l0 & ~63)) * 16;
                    const int half = (l0 >> 5) & 1, j = (l0 >> 4) & 1;
                    const int at = (half * 512 + (c * 4 + kg) * 8 + 4 * j) / 2;
                    *reinterpret_cast<u32x2*>(vt + at) = u32x2{h2[0], h2[1]};
                    *reinterpret_cast<u32x2*>(vt + 512 + at) = u32x2{l2[0], l2[1]};
                    const float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
                    const bool flagged = (__any(!(m < 32768.f)) != 0) || (__all(m < 0.0009765625f) != 0);
                    if (lane == 0) fl[1] = flagged ? 1 : 0;
                    if (flagged) {
                        float* v32 = out + 2 * (size_t)M * (N / 3) + ((size_t)bh * qkv_L + l0 + 4 * kg) * 16 + c;
#pragma unroll
                        for (int r = 0; r < 4; ++r) v32[r * 16] = v[r];
                    }
                }
            }
            return;
        }
    }
    if (rt * 16 + c >= M) return;
#pragma unroll
    for (int t = 0; t < NCT; ++t) {
        const int n = (cg * NCT + t) * 16 + 4 * kg;
        float4 v = make_float4(acc[t][0] * scale + bv[t].x, acc[t][1] * scale + bv[t].y, acc[t][2] * scale + bv[t].z,
                               acc[t][3] * scale + bv[t].w);
        if (res) { v.x += rv[t].x; v.y += rv[t].y; v.z += rv[t].z; v.w += rv[t].w; }
        if (act == ACT_RELU) { v.x = fmaxf(v.x, 0.f); v.y = fmaxf(v.y, 0.f); v.z = fmaxf(v.z, 0.f); v.w = fmaxf(v.w, 0.f); }
        else if (act == ACT_GELU) { v.x = gelu_erf(v.x); v.y = gelu_erf(v.y); v.z = gelu_erf(v.z); v.w = gelu_erf(v.w); }
        size_t at = (size_t)row * N + n;
        if (QKV) {  // columns [q | k | v] x heads x qkv_hd -> out[which][image * heads + head][token][qkv_hd]
            const int C = N / 3, which = n / C, cc = n - which * C, head = cc / qkv_hd, d = cc - head * qkv_hd;
            const int b = row / qkv_L, l = row - b * qkv_L;
            at = (size_t)which * M * C + (size_t)b * qkv_L * C + (size_t)head * qkv_L * qkv_hd + (size_t)l * qkv_hd + d;
        }
        if (!QKV && ct_W) {  // kernel-2 stride-2 transposed convolution: column (dy, dx, co) of coarse pixel (b, y, x)
            const int Cc = N >> 2, hw = ct_H * ct_W;
            const int q = n / Cc, co = n - q * Cc;
            const int b = row / hw, r = row - b * hw, y = r / ct_W, x = r - y * ct_W;
            at = (((size_t)b * 2 * ct_H + 2 * y + (q >> 1)) * 2 * ct_W + 2 * x + (q & 1)) * Cc + co;
        }
        *reinterpret_cast<float4*>(out + at) = v;
    }
}

// K = 64 / 128 / 256 / 512 with N a multiple of what a wave takes at that K, and few enough rows that k_igemm's tiles are
// not the better shape (8192; 65536 at K = 64, where k_igemm has a single chunk to work on and the product is bound by
// memory: 11.1 against 14.3 us for 65536 rows with a residual, 48 MB).
bool proj_small_supported(int M, int N, int K) {
    const int per_wave = K == 64 ? 64 : K == 128 ? 128 : K == 256 ? 64 : K == 512 ? 32 : 0;
    return per_wave && N >= per_wave && N % per_wave == 0 && M >= 1 && M <= (K == 64 ? 65536 : 8192);
}

static float* const no_f = nullptr;
static int* const no_i = nullptr;
hipError_t launch_proj_small(const float* a, const float* w_frag, const float* w, float wscale, const float* bias,
                             const float* res, float* out, int M, int N, int K, int act, hipStream_t stream, int ct_H,
                             int ct_W, bool layernorm) {
    if (!proj_small_supported(M, N, K) || !w_frag || !w) return hipErrorInvalidValue;
    if (ct_W && (res || N % 16 || ct_H <= 0 || M % (ct_H * ct_W))) return hipErrorInvalidValue;
    if (layernorm) {  // rows normalised over their K channels first (the affine part folded into W and bias)
        if (ct_W || K == 64) return hipErrorInvalidValue;
        const _Float16* wfl = reinterpret_cast<const _Float16*>(w_frag);
        const int rtl = (M + 15) / 16;
        if (K == 128)
            DANRA_LAUNCH_KERNEL((k_proj_small<4, 8, true>), dim3(rtl * (N / 128)), dim3(64), 0, stream, a, wfl, w, wscale, bias, res, out, M, N, act, 0, 0, 0, 0, no_f, no_f, no_i);
        else if (K == 256)
            DANRA_LAUNCH_KERNEL((k_proj_small<8, 4, true>), dim3(rtl * (N / 64)), dim3(64), 0, stream, a, wfl, w, wscale, bias, res, out, M, N, act, 0, 0, 0, 0, no_f, no_f, no_i);
        else
            DANRA_LAUNCH_KERNEL((k_proj_small<16, 2, true>), dim3(rtl * (N / 32)), dim3(64), 0, stream, a, wfl, w, wscale, bias, res, out, M, N, act, 0, 0, 0, 0, no_f, no_f, no_i);
        return hipGetLastError();
    }
    const _Float16* wf = reinterpret_cast<const _Float16*>(w_frag);
    const int rts = (M + 15) / 16;
    // NCT * KS = 32 fragment pairs per wave: 128 columns per wave at K = 128, 64 at 256, 32 at 512 (64 at K = 64)
    if (K == 64)
        DANRA_LAUNCH_KERNEL((k_proj_small<2, 4>), dim3(rts * (N / 64)), dim3(64), 0, stream, a, wf, w, wscale, bias, res, out, M, N, act, 0, 0, ct_H, ct_W, no_f, no_f, no_i);
    else if (K == 128)
        DANRA_LAUNCH_KERNEL((k_proj_small<4, 8>), dim3(rts * (N / 128)), dim3(64), 0, stream, a, wf, w, wscale, bias, res, out, M, N, act, 0, 0, ct_H, ct_W, no_f, no_f, no_i);
    else if (K == 256)
        DANRA_LAUNCH_KERNEL((k_proj_small<8, 4>), dim3(rts * (N / 64)), dim3(64), 0, stream, a, wf, w, wscale, bias, res, out, M, N, act, 0, 0, ct_H, ct_W, no_f, no_f, no_i);
    else
        DANRA_LAUNCH_KERNEL((k_proj_small<16, 2>), dim3(rts * (N / 32)), dim3(64), 0, stream, a, wf, w, wscale, bias, res, out, M, N, act, 0, 0, ct_H, ct_W, no_f, no_f, no_i);
    return hipGetLastError();
}

// The LayerNorm-fused QKV projection of an attention block on few rows through the same kernel: a wave normalises its 16
// tokens in registers, forms 64 / 128 / 64 / 32 of the 3 C columns (C = 64 / 128 / 256 / 512) and stores them head-split,
// qkv[which][image * heads + head][token][head_dim].
bool qkv_small_supported(int M, int C, int L, int hd) {
    // (at 65536 tokens of 64 channels the row-stationary k_gemm_k64, which stages the weights once per workgroup, is the
    // faster one: 18-20 against 25.5 us)
    const int max_rows = C == 64 ? 16384 : 8192;
    return (C == 64 || C == 128 || C == 256 || C == 512) && M >= 1 && M <= max_rows && hd % 4 == 0 && C % hd == 0 && L >= 1 &&
           M % L == 0;
}
bool qkv_small_presplits(int M, int C, int L, int hd) { return qkv_small_supported(M, C, L, hd) && C == 64 && hd == 16 && L % 64 == 0; }
hipError_t launch_qkv_small(const float* x, const float* w_frag, const float* w, float wscale, const float* bias, float* qkv,
                            int M, int C, int L, int hd, hipStream_t stream, float* pre_ks, float* pre_vs, int* pre_flags) {
    if (!qkv_small_supported(M, C, L, hd) || !w_frag || !w) return hipErrorInvalidValue;
    if ((pre_ks || pre_vs || pre_flags) && !(pre_ks && pre_vs && pre_flags && qkv_small_presplits(M, C, L, hd))) return hipErrorInvalidValue;
    const _Float16* wf = reinterpret_cast<const _Float16*>(w_frag);
    const int rts = (M + 15) / 16;
    const float* none = nullptr;
    if (C == 64)  // three waves per 16 tokens (q, k, v; each normalises the rows again): 64 registers instead of 172, 9.2 against 9.6 us
        DANRA_LAUNCH_KERNEL((k_proj_small<2, 4, true, true>), dim3(rts * 3), dim3(64), 0, stream, x, wf, w, wscale, bias, none, qkv, M, 3 * C, 0, L, hd, 0, 0, pre_ks, pre_vs, pre_flags);
    else if (C == 128)
        DANRA_LAUNCH_KERNEL((k_proj_small<4, 8, true, true>), dim3(rts * 3), dim3(64), 0, stream, x, wf, w, wscale, bias, none, qkv, M, 3 * C, 0, L, hd, 0, 0, no_f, no_f, no_i);
    else if (C == 256)
        DANRA_LAUNCH_KERNEL((k_proj_small<8, 4, true, true>), dim3(rts * 12), dim3(64), 0, stream, x, wf, w, wscale, bias, none, qkv, M, 3 * C, 0, L, hd, 0, 0, no_f, no_f, no_i);
    else
        DANRA_LAUNCH_KERNEL((k_proj_small<16, 2, true, true>), dim3(rts * 48), dim3(64), 0, stream, x, wf, w, wscale, bias, none, qkv, M, 3 * C, 0, L, hd, 0, 0, no_f, no_f, no_i);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// K and V of the head_dim-16 core [B*heads][L][16] in the pre-split form k_flash_hd16<PRE> reads (what the network's QKV
// projections write directly): one workgroup per (image, head, 64-key tile).
//   ks: per key 64 bytes, four groups of [4 halves hi | 4 halves lo'] (columns 4g .. 4g + 3), x = hi + 2^-11 lo'
//   vs: per tile [hi, lo'][32-key half][d][g][8 halves], slot 4j + r <-> key 16 j + 4 g + r of the half
//   flags: per 16 keys [K, V]: 1 where the group leaves the range of the split (a value of 2^15 or more or non-finite; for
//          V also nothing of 2^-10 or more)

__global__ __launch_bounds__(256) void k_presplit_kv(const float* __restrict__ K, const float* __restrict__ V,
                                                     float* __restrict__ ks, float* __restrict__ vs, int* __restrict__ flags,
                                                     int L) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const int tid = threadIdx.x, wave = tid >> 6;
    const int tiles = L / 64;
    const int bh = blockIdx.x / tiles, tile = blockIdx.x - bh * tiles;
    {   // K: thread = (key, column group); a wave = one group of 16 keys
        const int key = tile * 64 + (tid >> 2), g = tid & 3;
        const float4 k = *reinterpret_cast<const float4*>(K + ((size_t)bh * L + key) * 16 + 4 * g);
        unsigned h[2], l[2];
        split_scaled_pair_f16(k.x, k.y, h[0], l[0]);
        split_scaled_pair_f16(k.z, k.w, h[1], l[1]);
        *reinterpret_cast<u32x4*>(ks + ((size_t)bh * L + key) * 16 + 4 * g) = u32x4{h[0], h[1], l[0], l[1]};
        const float kmax = fmaxf(fmaxf(fabsf(k.x), fabsf(k.y)), fmaxf(fabsf(k.z), fabsf(k.w)));
        const bool bad = __any(!(kmax < 32768.f)) != 0;
        if ((tid & 63) == 0) flags[((size_t)bh * (L / 16) + 4 * tile + wave) * 2] = bad ? 1 : 0;
    }
    if (tid < 128) {   // V: thread = (32-key half, d, g); a wave = one half = two groups of 16 keys
        const int half = tid >> 6, d = (tid >> 2) & 15, g = tid & 3;
        float v[8];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[4 * j + r] = V[((size_t)bh * L + tile * 64 + half * 32 + 16 * j + 4 * g + r) * 16 + d];
        unsigned h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_scaled_pair_f16(v[2 * e], v[2 * e + 1], h[e], l[e]);
        float* base = vs + ((size_t)bh * L + tile * 64) * 16;             // this tile's 4 KB
        const int at = (half * 512 + (d * 4 + g) * 8) / 2;                // floats; hi block, then lo (2 x 512 halves further)
        *reinterpret_cast<u32x4*>(base + at) = u32x4{h[0], h[1], h[2], h[3]};
        *reinterpret_cast<u32x4*>(base + 512 + at) = u32x4{l[0], l[1], l[2], l[3]};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float m = fmaxf(fmaxf(fabsf(v[4 * j]), fabsf(v[4 * j + 1])), fmaxf(fabsf(v[4 * j + 2]), fabsf(v[4 * j + 3])));
            const bool bad = (__any(!(m < 32768.f)) != 0) || (__all(m < 0.0009765625f) != 0);
            if ((tid & 63) == 0) flags[((size_t)bh * (L / 16) + 4 * tile + 2 * half + j) * 2 + 1] = bad ? 1 : 0;
        }
    }
}

hipError_t launch_presplit_kv(const float* k, const float* v, float* ks, float* vs, int* flags, int n_bh, int L,
                              hipStream_t stream) {
    if (L % 64 || n_bh <= 0) return hipErrorInvalidValue;
    DANRA_LAUNCH_KERNEL(k_presplit_kv, dim3(n_bh * (L / 64)), dim3(256), 0, stream, k, v, ks, vs, flags, L);
    return hipGetLastError();
}

// The head_dim-16 core on pre-split K and V (see k_flash_hd16 PRE).  k32 / v32: the fp32 values, read only for the groups
// of 16 keys whose flag is set.
hipError_t launch_attention_hd16_pre(const float* q, const float* ks, const float* vs, const float* k32, const float* v32,
                                     const int* flags, float* out, int B, int heads, int L, hipStream_t stream) {
    if (L % 128 != 0 || !flags) return hipErrorInvalidValue;
    const float scale_log2e = 0.25f * 1.4426950408889634f;
    dim3 grid((L / 128) * B * heads);
    const FlashPre pre{k32, v32, flags};
    float* no_lse = nullptr;
    DANRA_LAUNCH_KERNEL((k_flash_hd16<2, 0, true, true, 1, true>), grid, dim3(256), 0, stream, q, ks, vs, out, no_lse, L, heads,
                       B * heads, scale_log2e, pre, QkvLayout{});
    return hipGetLastError();
}

static int g_hd16_fp32_products = 0;
void set_attention_hd16_fp32_products(int on) { g_hd16_fp32_products = on ? 1 : 0; }
int attention_hd16_fp32_products() { return g_hd16_fp32_products; }

hipError_t launch_attention_hd16(const float* q, const float* k, const float* v, float* out, float* lse2, int B,
                                 int heads, int L, hipStream_t stream) {
    if (L % 128 != 0) return hipErrorInvalidValue;
    const float scale_log2e = 0.25f * 1.4426950408889634f;
    dim3 grid((L / 128) * B * heads);
    const FlashPre no_pre{nullptr, nullptr, nullptr};
    if (g_hd16_fp32_products)
        DANRA_LAUNCH_KERNEL((k_flash_hd16<2, 0, false, false>), grid, dim3(256), 0, stream, q, k, v, out, lse2, L, heads,
                           B * heads, scale_log2e, no_pre, QkvLayout{});
    else
        DANRA_LAUNCH_KERNEL(k_flash_hd16<2>, grid, dim3(256), 0, stream, q, k, v, out, lse2, L, heads, B * heads, scale_log2e, no_pre,
                           QkvLayout{});
    return hipGetLastError();
}

// the same core on the output of a fused QKV projection, used in place: qkv [B][L][3][heads * 16]
hipError_t launch_attention_hd16_tokens(const float* qkv, float* out, float* lse2, int B, int heads, int L, hipStream_t stream) {
    if (L % 128 != 0) return hipErrorInvalidValue;
    const float scale_log2e = 0.25f * 1.4426950408889634f;
    dim3 grid((L / 128) * B * heads);
    const FlashPre no_pre{nullptr, nullptr, nullptr};
    const int C = heads * 16;
    const QkvLayout lay{3 * C, (long long)L * 3 * C, 16};
    const float *q = qkv, *k = qkv + C, *v = qkv + 2 * C;
    if (g_hd16_fp32_products)
        DANRA_LAUNCH_KERNEL((k_flash_hd16<2, 0, false, false, 1, false, true>), grid, dim3(256), 0, stream, q, k, v, out, lse2, L,
                           heads, B * heads, scale_log2e, no_pre, lay);
    else
        DANRA_LAUNCH_KERNEL((k_flash_hd16<2, 0, true, true, 1, false, true>), grid, dim3(256), 0, stream, q, k, v, out, lse2, L,
                           heads, B * heads, scale_log2e, no_pre, lay);
    return hipGetLastError();
}

hipError_t launch_attention(const float* q, const float* k, const float* v, float* out, int B, int heads, int L,
                            int hd, hipStream_t stream) {
    if (hd == 16 && L % 128 == 0) return launch_attention_hd16(q, k, v, out, nullptr, B, heads, L, stream);
    if (L % 64 == 0 && L >= 256) {
        if (hd == 32) return launch_flash_wide<2>(q, k, v, out, B, heads, L, stream);
        if (hd == 64) return launch_flash_wide<4>(q, k, v, out, B, heads, L, stream);
    }
    if (L == 64 && hd == 128) return launch_flash_wide_qt<8, 1>(q, k, v, out, B, heads, L, stream);
    if (L <= 16 && hd > 128) {
        const float scale = 1.0f / sqrtf((float)hd);
        const dim3 grid(B * heads), block(64 * L);
        if (hd <= 256 && L <= 4) hipLaunchKernelGGL((k_attn_tiny<4, 4>), grid, block, 0, stream, q, k, v, out, L, hd, heads, scale);
        else if (hd <= 256) hipLaunchKernelGGL((k_attn_tiny<4, 16>), grid, block, 0, stream, q, k, v, out, L, hd, heads, scale);
        else if (hd <= 512 && L <= 4) hipLaunchKernelGGL((k_attn_tiny<8, 4>), grid, block, 0, stream, q, k, v, out, L, hd, heads, scale);
        else if (hd <= 512) hipLaunchKernelGGL((k_attn_tiny<8, 16>), grid, block, 0, stream, q, k, v, out, L, hd, heads, scale);
        else return hipErrorInvalidValue;
        return hipGetLastError();
    }
    if (L <= 256) {
        if (hd == 32) return launch_attn_reg<2>(q, k, v, out, B, heads, L, stream);
        if (hd == 64) return launch_attn_reg<4>(q, k, v, out, B, heads, L, stream);
        if (hd == 128) return launch_attn_reg<8>(q, k, v, out, B, heads, L, stream);
    }
    if (hd <= 128) return launch_attn_small<2, 64>(q, k, v, out, B, heads, L, hd, stream);
    if (hd <= 256) return launch_attn_small<4, 32>(q, k, v, out, B, heads, L, hd, stream);
    if (hd <= 512) return launch_attn_small<8, 16>(q, k, v, out, B, heads, L, hd, stream);
    return hipErrorInvalidValue;
}

}  // namespace danra
