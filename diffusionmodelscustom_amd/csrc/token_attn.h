// What the kernels of danra_token_attention_* share: the arguments, the score of one (query, key) pair with its cap, distance bias
// and mask, and the matrix-core tiles.
//
//   score(i, j) = cap tanh(scale q_i.k_j / cap) - slope |pos_i - j|      (without a cap: scale q_i.k_j - slope |pos_i - j|)
//   pos_i       = i + kv_len - Lq                                          (the queries are the last of their sequence)
//   seen(i, j)  = j < limit_i  and  doc_q[i] == doc_k[j]                   limit_i = kv_len, or with the causal mask
//                                                                          min(kv_len, max(pos_i + 1, prefix))
// All scores are kept in units of log2 (p = 2^(score2 - ...)), so that the exponential is one instruction.
//
// Every product is a 32x32 matrix instruction.  The "owner" axis (the one a wave keeps in registers) lies on the columns: lane l
// holds column l % 32, the streamed axis lies on the rows, element e of the accumulator being row 8 (e / 4) + 4 (l / 32) + e % 4.
// So a column's statistics are private to two lanes, and the accumulator of one product, rounded to the operand's type, IS the right
// operand of the next one over the same streamed rows (its k index is a permutation of them that both operands share): P and dS
// never leave the registers.
#pragma once
#include "danra_kernels.h"

#include <cfloat>

namespace danra {
namespace token {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 32;  // columns of a tile: the rows of the owner axis that one wave holds

template <typename T>
struct Type;
template <>
struct Type<__bf16> {
    typedef bf16x8 Frag;
    // P is at most 2^kGrow and dS has float32's exponent: nothing to rescale
    static constexpr bool kNarrow = false;
    static __device__ __forceinline__ f32x16 mfma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float sum(Frag a, float c) {  // of the eight values and c
        typedef __bf16 Two __attribute__((ext_vector_type(2)));
        const Two one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
        for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2_f32_bf16(Two{a[j], a[j + 1]}, one, c, false);
        return c;
    }
};
template <>
struct Type<_Float16> {
    typedef f16x8 Frag;
    static constexpr bool kNarrow = true;
    static __device__ __forceinline__ f32x16 mfma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float sum(Frag a, float c) {
        typedef _Float16 Two __attribute__((ext_vector_type(2)));
        const Two one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
        for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2(Two{a[j], a[j + 1]}, one, c, false);
        return c;
    }
};
template <>
struct Type<float> {
    typedef f32x8 Frag;
    static constexpr bool kNarrow = false;
    static __device__ __forceinline__ f32x16 mfma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// other half of the wave: lanes l and l ^ 32 hold the same column
__device__ __forceinline__ float pair_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = max(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = min(x, __shfl_xor(x, o));
    return x;
}

// ------------------------------------------------------------------------------------------------------------------ tiles in LDS
// A tile is rows of `stride` elements; the 16-byte chunks of a row are permuted by an exclusive or with a function of the row, chosen
// so that both ways of reading spread over the banks: 16 consecutive rows at one chunk (row fragments), and 4 consecutive rows
// over 64 bytes (transposed fragments).
template <typename T, int DK>
struct Tile {
    static constexpr int kStride = DK <= 16 ? 16 : DK <= 32 ? 32 : DK <= 64 ? 64 : 128;  // elements
    static constexpr int kPer = 16 / (int)sizeof(T);                                      // elements of a chunk
    static constexpr int kChunks = kStride / kPer;
    static constexpr int kData = DK / kPer;  // chunks of a row that hold data
    static constexpr int kRowBytes = kStride * (int)sizeof(T);

    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (kChunks >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        else if constexpr (kChunks == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else if constexpr (kChunks == 4) return (r >> 2) & 3;
        else return (r >> 3) & 1;
    }
    static __device__ __forceinline__ char* chunk(char* tile, int r, int c) { return tile + r * kRowBytes + ((c ^ swizzle(r)) << 4); }
    static __device__ __forceinline__ const char* chunk(const char* tile, int r, int c) {
        return tile + r * kRowBytes + ((c ^ swizzle(r)) << 4);
    }

    // eight consecutive elements from `d` (a multiple of 8) of row r
    static __device__ __forceinline__ typename Type<T>::Frag row(const char* tile, int r, int d) {
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const typename Type<T>::Frag*>(chunk(tile, r, d / kPer));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(chunk(tile, r, d / kPer));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(chunk(tile, r, d / kPer + 1));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    static __device__ __forceinline__ void set_row(char* tile, int r, int d, const typename Type<T>::Frag& f) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<typename Type<T>::Frag*>(chunk(tile, r, d / kPer)) = f;
        } else {
            *reinterpret_cast<f32x4*>(chunk(tile, r, d / kPer)) = __builtin_shufflevector(f, f, 0, 1, 2, 3);
            *reinterpret_cast<f32x4*>(chunk(tile, r, d / kPer + 1)) = __builtin_shufflevector(f, f, 4, 5, 6, 7);
        }
    }

    // the transposed fragment: element j of lane l is tile[r0 + 8 (j / 4) + 4 (l / 32) + j % 4][d0 + l % 32], the order of the
    // accumulator elements 8 s .. 8 s + 7 for r0 = 16 s.  (Rows of 16 channels: the lanes of the channels behind them, whose results are not
    // written, read the same 16 again.)
    static __device__ __forceinline__ typename Type<T>::Frag column(const char* tile, int r0, int d0, int lane) {
        if constexpr (sizeof(T) == 2) {
            // a group of 16 lanes reads 4 rows x 16 columns, 8 bytes a lane, and receives the transpose
            const int i = lane & 15, r = r0 + 4 * (lane >> 5) + (i >> 2), d = (d0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3)) & (kStride - 1);
            typedef s16x4 __attribute__((address_space(3))) * Lds;
            const char* a = chunk(tile, r, d >> 3) + ((d & 4) << 1);
            const char* b = chunk(tile, r + 8, d >> 3) + ((d & 4) << 1);
            union {
                s16x4 h[2];
                typename Type<T>::Frag f;
            } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(a));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(b));
            return u.f;
        } else {
            const int d = (d0 + (lane & 31)) & (kStride - 1), r = r0 + 4 * (lane >> 5);
            typename Type<T>::Frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int rr = r + 8 * (j >> 2) + (j & 3);
                f[j] = *reinterpret_cast<const float*>(chunk(tile, rr, d >> 2) + ((d & 3) << 2));
            }
            return f;
        }
    }
};

typedef __attribute__((address_space(3))) char* LdsPtr;
typedef u32x4 Buffer;
constexpr unsigned kNowhere = 0x80000000u;  // an offset past the end of every buffer: reads as zero

// Loads that pass by the registers: 16 or 4 bytes a lane from buffer + offset to lds + 16 (4) lane; lds is the same for the wave.  They
// are written out because the compiler takes the builtin for a possible writer of whatever LDS is read next and waits for it there, which
// is the time that it is meant to overlap with.  So nothing but settle_loads waits for them: it stands in front of every barrier
// behind which a tile is read.  (No register is written; s_nop 4: the wait states between a vector instruction that has made one of
// the scalar operands and the load, and between m0 and the load.)
__device__ __forceinline__ unsigned lds_at(const char* lds) { return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(LdsPtr)lds); }
__device__ __forceinline__ void load_lds4(const Buffer& from, unsigned offset, char* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds_at(lds)), "v"(offset), "s"(from) : "memory", "m0");
}
// N loads of 16 bytes a lane, STEP bytes of LDS apart
template <int N, int STEP>
__device__ __forceinline__ void load_lds16(const Buffer& from, const unsigned (&offset)[N], char* lds) {
    const unsigned to = lds_at(lds);
    if constexpr (N > 4) {
        unsigned first[4], others[N - 4];
#pragma unroll
        for (int n = 0; n < N; ++n) (n < 4 ? first[n & 3] : others[n < 4 ? 0 : n - 4]) = offset[n];
        load_lds16<4, STEP>(from, first, lds);
        load_lds16<N - 4, STEP>(from, others, lds + 4 * STEP);
    } else if constexpr (N == 4) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds" ::"s"(to), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]),
                     "v"(offset[3]), "s"(from), "n"(STEP) : "memory", "m0", "scc");
    } else if constexpr (N == 3) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %4, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds" ::"s"(to), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]),
                     "s"(from), "n"(STEP) : "memory", "m0", "scc");
    } else if constexpr (N == 2) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" ::"s"(to), "v"(offset[0]), "v"(offset[1]), "s"(from),
                     "n"(STEP) : "memory", "m0", "scc");
    } else {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset[0]), "s"(from) : "memory", "m0");
    }
}
__device__ __forceinline__ void settle_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0); the compiler takes note of it
// a buffer of `bytes` bytes from p (the same for the wave): loads past its end give zero
__device__ __forceinline__ Buffer buffer(const void* p, unsigned bytes) {
    const unsigned long long at = (unsigned long long)p;
    return Buffer{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)at), (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(at >> 32) & 0xffffu),
                  (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// ROWS rows of a tile, brought to LDS by WAVES waves: each load of a wave fills 64 chunks in the order of the LDS, every lane asking for
// the chunk of memory that belongs there.  (settle_loads, then a barrier, stand in front of the tile's use.)
template <typename T, int DK, int ROWS, int WAVES>
struct Stage {
    typedef Tile<T, DK> Tl;
    static constexpr int kLoads = ROWS * Tl::kChunks / 64;           // of a wave, for the whole tile
    static constexpr int kEach = (kLoads + WAVES - 1) / WAVES;
    static_assert(ROWS * Tl::kChunks % 64 == 0, "whole waves");
    static __device__ __forceinline__ int row(int n, int wave, int lane) { return ((wave + n * WAVES) * 64 + lane) / Tl::kChunks; }
    static __device__ __forceinline__ int chunk(int n, int wave, int lane) {
        return ((wave + n * WAVES) * 64 + lane) % Tl::kChunks ^ Tl::swizzle(row(n, wave, lane));
    }
    // where lane's chunk of load n lies in its row, in bytes (kNowhere: past the head's channels)
    static __device__ __forceinline__ unsigned column(int n, int wave, int lane, int D) {
        const int c = chunk(n, wave, lane);
        return c * Tl::kPer < D ? (unsigned)c * 16u : kNowhere;
    }
    static_assert(kLoads % WAVES == 0 || kLoads < WAVES, "each wave has kEach loads, or the first kLoads waves have one");
    static __device__ __forceinline__ void load(const Buffer& from, const unsigned (&offset)[kEach], char* tile, int wave) {
        if (kLoads % WAVES == 0 || wave < kLoads) load_lds16<kEach, WAVES * 1024>(from, offset, tile + wave * 1024);
    }
};

// the same for consecutive rows `stride` bytes apart: the lanes' offsets are the same for every tile
template <typename T, int DK, int ROWS, int WAVES>
struct Rowwise {
    typedef Stage<T, DK, ROWS, WAVES> St;
    unsigned at[St::kEach];
    __device__ __forceinline__ void prepare(unsigned stride, int D, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < St::kEach; ++n) {
            const unsigned c = St::column(n, wave, lane, D);
            at[n] = c == kNowhere ? kNowhere : (unsigned)St::row(n, wave, lane) * stride + c;
        }
    }
    // `count` rows from p; `dead(r)`: row r reads as zero (asked only with `some`)
    template <typename Dead>
    __device__ __forceinline__ void load(const void* p, int count, unsigned stride, int D, char* tile, int wave, int lane, bool some, Dead dead) {
        const Buffer from = buffer(p, (unsigned)(min(count, ROWS) - 1) * stride + (unsigned)(D * sizeof(T)));
        if (!some) {
            St::load(from, at, tile, wave);
        } else {
            unsigned offset[St::kEach];
#pragma unroll
            for (int n = 0; n < St::kEach; ++n) offset[n] = dead(St::row(n, wave, lane)) ? kNowhere : at[n];
            St::load(from, offset, tile, wave);
        }
    }
};

// the owner's fragments: lane l holds row l % 32 (its address, or null for zeros), elements 16 s + 8 (l / 32) .. + 7 of step s
template <typename T, int DK>
__device__ __forceinline__ void load_owner(typename Type<T>::Frag (&f)[DK / 16], const T* row, int D, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int s = 0; s < DK / 16; ++s) {
        const int d = 16 * s + 8 * half;
        union {
            u32x4 u[sizeof(T) / 2];
            typename Type<T>::Frag f;
        } x;
#pragma unroll
        for (int n = 0; n < (int)sizeof(T) / 2; ++n) x.u[n] = u32x4{0, 0, 0, 0};
        if (row && d < D) {
#pragma unroll
            for (int n = 0; n < (int)sizeof(T) / 2; ++n) x.u[n] = reinterpret_cast<const u32x4*>(row + d)[n];
        }
        f[s] = x.f;
    }
}

// accumulator elements 8 s .. 8 s + 7, rounded to the operand's type
template <typename T>
__device__ __forceinline__ typename Type<T>::Frag round_frag(const f32x16& c, int s) {
    typename Type<T>::Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)c[8 * s + j];
    return f;
}
// what that rounding leaves of them, in the operand's type
template <typename T>
__device__ __forceinline__ typename Type<T>::Frag rest_frag(const f32x16& c, const typename Type<T>::Frag& rounded, int s) {
    typename Type<T>::Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)(c[8 * s + j] - (float)rounded[j]);
    return f;
}

// ------------------------------------------------------------------------------------------------------------------ rows and masks
// The query rows of one key head: row r is query r / G of head hk * G + r % G, so that the G heads that share keys are one axis.
struct Rows {
    int G;
    unsigned magic;  // ceil(2^32 / G); r / G = mulhi(r, magic) for r G < 2^32
    __device__ __forceinline__ int query(int r) const { return G == 1 ? r : (int)__umulhi((unsigned)r, magic); }
};

struct Mask {
    int kv_len, shift, prefix, causal;  // shift = kv_len - Lq: pos_i = i + shift
    __device__ __forceinline__ int limit(int i) const {
        return causal ? min(kv_len, max(i + shift + 1, prefix)) : kv_len;
    }
};

__device__ __forceinline__ Mask make_mask(const TokenAttnArgs& a, int b) {
    Mask m;
    m.kv_len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Lk) : a.Lk;
    m.shift = m.kv_len - a.Lq;
    m.prefix = a.prefix ? a.prefix[b] : 0;
    m.causal = a.causal;
    return m;
}

// score2 = out * (bend(x) - slope / out * |distance|) for the product x = q.k, out > 0: so the exponent of a score is one multiply-add and the
// largest score is the largest of the bent products.  A negative scale is taken into the owner's fragments (owner_sign).
struct Score {
    float in, out;
};

// Three forms of the cap.  kQuick: cap tanh(y) = cap - 2 cap / (1 + e^{2y}), and the softmax does not see the constant cap, so it is left out:
// one exponential, one reciprocal.  Its error is an absolute one of the score, about 2 cap 2^-24, which is the relative error of a P: at
// cap 256 a thirtieth of half a step of float16.  kExact: cap tanh32(y), whose error is relative to the score: float32 tensors, and
// two-byte ones with a larger cap (launchers: cap_of; 16 heads of 4096 tokens, quick and exact: bfloat16, D = 128, forward 190 and 271 us,
// dk and dv 474 and 543, dq 299 and 365; float16, D = 64, 138 and 228, 268 and 352, 217 and 301).
enum Cap { kNoCap, kQuick, kExact };
inline Cap cap_of(const TokenAttnArgs& a) { return !(a.cap > 0.f) ? kNoCap : a.type == TOKEN_F32 || a.cap > 256.f ? kExact : kQuick; }

template <Cap CAP>
__device__ __forceinline__ Score make_score(const TokenAttnArgs& a) {
    Score s;
    const float scale = fmaxf(fabsf(a.scale), 1e-30f);  // (scale 0: nothing of the product is left at 1e-30 either)
    if constexpr (CAP == kNoCap) {
        s.in = 1.f;
        s.out = scale * kLog2e;
    } else if constexpr (CAP == kQuick) {
        s.in = fminf(2.f * kLog2e * scale / a.cap, FLT_MAX);  // (an infinite factor would make no number of a product of 0)
        s.out = 2.f * a.cap * kLog2e;
    } else {
        s.in = fminf(scale / a.cap, FLT_MAX);
        s.out = a.cap * kLog2e;
    }
    return s;
}

// the owner's fragments with the sign of the scale
template <typename T, int N>
__device__ __forceinline__ void owner_sign(typename Type<T>::Frag (&f)[N], float scale) {
    if (scale < 0.f) {
#pragma unroll
        for (int n = 0; n < N; ++n) f[n] = -f[n];
    }
}

// tanh to about 1e-7 relative without branches: an odd polynomial up to 0.55 (least squares of (tanh y / y - 1) / y^2 over y^2; 6e-8), from there
// 1 - 2 e / (1 + e) with e = 2^(-2 y log2 e), where nothing cancels.  (The library's tanhf costs the float32 kernels of a 1024-token map
// 10 us of 70.)
__device__ __forceinline__ float tanh32(float y) {
    const float a = fabsf(y), u = y * y;
    float p = fmaf(-0.006615746766328812f, u, 0.021312739700078964f);
    p = fmaf(p, u, -0.053910065442323685f);
    p = fmaf(p, u, 0.13333117961883545f);
    p = fmaf(p, u, -0.3333333134651184f);
    const float e = __builtin_amdgcn_exp2f(-2.f * kLog2e * a);
    const float big = fmaf(-2.f * e, __builtin_amdgcn_rcpf(1.f + e), 1.f), small = fmaf(y * u, p, y);
    return a < 0.55f ? small : copysignf(big, y);
}

template <Cap CAP>
__device__ __forceinline__ float bend(float x, const Score& s) {
    if constexpr (CAP == kNoCap) return x;
    else if constexpr (CAP == kQuick) return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s.in * x));
    else return tanh32(s.in * x);
}
// the cap's derivative 1 - tanh^2 at z = bend(x), up to a constant factor: with z = -1 / (1 + e^{2y}) it is -4 (z + z^2)
template <Cap CAP>
__device__ __forceinline__ float bend_slope(float z) {
    if constexpr (CAP == kQuick) return fmaf(z, z, z);
    else return fmaf(-z, z, 1.f);
}
template <Cap CAP>
__device__ __forceinline__ constexpr float bend_factor() { return CAP == kQuick ? -4.f : 1.f; }

// ------------------------------------------------------------------------------------------------------------------ tiles of a loop
// Which of the streamed tiles [first, last) a workgroup visits: all of them, or those whose range of document ids overlaps its own;
// and what is known of each.  64 tiles are looked at at once, one a lane, so that the loop waits for no load of its own between tiles.
// Every wave of the workgroup finds the same tiles; `same` is the wave's own.
struct Visit {
    int t;      // -1: none left
    bool wanted;  // its documents overlap the wave's own (true without documents)
    bool same;  // every key and row of the tile is of the wave's one document (true without documents)
    bool dead;  // some rows of the tile have to read as zero whatever they hold
};
struct TileList {
    const int4* ranges;  // per tile {lowest id, highest id, 1 if all ids are equal, 1 if some are negative}, the negative ones left
                         // out (lowest > highest: none); or null
    const int* flags;    // per tile: `dead`, or null (then the fourth of the ranges)
    int lo, hi;          // the workgroup's range of ids
    int my_lo, my_hi;    // the wave's
    int base, last;
    unsigned long long bits, my_bits, same_bits, dead_bits;
    __device__ __forceinline__ void look(int lane) {
        const int t = base + lane;
        bool wanted = t < last, mine = true, same = true, dead = false;
        if (wanted && ranges) {
            const int4 g = ranges[t];
            wanted = g.x <= hi && g.y >= lo && g.x <= g.y;
            mine = g.x <= my_hi && g.y >= my_lo;
            same = g.z && g.x == my_lo && my_lo == my_hi;
            dead = g.w;
        }
        if (t < last && flags) dead = flags[t];
        bits = __ballot(wanted);
        my_bits = __ballot(mine);
        same_bits = __ballot(same);
        dead_bits = __ballot(dead);
    }
    __device__ __forceinline__ Visit next(int lane) {
        while (!bits) {
            base += 64;
            if (base >= last) return Visit{-1, false, false, false};
            look(lane);
        }
        const int n = __builtin_ctzll(bits);
        bits &= bits - 1;
        return Visit{base + n, (bool)(my_bits >> n & 1), (bool)(same_bits >> n & 1), (bool)(dead_bits >> n & 1)};
    }
    __device__ __forceinline__ int count(int lane) const {  // of the tiles from here on (a list that was just started)
        if (!ranges) return max(last - base, 0);
        int n = 0;
        for (int t = base; t < last; t += 64) {
            bool wanted = t + lane < last;
            if (wanted) {
                const int4 g = ranges[t + lane];
                wanted = g.x <= hi && g.y >= lo && g.x <= g.y;
            }
            n += __builtin_popcountll(__ballot(wanted));
        }
        return n;
    }
    __device__ __forceinline__ void skip(int n, int lane) {
        if (!ranges) {
            base += n;
            bits = 0;
            if (base < last) look(lane);
            return;
        }
        while (base < last) {
            const int here = __builtin_popcountll(bits);
            if (n < here) {
                for (; n > 0; --n) bits &= bits - 1;
                return;
            }
            n -= here;
            base += 64;
            bits = 0;
            if (base < last) look(lane);
        }
    }
    __device__ __forceinline__ void start(const int4* r, const int* f, int lo_, int hi_, int my_lo_, int my_hi_, int first, int end, int lane) {
        ranges = r;
        flags = f;
        lo = lo_;
        hi = hi_;
        my_lo = my_lo_;
        my_hi = my_hi_;
        base = first;
        last = end;
        bits = 0;
        if (base < last) look(lane);
    }
};

// (kernels_token_attn_fwd.hip) {lowest, highest, all equal, some negative} of the document ids of each `per` consecutive places, place p standing
// for ids[p / group]
hipError_t launch_ranges(const int* ids, int4* out, int length, int group, int per, int tiles, int batch, hipStream_t stream);

// The loop over a workgroup's tiles with two buffers: the next tile is on its way while one is worked on.  Written out for either buffer,
// so that every address in LDS is a register and a constant.
template <int N>
struct Const {
    __device__ __forceinline__ constexpr int operator()() const { return N; }
};
template <typename Next, typename Load, typename Work>
__device__ __forceinline__ void two_buffers(Next next, Load stage, Work work) {
    Visit a = next();
    if (a.t < 0) return;
    stage(a, 0);
    settle_loads();
    __syncthreads();
    for (;;) {
        const Visit b = next();
        if (b.t >= 0) stage(b, 1);
        work(a, Const<0>());
        if (b.t < 0) return;
        settle_loads();
        __syncthreads();
        a = next();
        if (a.t >= 0) stage(a, 0);
        work(b, Const<1>());
        if (a.t < 0) return;
        settle_loads();
        __syncthreads();
    }
}

// parts of a workspace, each on 16 bytes; without a base their size alone
struct Parts {
    char* base;
    size_t bytes = 0;
    template <typename P>
    void take(P*& p, size_t n) {
        if (base) p = reinterpret_cast<P*>(base + bytes);
        bytes += (n * sizeof(P) + 15) / 16 * 16;
    }
};

// workgroup index -> (tile, batch and key head): the heads vary fastest, so that (consecutive workgroups go to the 8 XCDs in turn)
// the tiles of one head share an XCD's L2 where the number of heads is a multiple of 8
__device__ __forceinline__ void place(int heads, int& tile, int& bh) {
    bh = blockIdx.x % heads;
    tile = blockIdx.x / heads;
}

}  // namespace token
}  // namespace danra
