// Root-mean-square norm of every query and key head with a gain per channel, and the position rotation, in one pass:
//   n = x r,  r = (mean(x^2) + eps)^-1/2,  y = rot(n w)           rot: the pair (a, b) becomes (a cos - b sin, b cos + a sin)
// and its backward pass:
//   g = rot^-1(dy),  dx = r (g w - n mean(g w n)),  dw = sum over all heads of g n
// Statistics and rotation are float32.  The passes are bound by their one reading and one writing of the heads, so the work is
// laid out for wide accesses: a lane holds V pairs of a head, both members of a pair in the lane (two vectors of V channels, or 2 V
// adjacent ones), D / 2V lanes form a head, and the cosines and sines that a lane needs are read once per token and kept for all the
// heads that its workgroup takes.  The gains' gradient is summed per lane in float32, then over the workgroup through LDS and by a second
// kernel over the workgroups in float64 (there are few of those sums, and in float32 they made the gradient four times as far off as its
// rounding), each in a fixed order.
//
// Measured (bfloat16, D = 128, 8192 tokens of 16 + 4 heads, 84 MB forward and 126 backward): 28 us and 37 + 4 for the gains, 3.0 and 3.4
// TB/s, against the 4.7 TB/s of a large copy.  The length of the pass does not explain it (the clipping's second pass moves twice as
// many bytes at 5.9 TB/s, its reads partly from the cache): a workgroup per CU goes through five rounds of asking for kHeads heads, waiting,
// reducing and writing, with no load under way in between.
#include "danra_kernels.h"

namespace danra {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ void set(T* p, const float* x) {
    union {
        typename Vec<T, V>::type v;
        T t[V];
    } u;
#pragma unroll
    for (int e = 0; e < V; ++e) u.t[e] = (T)x[e];
    *reinterpret_cast<typename Vec<T, V>::type*>(p) = u.v;
}

// Where a lane's 2 V channels lie: x[0 .. V) from `first`, x[V .. 2V) from `second`.  For adjacent pairs (and for the channels that are
// not rotated) the two are neighbours, and pair e is (x[2e], x[2e + 1]); otherwise pair e is (x[e], x[V + e]).
struct Place {
    int first, second, pair;  // pair: index of the first pair in the tables, or -1 where nothing is rotated
};
template <int V>
__device__ __forceinline__ Place place_of(int unit, int R, int interleaved) {
    const int turned = R / (2 * V);
    Place p;
    p.pair = unit < turned ? unit * V : -1;
    if (unit < turned && !interleaved) {
        p.first = unit * V;
        p.second = R / 2 + unit * V;
    } else {
        p.first = unit * 2 * V;
        p.second = p.first + V;
    }
    return p;
}

// a lane's channels of one head as they come from memory
template <typename T, int V>
struct Pair {
    union Half {
        typename Vec<T, V>::type v;
        T t[V];
    } lo, hi;
    __device__ __forceinline__ void load(const T* row, const Place& at) {
        lo.v = *reinterpret_cast<const typename Vec<T, V>::type*>(row + at.first);
        hi.v = *reinterpret_cast<const typename Vec<T, V>::type*>(row + at.second);
    }
    __device__ __forceinline__ void get(float* x) const {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[e] = (float)lo.t[e];
            x[V + e] = (float)hi.t[e];
        }
    }
};

template <int V>
__device__ __forceinline__ void rotate(float* x, const float* c, const float* s, bool adjacent, float sign) {
    if (adjacent) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float a = x[2 * e], b = x[2 * e + 1], t = sign * s[e];
            x[2 * e] = fmaf(a, c[e], -b * t);
            x[2 * e + 1] = fmaf(b, c[e], a * t);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float a = x[e], b = x[V + e], t = sign * s[e];
            x[e] = fmaf(a, c[e], -b * t);
            x[V + e] = fmaf(b, c[e], a * t);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void get_gain(float* w, const void* p, int f32, const Place& at) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) w[e] = 1.f;
        return;
    }
    // (a gain tensor may start anywhere its type may: element by element, once per workgroup)
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = f32 ? static_cast<const float*>(p)[at.first + e] : (float)static_cast<const T*>(p)[at.first + e];
        w[V + e] = f32 ? static_cast<const float*>(p)[at.second + e] : (float)static_cast<const T*>(p)[at.second + e];
    }
}

template <int V>
__device__ __forceinline__ void get_turn(float* c, float* s, const TokenRotaryArgs& a, const Place& at, long long token) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        c[e] = 1.f;
        s[e] = 0.f;
    }
    if (at.pair < 0) return;
    const long long pos = a.positions ? a.positions[token] : token % a.L;
    const bool in = pos >= 0 && pos < a.table;  // a position outside the tables turns the rotated channels into NaN
    const size_t from = (size_t)(in ? pos : 0) * (a.R / 2) + at.pair;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        c[e] = in ? a.cosine[from + e] : __builtin_nanf("");
        s[e] = in ? a.sine[from + e] : __builtin_nanf("");
    }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// grid: x = groups of tokens, y = spans of heads.  LANES lanes (a power of two, units <= LANES) take one head of one token at a time.
template <typename T, int V, int LANES>
__global__ __launch_bounds__(256) void k_token_rotary_fwd(const TokenRotaryArgs a) {
    const int unit = threadIdx.x % LANES, units = a.D / (2 * V);
    const long long token = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (token >= (long long)a.B * a.L) return;  // (whole groups)
    const bool mine = unit < units;
    const Place at = place_of<V>(mine ? unit : 0, a.R, a.interleaved);
    const bool adjacent = a.interleaved;
    const int b = (int)(token / a.L), l = (int)(token - (long long)b * a.L);
    float c[V], s[V];
    get_turn<V>(c, s, a, at, token);
    const int h0 = blockIdx.y * a.span, h1 = min(h0 + a.span, a.heads[0] + a.heads[1]);
    const float per = 1.f / (float)a.D;
    constexpr int kHeads = 4;  // read ahead
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int from = max(h0 - which * a.heads[0], 0), to = which ? h1 - a.heads[0] : min(h1, a.heads[0]);
        if (from >= to) continue;
        float w[2 * V];
        get_gain<T, V>(w, a.w[which], a.w_f32, at);
        const T* x = static_cast<const T*>(a.x[which]) + (long long)b * a.x_stride[which][0] + (long long)l * a.x_stride[which][1];
        T* y = static_cast<T*>(a.y[which]) + (size_t)token * a.heads[which] * a.D;
        for (int h = from; h < to; h += kHeads) {
            Pair<T, V> raw[kHeads];
#pragma unroll
            for (int u = 0; u < kHeads; ++u) raw[u].load(x + (long long)min(h + u, to - 1) * a.x_stride[which][2], at);
#pragma unroll
            for (int u = 0; u < kHeads; ++u) {
                float v[2 * V];
                raw[u].get(v);
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 2 * V; ++e) sum = fmaf(v[e], v[e], sum);
                const float mean = group_sum<LANES>(mine ? sum : 0.f) * per;
                const float r = 1.f / sqrtf(mean + a.eps);
#pragma unroll
                for (int e = 0; e < 2 * V; ++e) v[e] = v[e] * r * w[e];
                rotate<V>(v, c, s, adjacent, 1.f);
                if (mine && h + u < to) {
                    set<T, V>(y + (size_t)(h + u) * a.D + at.first, v);
                    set<T, V>(y + (size_t)(h + u) * a.D + at.second, v + V);
                }
            }
        }
    }
}

// grid: a.blocks workgroups, each taking every a.blocks-th (group of tokens, span of heads)
template <typename T, int V, int LANES>
__global__ __launch_bounds__(256) void k_token_rotary_bwd(const TokenRotaryArgs a) {
    constexpr int kGroups = 256 / LANES;
    const int unit = threadIdx.x % LANES, units = a.D / (2 * V), group = threadIdx.x / LANES;
    const bool mine = unit < units;
    const Place at = place_of<V>(mine ? unit : 0, a.R, a.interleaved);
    const bool adjacent = a.interleaved;
    const long long tokens = (long long)a.B * a.L, packs = (tokens + kGroups - 1) / kGroups;
    const int heads = a.heads[0] + a.heads[1], spans = (heads + a.span - 1) / a.span;
    const float per = 1.f / (float)a.D;
    constexpr int kHeads = 2;  // read ahead
    float dw[2][2 * V], w[2][2 * V];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        get_gain<T, V>(w[which], a.w[which], a.w_f32, at);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) dw[which][e] = 0.f;
    }
    for (long long item = blockIdx.x; item < packs * spans; item += gridDim.x) {
        const long long token = item / spans * kGroups + group;
        if (token >= tokens) continue;
        const int h0 = (int)(item % spans) * a.span, h1 = min(h0 + a.span, heads);
        const int b = (int)(token / a.L), l = (int)(token - (long long)b * a.L);
        float c[V], s[V];
        get_turn<V>(c, s, a, at, token);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int from = max(h0 - which * a.heads[0], 0), to = which ? h1 - a.heads[0] : min(h1, a.heads[0]);
            const T* x = static_cast<const T*>(a.x[which]) + (long long)b * a.x_stride[which][0] + (long long)l * a.x_stride[which][1];
            const T* dy = static_cast<const T*>(a.dy[which]) + (long long)b * a.dy_stride[which][0] + (long long)l * a.dy_stride[which][1];
            T* dx = static_cast<T*>(a.y[which]) + (size_t)token * a.heads[which] * a.D;
            for (int h = from; h < to; h += kHeads) {
                Pair<T, V> raw[kHeads], raw_dy[kHeads];
#pragma unroll
                for (int u = 0; u < kHeads; ++u) {
                    raw[u].load(x + (long long)min(h + u, to - 1) * a.x_stride[which][2], at);
                    raw_dy[u].load(dy + (long long)min(h + u, to - 1) * a.dy_stride[which][2], at);
                }
#pragma unroll
                for (int u = 0; u < kHeads; ++u) {
                    float v[2 * V], g[2 * V];
                    raw[u].get(v);
                    raw_dy[u].get(g);
                    rotate<V>(g, c, s, adjacent, -1.f);
                    float sum = 0.f, dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 2 * V; ++e) {
                        sum = fmaf(v[e], v[e], sum);
                        dot = fmaf(g[e] * w[which][e], v[e], dot);
                    }
                    sum = group_sum<LANES>(mine ? sum : 0.f);
                    dot = group_sum<LANES>(mine ? dot : 0.f);
                    const float r = 1.f / sqrtf(sum * per + a.eps);
                    const float pull = dot * r * per;  // mean(g w n)
                    if (h + u < to) {
#pragma unroll
                        for (int e = 0; e < 2 * V; ++e) {
                            const float n = v[e] * r;
                            dw[which][e] = fmaf(g[e], n, dw[which][e]);
                            v[e] = r * fmaf(-n, pull, g[e] * w[which][e]);
                        }
                        if (mine) {
                            set<T, V>(dx + (size_t)(h + u) * a.D + at.first, v);
                            set<T, V>(dx + (size_t)(h + u) * a.D + at.second, v + V);
                        }
                    }
                }
            }
        }
    }
    if (!a.partial) return;
    __shared__ float sums[kGroups * LANES * 2 * V];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (mine) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sums[group * a.D + at.first + e] = dw[which][e];
                sums[group * a.D + at.second + e] = dw[which][V + e];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += 256) {
            double t = 0.0;
            for (int k = 0; k < kGroups; ++k) t += sums[k * a.D + d];
            a.partial[((size_t)blockIdx.x * 2 + which) * a.D + d] = (float)t;
        }
    }
}

// dw[which][d] = sum over the workgroups: 4 channels x 64 slices of the workgroups, the slices added in order
template <typename T>
__global__ __launch_bounds__(256) void k_token_rotary_gains(const TokenRotaryArgs a) {
    __shared__ double s[64][4];
    const int which = blockIdx.y, d = blockIdx.x * 4 + (threadIdx.x & 3), slice = threadIdx.x >> 2;
    double t = 0.0;
#pragma unroll 8
    for (int k = slice; k < a.blocks; k += 64) t += a.partial[((size_t)k * 2 + which) * a.D + d];
    s[slice][threadIdx.x & 3] = t;
    __syncthreads();
    if (threadIdx.x < 4 && a.dw[which]) {
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < 64; ++k) sum += s[k][threadIdx.x];
        if (a.w_f32) static_cast<float*>(a.dw[which])[d] = (float)sum;
        else static_cast<T*>(a.dw[which])[d] = (T)(float)sum;
    }
}

constexpr int kRotaryBlocks = 1024;

// pairs of a lane: as many as fill 16 bytes, where the rotated and the other channels both divide into such lanes
int pairs_of(const TokenRotaryArgs& a) {
    int v = a.type == TOKEN_F32 ? 4 : 8;
    while (v > 1 && (a.R / 2 % v || (a.D - a.R) / 2 % v)) v /= 2;
    return v;
}

template <typename T, int V, int LANES>
hipError_t rotary(TokenRotaryArgs& a, bool backward, hipStream_t stream) {
    const long long tokens = (long long)a.B * a.L;
    const int heads = a.heads[0] + a.heads[1], groups = 256 / LANES;
    const long long packs = (tokens + groups - 1) / groups;
    // All heads of a token to one group of lanes where there are tokens enough for a workgroup per CU, so that the cosines and sines are read
    // once; down to one head each (8192 tokens of 16 + 4 heads, D = 128: 28 us, backward 37; one head each 68 and 69; 16 single tokens of 40
    // heads: 7 us with one head each, 28 with all).
    long long span = packs * heads / 256;
    a.span = span < 1 ? 1 : span > heads ? heads : (int)span;
    const int spans = (heads + a.span - 1) / a.span;
    if (!backward) {
        DANRA_LAUNCH_KERNEL((k_token_rotary_fwd<T, V, LANES>), dim3((unsigned)packs, spans), dim3(256), 0, stream, a);
    } else {
        a.blocks = packs * spans < 1 ? 1 : packs * spans < kRotaryBlocks ? (int)(packs * spans) : kRotaryBlocks;
        if (!a.dw[0] && !a.dw[1]) a.partial = nullptr;
        DANRA_LAUNCH_KERNEL((k_token_rotary_bwd<T, V, LANES>), dim3(a.blocks), dim3(256), 0, stream, a);
        if (a.partial) DANRA_LAUNCH_KERNEL((k_token_rotary_gains<T>), dim3(a.D / 4, 2), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

template <typename T, int V>
hipError_t rotary_lanes(TokenRotaryArgs& a, bool backward, hipStream_t stream) {
    const int units = a.D / (2 * V);
    if constexpr (V >= 8) {
        if (units <= 1) return rotary<T, V, 1>(a, backward, stream);
        if (units <= 2) return rotary<T, V, 2>(a, backward, stream);
    }
    if constexpr (V >= 4) {
        if (units <= 4) return rotary<T, V, 4>(a, backward, stream);
        if (units <= 8) return rotary<T, V, 8>(a, backward, stream);
    }
    if constexpr (V >= 2 && V <= 4) {
        if (units <= 16) return rotary<T, V, 16>(a, backward, stream);
    }
    if constexpr (V == 2) return rotary<T, V, 32>(a, backward, stream);
    if constexpr (V == 1) return rotary<T, V, 64>(a, backward, stream);
    return hipErrorInvalidValue;
}

template <typename T>
hipError_t rotary_type(TokenRotaryArgs& a, bool backward, hipStream_t stream) {
    switch (pairs_of(a)) {
        case 8:
            if constexpr (sizeof(T) == 2) return rotary_lanes<T, 8>(a, backward, stream);
            return hipErrorInvalidValue;
        case 4: return rotary_lanes<T, 4>(a, backward, stream);
        case 2: return rotary_lanes<T, 2>(a, backward, stream);
        default: return rotary_lanes<T, 1>(a, backward, stream);
    }
}

hipError_t rotary_any(TokenRotaryArgs& a, bool backward, hipStream_t stream) {
    switch (a.type) {
        case TOKEN_F32: return rotary_type<float>(a, backward, stream);
        case TOKEN_BF16: return rotary_type<__bf16>(a, backward, stream);
        default: return rotary_type<_Float16>(a, backward, stream);
    }
}

}  // namespace

size_t token_rotary_bwd_workspace(const TokenRotaryArgs& a) { return (size_t)kRotaryBlocks * 2 * a.D * sizeof(float); }
hipError_t launch_token_rotary_fwd(TokenRotaryArgs a, hipStream_t stream) { return rotary_any(a, false, stream); }
hipError_t launch_token_rotary_bwd(TokenRotaryArgs a, hipStream_t stream) { return rotary_any(a, true, stream); }

}  // namespace danra
