// The 2-norm of a list of tensors and their scaling: out = g * min(1, max_norm / (norm + eps)).
//
// Two launches for each kClipTensors tensors: one pass that reads them (partial sums of squares, one per workgroup) and one that reads
// them again and writes.  Every workgroup of the second pass adds the partial sums up for itself, in the same fixed order, so that there
// is no third launch and no counter: at most 2048 doubles from L2, and the result does not depend on the order in which workgroups end.
// Squares are summed in float64: a gradient of 1e20 does not overflow and a billion small ones are not lost, and at 8 TB/s
// of HBM the float64 adds are not what bounds the pass: 453 M bfloat16 values 202 us, 4.5 TB/s, and 513 us to read them again and write
// them as float32, 5.3 TB/s.  Half or twice as many workgroups (kClipBlocks) measure the same there, and 31 and 37 us against 32 for the
// second pass over a network's 146 tensors (95 MB).
//
// The tensors' addresses travel as kernel arguments (a table in device memory would need a copy from pageable memory, which a captured
// graph cannot hold).  A tensor is cut in chunks of kClipChunk elements; each workgroup takes a run of consecutive chunks.
#include "danra_kernels.h"

namespace danra {

namespace {

constexpr int kClipTensors = 160;   // 24 bytes each: the arguments stay under 4 KB
constexpr int kClipChunk = 4096;
constexpr int kClipBlocks = 2048;   // partial sums over all launches (8 workgroups for each of 256 CUs)

struct ClipTable {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    unsigned first[kClipTensors];   // the tensor's first chunk
    unsigned facts[kClipTensors];   // elements of its last chunk | input type << 16 | output type << 20
    int count;
    unsigned chunks, each;          // each: chunks of a workgroup
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ double square_sum(const T* p, int n, bool wide) {
    constexpr int V = 16 / (int)sizeof(T), N = kClipChunk / (256 * V);
    double sum = 0.0;
    if (wide && n == kClipChunk) {
        u32x4 v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = reinterpret_cast<const u32x4*>(p)[threadIdx.x + 256 * k];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            union {
                u32x4 u;
                T t[V];
            } x;
            x.u = v[k];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double g = (double)(float)x.t[e];
                sum = fma(g, g, sum);
            }
        }
    } else {
        for (int e = threadIdx.x; e < n; e += 256) {
            const double g = (double)(float)p[e];
            sum = fma(g, g, sum);
        }
    }
    return sum;
}

// sum over a workgroup of 256, the same for every thread
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double s[4];
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// the last tensor whose first chunk is at most c
__device__ __forceinline__ int tensor_of(const ClipTable& t, unsigned c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// a workgroup's chunks, from the first to the last, or BACKWARD
template <bool BACKWARD, typename Fn>
__device__ __forceinline__ void each_chunk(const ClipTable& t, Fn fn) {
    const unsigned begin = blockIdx.x * t.each, end = min(t.chunks, begin + t.each);
    if (begin >= end) return;
    int n = tensor_of(t, BACKWARD ? end - 1 : begin);
    for (unsigned k = 0; k < end - begin; ++k) {
        const unsigned c = BACKWARD ? end - 1 - k : begin + k;
        while (BACKWARD ? t.first[n] > c : n + 1 < t.count && t.first[n + 1] <= c) n += BACKWARD ? -1 : 1;
        const bool last = c + 1 == (n + 1 < t.count ? t.first[n + 1] : t.chunks);
        const unsigned facts = t.facts[n];
        fn(n, (size_t)(c - t.first[n]) * kClipChunk, last ? (int)(facts & 0xffff) : kClipChunk, (int)(facts >> 16 & 15), (int)(facts >> 20));
    }
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

__global__ __launch_bounds__(256) void k_clip_squares(const ClipTable t, double* __restrict__ partial) {
    double sum = 0.0;
    each_chunk<false>(t, [&](int n, size_t at, int len, int type, int) {
        const bool wide = aligned16(t.in[n]);
        if (type == TOKEN_F32) sum += square_sum(static_cast<const float*>(t.in[n]) + at, len, wide);
        else if (type == TOKEN_BF16) sum += square_sum(static_cast<const __bf16*>(t.in[n]) + at, len, wide);
        else sum += square_sum(static_cast<const _Float16*>(t.in[n]) + at, len, wide);
    });
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* p, O* o, int n, float f) {
    // four elements a thread and step: 8 or 16 bytes either way
    typedef T T4 __attribute__((ext_vector_type(4)));
    typedef O O4 __attribute__((ext_vector_type(4)));
    if (n == kClipChunk && aligned16(p) && aligned16(o)) {
        T4 v[kClipChunk / 1024];
#pragma unroll
        for (int k = 0; k < kClipChunk / 1024; ++k) v[k] = reinterpret_cast<const T4*>(p)[threadIdx.x + 256 * k];
#pragma unroll
        for (int k = 0; k < kClipChunk / 1024; ++k) {
            O4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (O)((float)v[k][e] * f);
            reinterpret_cast<O4*>(o)[threadIdx.x + 256 * k] = y;
        }
    } else {
        for (int e = threadIdx.x; e < n; e += 256) o[e] = (O)((float)p[e] * f);
    }
}

template <typename T>
__device__ __forceinline__ void scale_to(const T* p, void* o, size_t at, int len, int type, float f) {
    if (type == TOKEN_F32) scale_chunk(p + at, static_cast<float*>(o) + at, len, f);
    else if (type == TOKEN_BF16) scale_chunk(p + at, static_cast<__bf16*>(o) + at, len, f);
    else scale_chunk(p + at, static_cast<_Float16*>(o) + at, len, f);
}

__global__ __launch_bounds__(256) void k_clip_scale(const ClipTable t, const double* __restrict__ partial, int partials, float max_norm,
                                                    float eps, float* __restrict__ norm_out) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < partials; k += 256) sum += partial[k];
    const double norm = sqrt(block_sum(sum));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double ratio = (double)max_norm / (norm + (double)eps);
    const float f = ratio >= 1.0 ? 1.f : (float)ratio;  // (a norm that is no number scales to no number)
    // (backward: what the first pass read last may still be in the caches)
    each_chunk<true>(t, [&](int n, size_t at, int len, int type, int out_type) {
        if (f == 1.f && t.in[n] == t.out[n]) return;     // below the limit and in place: there is nothing to write
        if (type == TOKEN_F32) scale_to(static_cast<const float*>(t.in[n]), t.out[n], at, len, out_type, f);
        else if (type == TOKEN_BF16) scale_to(static_cast<const __bf16*>(t.in[n]), t.out[n], at, len, out_type, f);
        else scale_to(static_cast<const _Float16*>(t.in[n]), t.out[n], at, len, out_type, f);
    });
}

int clip_tables(int count) { return (count + kClipTensors - 1) / kClipTensors; }
int clip_blocks_each(int count) {  // workgroups of a launch
    const int tables = clip_tables(count);
    return tables <= 16 ? kClipBlocks / (tables > 0 ? tables : 1) : 128;
}

}  // namespace

size_t clip_gradients_workspace(int count) { return (size_t)clip_tables(count) * clip_blocks_each(count) * sizeof(double) + sizeof(double); }

hipError_t launch_clip_gradients(const void* const* in, void* const* out, const size_t* numel, const int* in_type, const int* out_type,
                                 int count, float max_norm, float eps, float* norm, void* workspace, hipStream_t stream) {
    const int most = clip_blocks_each(count);
    double* partial = static_cast<double*>(workspace);
    const bool only_norm = __builtin_isinf(max_norm);
    int partials = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int at = 0;
        bool told = false;
        for (int i = 0; i < count || (pass == 1 && !told);) {
            ClipTable t;
            t.count = 0;
            t.chunks = 0;
            for (; i < count && t.count < kClipTensors; ++i) {
                if (!numel[i]) continue;
                const size_t chunks = (numel[i] + kClipChunk - 1) / kClipChunk;
                t.in[t.count] = in[i];
                t.out[t.count] = out[i];
                t.first[t.count] = t.chunks;
                t.facts[t.count] = (unsigned)(numel[i] - (chunks - 1) * kClipChunk) | (unsigned)in_type[i] << 16 | (unsigned)out_type[i] << 20;
                t.chunks += (unsigned)chunks;
                ++t.count;
            }
            int blocks = t.chunks < (unsigned)most ? (int)t.chunks : most;
            if (blocks == 0 && pass == 0) continue;
            if (blocks == 0 || (pass == 1 && only_norm)) blocks = 1;
            t.each = (t.chunks + blocks - 1) / blocks;
            if (pass == 1 && only_norm) t.chunks = 0;  // (the norm alone is asked for)
            if (pass == 0) {
                DANRA_LAUNCH_KERNEL(k_clip_squares, dim3(blocks), dim3(256), 0, stream, t, partial + at);
                at += blocks;
            } else {
                DANRA_LAUNCH_KERNEL(k_clip_scale, dim3(blocks), dim3(256), 0, stream, t, partial, partials, max_norm, eps, told ? nullptr : norm);
                told = true;
                if (only_norm) break;
            }
        }
        if (pass == 0) partials = at;
    }
    return hipGetLastError();
}

}  // namespace danra
