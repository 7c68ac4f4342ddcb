// grad_norm.cuh - the clip factor of a global gradient norm, shared by the kernels that apply it (grad_norm.cu's
// scaling kernel and the clipped Adam kernels in adam.cu), so that clipping first and stepping after gives the same
// bits as the step that clips.
//
// The norm is taken in two stages. Each block of the norm kernel leaves one float64 partial (a sum of squares, a sum
// of absolute values, or a maximum) in the workspace; every block of the kernel that follows reduces the same few
// hundred partials in the same order, so no block waits for another and no atomic decides an order.
//   norm = sqrt(sum), sum or max, rounded once to the caller's type (float32, or float64)
//   factor = min(1, max_norm / (norm + 1e-6)) in float64 from the rounded norm; NaN where the norm is NaN
#pragma once

#include "common.cuh"

namespace splat {
namespace gradnorm {

constexpr int kMaxPartials = 1024;  // of one launch

struct Clip {
    const double* partials;  // of the norm kernel; not read when `given`
    int count;               // partials
    int norm_type;
    int given;     // the norm is the caller's, read from *norm
    int norm_f64;  // *norm is float64
    void* norm;
    double max_norm;
};

// NaN-propagating maximum of two values that are not negative.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

__device__ __forceinline__ double combine(double a, double b, int norm_type) {
    return norm_type == SPLAT_NORM_INF ? max_nan(a, b) : a + b;
}

// The partials' total, by one warp, in an order that depends on their number only.
__device__ __forceinline__ double warp_total(const double* partials, int count, int norm_type) {
    double acc = 0.0;
    for (int i = threadIdx.x & 31; i < count; i += 32) acc = combine(acc, partials[i], norm_type);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc = combine(acc, __shfl_xor_sync(kFullMask, acc, off), norm_type);
    return acc;
}

// The norm as the caller reads it: rounded to its type.
__device__ __forceinline__ double rounded_norm(double total, int norm_type, int norm_f64) {
    const double norm = norm_type == SPLAT_NORM_L2 ? sqrt(total) : total;
    return norm_f64 ? norm : static_cast<double>(static_cast<float>(norm));
}

__device__ __forceinline__ void store_norm(const Clip& c, double norm) {
    if (c.norm_f64)
        *static_cast<double*>(c.norm) = norm;
    else
        *static_cast<float*>(c.norm) = static_cast<float>(norm);
}

__device__ __forceinline__ double factor_of(double norm, double max_norm) {
    const double f = max_norm / (norm + 1e-6);
    return f < 1.0 || f != f ? f : 1.0;
}

// The factor, in every thread of the block (which must call it as one); block 0 stores the norm it computed when
// `store`.
__device__ __forceinline__ double block_factor(const Clip& c, bool store) {
    __shared__ double s_factor;
    if (threadIdx.x < 32) {
        double norm;
        if (c.given) {
            norm = c.norm_f64 ? *static_cast<const double*>(c.norm)
                              : static_cast<double>(*static_cast<const float*>(c.norm));
        } else {
            norm = rounded_norm(warp_total(c.partials, c.count, c.norm_type), c.norm_type, c.norm_f64);
            if (store && blockIdx.x == 0 && threadIdx.x == 0) store_norm(c, norm);
        }
        if (threadIdx.x == 0) s_factor = factor_of(norm, c.max_norm);
    }
    __syncthreads();
    return s_factor;
}

// Host: a norm kind's code is known.
inline bool known_norm(int norm_type) {
    return norm_type == SPLAT_NORM_INF || norm_type == SPLAT_NORM_L1 || norm_type == SPLAT_NORM_L2;
}

// Host: partials of the tensors in `workspace` (grad_norm.cu); *count of them. Arguments already checked.
int enqueue_partials(int count, const void* const* grads, const long long* n, const unsigned char* dtypes,
                     int norm_type, double* partials, int* partial_count, cudaStream_t stream);

}  // namespace gradnorm
}  // namespace splat
