// grad_norm.cu - the global norm over a list of gradient tensors, and the tensors scaled by the clip factor.
//
//   norm = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|, over every element of every tensor
//   out  = g * min(1, max_norm / (norm + 1e-6))
// The tensors (float32, bfloat16, float16 or float64, mixed) are described by a table passed by value and cut into
// chunks of 16 KiB from the 16-byte boundary at or before their first element, so that all but the first and the last
// 16 bytes of a tensor move as 16-byte vectors wherever it starts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <memory>
#include <new>

#include "grad_norm.cuh"

namespace splat {
namespace gradnorm {

constexpr int kThreads = 256;
constexpr int kVecBytes = 16;
constexpr int kUnroll = 4;
constexpr int kChunkVecs = kThreads * kUnroll;
constexpr int kChunkBytes = kChunkVecs * kVecBytes;

// Tables of up to 1000 tensors (29 KB of the 32764 bytes a kernel's parameters may take); longer lists take several
// launches.
constexpr int kTableMax = 1000;

template <int CAP>
struct Table {
    const void* src[CAP];
    void* dst[CAP];
    long long n[CAP];
    uint32_t first_chunk[CAP];  // prefix of chunks over the tensors
    uint8_t dtype[CAP];
    int count;
    uint32_t chunks;
};

// The tensor that a chunk belongs to: the last one whose first chunk is not behind it (empty tensors are not in the
// table).
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, uint32_t chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first_chunk[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double widen(float x) { return static_cast<double>(x); }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ double widen(__nv_bfloat16 x) { return static_cast<double>(__bfloat162float(x)); }
__device__ __forceinline__ double widen(__half x) { return static_cast<double>(__half2float(x)); }

template <int NORM>
__device__ __forceinline__ void add(double& acc, double g) {
    if (NORM == SPLAT_NORM_L2)
        acc = fma(g, g, acc);
    else if (NORM == SPLAT_NORM_L1)
        acc += fabs(g);
    else
        acc = max_nan(acc, fabs(g));
}

__device__ __forceinline__ float scaled(float g, double f) { return g * static_cast<float>(f); }
__device__ __forceinline__ double scaled(double g, double f) { return g * f; }
// The product in float32, rounded once more to the tensor's type.
__device__ __forceinline__ __nv_bfloat16 scaled(__nv_bfloat16 g, double f) {
    return __float2bfloat16_rn(__bfloat162float(g) * static_cast<float>(f));
}
__device__ __forceinline__ __half scaled(__half g, double f) {
    return __float2half_rn(__half2float(g) * static_cast<float>(f));
}

template <typename T>
union Vec {
    uint4 raw;
    T v[kVecBytes / sizeof(T)];
    __device__ Vec() {}
};

// Elements [e, e + V) of the chunk's k-th vector of this thread, counted from the boundary `base`; `head` of the first
// vector's elements lie before the tensor, and it ends at `end`.
template <typename T, int NORM>
__device__ __forceinline__ void accumulate(const T* src, long long n, uint32_t chunk, double& acc) {
    constexpr int V = kVecBytes / sizeof(T);
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(src) & (kVecBytes - 1)) / sizeof(T));
    const T* base = src - head;
    const long long end = n + head;
    const long long first = static_cast<long long>(chunk) * kChunkVecs;
    if ((first > 0 || head == 0) && (first + kChunkVecs) * V <= end) {  // the whole chunk lies inside
        Vec<T> x[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            x[k].raw = reinterpret_cast<const uint4*>(base)[first + k * kThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) add<NORM>(acc, widen(x[k].v[j]));
    } else {
        for (int k = 0; k < kUnroll; ++k) {
            const long long e = (first + k * kThreads + threadIdx.x) * V;
            if (e >= head && e + V <= end) {
                Vec<T> x;
                x.raw = *reinterpret_cast<const uint4*>(base + e);
#pragma unroll
                for (int j = 0; j < V; ++j) add<NORM>(acc, widen(x.v[j]));
            } else {
                for (int j = 0; j < V; ++j)
                    if (e + j >= head && e + j < end) add<NORM>(acc, widen(base[e + j]));
            }
        }
    }
}

template <int CAP, int NORM>
__global__ void __launch_bounds__(kThreads) k_norm_partials(const __grid_constant__ Table<CAP> t, double* partials) {
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const uint32_t chunk = c - t.first_chunk[k];
        switch (t.dtype[k]) {
            case SPLAT_F32: accumulate<float, NORM>(static_cast<const float*>(t.src[k]), t.n[k], chunk, acc); break;
            case SPLAT_BF16:
                accumulate<__nv_bfloat16, NORM>(static_cast<const __nv_bfloat16*>(t.src[k]), t.n[k], chunk, acc);
                break;
            case SPLAT_F16: accumulate<__half, NORM>(static_cast<const __half*>(t.src[k]), t.n[k], chunk, acc); break;
            default: accumulate<double, NORM>(static_cast<const double*>(t.src[k]), t.n[k], chunk, acc); break;
        }
    }
    __shared__ double s_warp[kThreads / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc = combine(acc, __shfl_xor_sync(kFullMask, acc, off), NORM);
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; ++w) acc = combine(acc, s_warp[w], NORM);
        partials[blockIdx.x] = acc;
    }
}

__global__ void __launch_bounds__(32) k_norm_finish(Clip c) {
    const double norm = rounded_norm(warp_total(c.partials, c.count, c.norm_type), c.norm_type, c.norm_f64);
    if (threadIdx.x == 0) store_norm(c, norm);
}

// Writes the tensor's scaled chunk; src and dst are the same, or do not overlap.
template <typename T>
__device__ __forceinline__ void scale_chunk(const T* src, T* dst, long long n, uint32_t chunk, double f) {
    constexpr int V = kVecBytes / sizeof(T);
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(src) & (kVecBytes - 1)) / sizeof(T));
    const bool vec = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & (kVecBytes - 1)) == 0;
    const T* base = src - head;
    T* out = dst - head;
    const long long end = n + head;
    const long long first = static_cast<long long>(chunk) * kChunkVecs;
    for (int k = 0; k < kUnroll; ++k) {
        const long long e = (first + k * kThreads + threadIdx.x) * V;
        if (e >= head && e + V <= end) {
            Vec<T> x;
            x.raw = *reinterpret_cast<const uint4*>(base + e);
#pragma unroll
            for (int j = 0; j < V; ++j) x.v[j] = scaled(x.v[j], f);
            if (vec) {
                *reinterpret_cast<uint4*>(out + e) = x.raw;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) out[e + j] = x.v[j];
            }
        } else {
            for (int j = 0; j < V; ++j)
                if (e + j >= head && e + j < end) out[e + j] = scaled(base[e + j], f);
        }
    }
}

template <int CAP>
__global__ void __launch_bounds__(kThreads)
    k_clip_scale(const __grid_constant__ Table<CAP> t, const __grid_constant__ Clip c, int in_place, int store) {
    const double f = block_factor(c, store != 0);
    if (in_place && f == 1.0) return;  // x * 1 is x, NaN and infinities too
    for (uint32_t i = blockIdx.x; i < t.chunks; i += gridDim.x) {
        const int k = tensor_of(t, i);
        const uint32_t chunk = i - t.first_chunk[k];
        switch (t.dtype[k]) {
            case SPLAT_F32:
                scale_chunk(static_cast<const float*>(t.src[k]), static_cast<float*>(t.dst[k]), t.n[k], chunk, f);
                break;
            case SPLAT_BF16:
                scale_chunk(static_cast<const __nv_bfloat16*>(t.src[k]), static_cast<__nv_bfloat16*>(t.dst[k]), t.n[k],
                            chunk, f);
                break;
            case SPLAT_F16:
                scale_chunk(static_cast<const __half*>(t.src[k]), static_cast<__half*>(t.dst[k]), t.n[k], chunk, f);
                break;
            default:
                scale_chunk(static_cast<const double*>(t.src[k]), static_cast<double*>(t.dst[k]), t.n[k], chunk, f);
                break;
        }
    }
}

int size_of(int dtype) { return dtype == SPLAT_F32 ? 4 : dtype == SPLAT_F64 ? 8 : 2; }

// Fills the table from tensor `from` on, skipping empty ones; returns the first tensor that did not fit.
template <int CAP>
int fill(Table<CAP>& t, int from, int count, const void* const* src, void* const* dst, const long long* n,
         const unsigned char* dtypes) {
    t.count = 0;
    long long chunks = 0;
    int i = from;
    for (; i < count && t.count < CAP; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t head = reinterpret_cast<uintptr_t>(src[i]) & (kVecBytes - 1);
        const long long mine = (static_cast<long long>(head) + n[i] * size_of(dtypes[i]) + kChunkBytes - 1) / kChunkBytes;
        if (chunks + mine >= (1ll << 32)) break;  // not reached by what a device holds (64 TB)
        t.src[t.count] = src[i];
        t.dst[t.count] = dst ? dst[i] : nullptr;
        t.n[t.count] = n[i];
        t.dtype[t.count] = dtypes[i];
        t.first_chunk[t.count++] = static_cast<uint32_t>(chunks);
        chunks += mine;
    }
    t.chunks = static_cast<uint32_t>(chunks);
    return i;
}

template <int CAP>
void launch_partials(const Table<CAP>& t, int norm_type, double* partials, unsigned int grid, cudaStream_t st) {
    if (norm_type == SPLAT_NORM_L2)
        k_norm_partials<CAP, SPLAT_NORM_L2><<<grid, kThreads, 0, st>>>(t, partials);
    else if (norm_type == SPLAT_NORM_L1)
        k_norm_partials<CAP, SPLAT_NORM_L1><<<grid, kThreads, 0, st>>>(t, partials);
    else
        k_norm_partials<CAP, SPLAT_NORM_INF><<<grid, kThreads, 0, st>>>(t, partials);
    note_launch();
}

template <int CAP>
int partials_of(int count, const void* const* grads, const long long* n, const unsigned char* dtypes, int norm_type,
                double* partials, int* partial_count, cudaStream_t st) {
    Table<CAP> t;
    int used = 0;
    for (int i = 0; i < count;) {
        i = fill(t, i, count, grads, nullptr, n, dtypes);
        if (t.count == 0) break;
        const unsigned int grid = std::min<unsigned int>(t.chunks, std::min(8 * sm_count(), kMaxPartials));
        launch_partials(t, norm_type, partials + used, grid, st);
        used += static_cast<int>(grid);
        SPLAT_TRY(check_launch("gradient norm"));
    }
    *partial_count = used;
    return SPLAT_OK;
}

int enqueue_partials(int count, const void* const* grads, const long long* n, const unsigned char* dtypes,
                     int norm_type, double* partials, int* partial_count, cudaStream_t st) {
    if (count <= 16) return partials_of<16>(count, grads, n, dtypes, norm_type, partials, partial_count, st);
    if (count <= 128) return partials_of<128>(count, grads, n, dtypes, norm_type, partials, partial_count, st);
    return partials_of<kTableMax>(count, grads, n, dtypes, norm_type, partials, partial_count, st);
}

template <int CAP>
int scale_all(int count, const void* const* grads, void* const* outs, const long long* n, const unsigned char* dtypes,
              const Clip& c, int in_place, cudaStream_t st) {
    Table<CAP> t;
    bool stored = false;
    for (int i = 0; i < count;) {
        i = fill(t, i, count, grads, outs, n, dtypes);
        if (t.count == 0) break;
        const unsigned int grid = std::min<unsigned int>(t.chunks, 8 * sm_count());
        k_clip_scale<CAP><<<grid, kThreads, 0, st>>>(t, c, in_place, stored ? 0 : 1);
        stored = true;
        note_launch();
        SPLAT_TRY(check_launch("splat_grad_clip"));
    }
    return SPLAT_OK;
}

int check_list(const char* what, int count, const void* const* grads, const long long* n,
               const unsigned char* dtypes, int norm_f64) {
    SPLAT_REQUIRE(count >= 0, "%s: negative count", what);
    SPLAT_REQUIRE(count == 0 || (grads && n && dtypes), "%s: the list of tensors is missing", what);
    for (int i = 0; i < count; ++i) {
        SPLAT_REQUIRE(n[i] >= 0, "%s: tensor %d has negative size", what, i);
        SPLAT_REQUIRE(dtypes[i] <= SPLAT_F64, "%s: tensor %d has an unknown type", what, i);
        SPLAT_REQUIRE(dtypes[i] != SPLAT_F64 || norm_f64, "%s: tensor %d is float64, the norm is not", what, i);
        if (n[i] == 0) continue;
        SPLAT_REQUIRE(grads[i], "%s: tensor %d has a null buffer", what, i);
        SPLAT_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % size_of(dtypes[i]) == 0,
                      "%s: tensor %d is not aligned to its type", what, i);
    }
    return SPLAT_OK;
}

struct Span {
    uintptr_t begin, end;
    bool written;
};

// What is written overlaps nothing else: the outputs one another, or (out of place) any input.
int check_overlap(int count, const void* const* grads, void* const* outs, const long long* n,
                  const unsigned char* dtypes, bool in_place) {
    std::unique_ptr<Span[]> s(new (std::nothrow) Span[2 * static_cast<size_t>(count)]);
    SPLAT_REQUIRE(s, "splat_grad_clip: out of host memory");
    int k = 0;
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t bytes = static_cast<uintptr_t>(n[i]) * size_of(dtypes[i]);
        const uintptr_t o = reinterpret_cast<uintptr_t>(outs[i]), g = reinterpret_cast<uintptr_t>(grads[i]);
        s[k++] = {o, o + bytes, true};
        if (!in_place) s[k++] = {g, g + bytes, false};
    }
    std::sort(s.get(), s.get() + k, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t written_to = 0, read_to = 0;
    for (int i = 0; i < k; ++i) {
        SPLAT_REQUIRE(s[i].begin >= written_to && (!s[i].written || s[i].begin >= read_to),
                      "splat_grad_clip: a tensor that is written overlaps another tensor of the call");
        uintptr_t& to = s[i].written ? written_to : read_to;
        to = std::max(to, s[i].end);
    }
    return SPLAT_OK;
}

size_t partial_bytes(int count) {
    const size_t launches = count <= 0 ? 1 : (static_cast<size_t>(count) + kTableMax - 1) / kTableMax;
    return launches * kMaxPartials * sizeof(double);
}

}  // namespace gradnorm
}  // namespace splat

using namespace splat;

extern "C" {

size_t splat_grad_workspace_size(int count) { return gradnorm::partial_bytes(count); }

int splat_grad_norm(int count, const void* const* grads, const long long* n, const unsigned char* dtypes, int norm_type,
                    void* norm, int norm_is_f64, void* workspace, size_t workspace_bytes, void* stream) {
    SPLAT_TRY(gradnorm::check_list("splat_grad_norm", count, grads, n, dtypes, norm_is_f64));
    SPLAT_REQUIRE(gradnorm::known_norm(norm_type), "splat_grad_norm: unknown norm type %d", norm_type);
    SPLAT_REQUIRE(norm, "splat_grad_norm: the norm's buffer is missing");
    SPLAT_REQUIRE(workspace && workspace_bytes >= gradnorm::partial_bytes(count),
                  "splat_grad_norm: workspace too small");
    gradnorm::Clip c{static_cast<const double*>(workspace), 0, norm_type, 0, norm_is_f64, norm, 0.0};
    SPLAT_TRY(gradnorm::enqueue_partials(count, grads, n, dtypes, norm_type, static_cast<double*>(workspace), &c.count,
                                         as_stream(stream)));
    gradnorm::k_norm_finish<<<1, 32, 0, as_stream(stream)>>>(c);
    note_launch();
    return check_launch("splat_grad_norm");
}

int splat_grad_clip(int count, const void* const* grads, void* const* outs, const long long* n,
                    const unsigned char* dtypes, int norm_type, double max_norm, void* norm, int norm_is_f64,
                    void* workspace, size_t workspace_bytes, void* stream) {
    SPLAT_TRY(gradnorm::check_list("splat_grad_clip", count, grads, n, dtypes, norm_is_f64));
    SPLAT_REQUIRE(norm_type == SPLAT_NORM_GIVEN || gradnorm::known_norm(norm_type),
                  "splat_grad_clip: unknown norm type %d", norm_type);
    SPLAT_REQUIRE(max_norm >= 0.0, "splat_grad_clip: max_norm must not be negative");
    SPLAT_REQUIRE(norm, "splat_grad_clip: the norm's buffer is missing");
    const bool given = norm_type == SPLAT_NORM_GIVEN;
    SPLAT_REQUIRE(given || (workspace && workspace_bytes >= gradnorm::partial_bytes(count)),
                  "splat_grad_clip: workspace too small");
    SPLAT_REQUIRE(count == 0 || outs, "splat_grad_clip: the list of outputs is missing");
    int same = 0, other = 0;
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        SPLAT_REQUIRE(outs[i], "splat_grad_clip: output %d is null", i);
        SPLAT_REQUIRE(reinterpret_cast<uintptr_t>(outs[i]) % gradnorm::size_of(dtypes[i]) == 0,
                      "splat_grad_clip: output %d is not aligned to its type", i);
        ++(outs[i] == grads[i] ? same : other);
    }
    SPLAT_REQUIRE(same == 0 || other == 0, "splat_grad_clip: some tensors are clipped in place, others are not");
    SPLAT_TRY(gradnorm::check_overlap(count, grads, outs, n, dtypes, same > 0));
    gradnorm::Clip c{static_cast<const double*>(workspace), 0, norm_type, given, norm_is_f64, norm, max_norm};
    const cudaStream_t st = as_stream(stream);
    if (!given) {
        SPLAT_TRY(gradnorm::enqueue_partials(count, grads, n, dtypes, norm_type, static_cast<double*>(workspace),
                                             &c.count, st));
        if (same + other == 0) {  // nothing to scale: the norm (0) is still the call's
            gradnorm::k_norm_finish<<<1, 32, 0, st>>>(c);
            note_launch();
            return check_launch("splat_grad_clip");
        }
    }
    if (count <= 16) return gradnorm::scale_all<16>(count, grads, outs, n, dtypes, c, same > 0, st);
    if (count <= 128) return gradnorm::scale_all<128>(count, grads, outs, n, dtypes, c, same > 0, st);
    return gradnorm::scale_all<gradnorm::kTableMax>(count, grads, outs, n, dtypes, c, same > 0, st);
}

}  // extern "C"
