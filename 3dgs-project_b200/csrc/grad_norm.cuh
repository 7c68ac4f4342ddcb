// grad_norm.cuh - the clip factor of a global gradient norm, shared by the kernels that apply it (grad_norm.cu's
// scaling kernel and the clipped Adam kernels in adam.cu), so that clipping first and stepping after gives the same
// bits as the step that clips.
//
// The norm of a long list is taken in two stages: each block of the norm kernel leaves one float64 partial (a sum of
// squares, a sum of absolute values, or a maximum) in the workspace, and one warp, of a kernel of its own or of every
// block that uses the norm, reduces the few hundred of them in an order that depends on their number only. A short list
// takes one launch, in which the blocks of a cluster exchange their partials.
//   norm = sqrt(sum), sum or max, rounded once to the caller's type (float32, or float64)
//   factor = min(1, max_norm / (norm + 1e-6)) in float64 from the rounded norm; NaN where the norm is NaN, or infinite
//            like max_norm
#pragma once

#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace splat {
namespace gradnorm {

constexpr int kTeam = 256;  // threads that read one chunk together
constexpr int kVecBytes = 16;
constexpr int kUnroll = 4;
constexpr int kChunkVecs = kTeam * kUnroll;
constexpr int kChunkBytes = kChunkVecs * kVecBytes;

constexpr int kMaxPartials = 1024;  // of one launch

// Lists of at most kSmallChunks chunks (1 MiB) take one launch: a cluster reads them all and adds its blocks' sums
// through distributed shared memory. Eight SMs are slower than all of them on the longer of these lists, but each launch
// saved is 3 us of the host's time. The norm of 43 chunks (3000 3D Gaussians): 5.0 us on the device and 9.8 us a call,
// against 3.5 and 12.7 in two launches. At 86 chunks clipping takes 12.3 us on the device and 16.0 a call, against 5.6
// and 15.7 in two: there the device has caught up with the host. In a captured graph, where the host's time does not
// count, the longer of these lists would be faster in two launches too; the rule does not look at captures.
constexpr int kSmallCluster = 8;
constexpr int kSmallThreads = 1024;
constexpr int kSmallChunks = 64;
constexpr int kSmallTensors = 64;

// Tables of up to 1000 tensors (29 KB of the 32764 bytes that a kernel's parameters may take); longer lists take
// several launches.
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

// Where the clip factor comes from: a norm in device memory, the caller's or one that the launch before computed, or
// (partials given) the partials of the launch before, which every block reduces for itself and block 0 stores as *norm.
struct Clip {
    void* norm;
    double max_norm;
    int norm_f64;  // *norm is float64
    int norm_type;
    int count;
    const double* partials;
};

// ---- programmatic dependent launch: the second kernel of a call starts while the first one drains ----

// Lets the kernel launched behind this one (as its dependent) start; it still waits for this one's results.
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Waits until the kernel this one depends on has finished and its writes are visible; returns at once in a kernel
// that was launched without such a dependence.
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Host: launches `kernel` on the stream, as a dependent of the kernel before it (which is one of the same call) when
// `dependent`, in clusters when `cluster` > 1.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), unsigned int grid, unsigned int threads, cudaStream_t st, bool dependent,
                   unsigned int cluster, const Args&... args) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cfg.attrs = attr;
    if (dependent) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- the norm ----

// NaN-propagating maximum of two values that are not negative.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

__device__ __forceinline__ double combine(double a, double b, int norm_type) {
    return norm_type == SPLAT_NORM_INF ? max_nan(a, b) : a + b;
}

__device__ __forceinline__ double warp_combine(double acc, int norm_type) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc = combine(acc, __shfl_xor_sync(kFullMask, acc, off), norm_type);
    return acc;
}

// The partials' total, by one warp, in an order that depends on their number only.
__device__ __forceinline__ double warp_total(const double* partials, int count, int norm_type) {
    double acc = 0.0;
    for (int i = threadIdx.x & 31; i < count; i += 32) acc = combine(acc, partials[i], norm_type);
    return warp_combine(acc, norm_type);
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

__device__ __forceinline__ double load_norm(const Clip& c) {
    return c.norm_f64 ? *static_cast<const double*>(c.norm) : static_cast<double>(*static_cast<const float*>(c.norm));
}

// The clip factor, in every thread of the block (which must call it as one), once the launch before has finished.
__device__ __forceinline__ double block_factor(const Clip& c) {
    __shared__ double s_factor;
    wait_for_primary();
    if (!c.partials) return factor_of(load_norm(c), c.max_norm);
    if (threadIdx.x < 32) {
        const double norm = rounded_norm(warp_total(c.partials, c.count, c.norm_type), c.norm_type, c.norm_f64);
        if (threadIdx.x == 0) {
            if (blockIdx.x == 0) store_norm(c, norm);
            s_factor = factor_of(norm, c.max_norm);
        }
    }
    __syncthreads();
    return s_factor;
}

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

// How soon the L2 lets go of the lines that a load brings in.
enum class Evict { kFirst, kNormal };

__device__ __forceinline__ uint64_t l2_policy(Evict e) {
    uint64_t p;
    if (e == Evict::kNormal)
        asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    else
        asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}

__device__ __forceinline__ uint4 load_hinted(const void* p, uint64_t policy) {
    uint4 v;
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p), "l"(policy));
    return v;
}

template <typename T>
union Vec {
    uint4 raw;
    T v[kVecBytes / sizeof(T)];
    __device__ Vec() {}
};

// Where a chunk's vectors lie: from the 16-byte boundary at or before the tensor's first element, which is `head`
// elements behind it; the tensor ends `end` elements behind the boundary.
template <typename T>
struct Span {
    static constexpr int V = kVecBytes / sizeof(T);
    int head;
    long long end, first;  // first: the chunk's first vector
    __device__ Span(const T* src, long long n, uint32_t chunk)
        : head(static_cast<int>((reinterpret_cast<uintptr_t>(src) & (kVecBytes - 1)) / sizeof(T))),
          end(n + head),
          first(static_cast<long long>(chunk) * kChunkVecs) {}
    __device__ bool whole() const { return (first > 0 || head == 0) && (first + kChunkVecs) * V <= end; }
    __device__ bool inside(long long e) const { return e >= head && e + V <= end; }
    // the first element of this thread's k-th vector, counted from the boundary
    __device__ long long element(int k, int thread) const { return (first + k * kTeam + thread) * V; }
};

// Adds the chunk's elements, read by kTeam threads (`thread` of them is this one).
template <typename T, int NORM>
__device__ __forceinline__ void accumulate(const T* src, long long n, uint32_t chunk, int thread, uint64_t policy,
                                           double& acc) {
    constexpr int V = Span<T>::V;
    const Span<T> s(src, n, chunk);
    const T* base = src - s.head;
    if (s.whole()) {
        Vec<T> x[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) x[k].raw = load_hinted(base + s.element(k, thread), policy);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) add<NORM>(acc, widen(x[k].v[j]));
    } else {
        // the tensor's first or last chunk: the vectors inside it, all loaded before any is used (zeros add nothing),
        // then the elements of the one or two that it ends in
        Vec<T> x[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            x[k].raw = s.inside(s.element(k, thread)) ? load_hinted(base + s.element(k, thread), policy)
                                                      : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) add<NORM>(acc, widen(x[k].v[j]));
#pragma unroll 1
        for (int k = 0; k < kUnroll; ++k) {
            const long long e = s.element(k, thread);
            if (s.inside(e) || e >= s.end || e + V <= s.head) continue;
#pragma unroll 1
            for (int j = 0; j < V; ++j)
                if (e + j >= s.head && e + j < s.end) add<NORM>(acc, widen(base[e + j]));
        }
    }
}

// This thread's share of the sum over chunks team, team + teams, ... of the table. With `keep`, all but the last so many
// chunks leave the L2 first, so that those are still there for the pass that follows.
template <int CAP, int NORM>
__device__ __forceinline__ double accumulate_table(const Table<CAP>& t, uint32_t team, uint32_t teams, int thread,
                                                   uint32_t keep) {
    double acc = 0.0;
    for (uint32_t c = team; c < t.chunks; c += teams) {
        const int k = tensor_of(t, c);
        const uint32_t chunk = c - t.first_chunk[k];
        const void* src = t.src[k];
        const uint64_t policy =
            l2_policy(keep == 0 || t.chunks - c <= keep ? Evict::kNormal : Evict::kFirst);
        switch (t.dtype[k]) {
            case SPLAT_F32:
                accumulate<float, NORM>(static_cast<const float*>(src), t.n[k], chunk, thread, policy, acc);
                break;
            case SPLAT_BF16:
                accumulate<__nv_bfloat16, NORM>(static_cast<const __nv_bfloat16*>(src), t.n[k], chunk, thread, policy,
                                                acc);
                break;
            case SPLAT_F16:
                accumulate<__half, NORM>(static_cast<const __half*>(src), t.n[k], chunk, thread, policy, acc);
                break;
            default:
                accumulate<double, NORM>(static_cast<const double*>(src), t.n[k], chunk, thread, policy, acc);
                break;
        }
    }
    return acc;
}

// The block's total of `acc`, in thread 0.
template <int THREADS, int NORM>
__device__ __forceinline__ double block_total(double acc) {
    __shared__ double s_warp[THREADS / 32];
    acc = warp_combine(acc, NORM);
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x < 32) {
        acc = threadIdx.x < THREADS / 32 ? s_warp[threadIdx.x] : 0.0;
        acc = warp_combine(acc, NORM);
    }
    return acc;
}

// The norm of a small table, in every thread of every block of the cluster (kSmallCluster blocks of kSmallThreads
// threads, which must all call it): every cluster that calls it gets the same bits. On return every block of the
// cluster has read its share of the table.
template <int CAP, int NORM>
__device__ __forceinline__ double cluster_norm(const Table<CAP>& t, int norm_f64) {
    namespace cg = cooperative_groups;
    __shared__ double s_block, s_norm;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int kTeams = kSmallThreads / kTeam;
    const uint32_t rank = cluster.block_rank();
    double acc = accumulate_table<CAP, NORM>(t, rank * kTeams + threadIdx.x / kTeam, kSmallCluster * kTeams,
                                             threadIdx.x % kTeam, 0u);
    acc = block_total<kSmallThreads, NORM>(acc);
    if (threadIdx.x == 0) s_block = acc;
    cluster.sync();
    if (threadIdx.x < 32) {
        acc = threadIdx.x < kSmallCluster ? *cluster.map_shared_rank(&s_block, threadIdx.x) : 0.0;
        acc = warp_combine(acc, NORM);
        if (threadIdx.x == 0) s_norm = rounded_norm(acc, NORM, norm_f64);
    }
    cluster.sync();  // no block leaves while another reads its sum
    return s_norm;
}

// ---- host ----

// A norm kind's code is known.
inline bool known_norm(int norm_type) {
    return norm_type == SPLAT_NORM_INF || norm_type == SPLAT_NORM_L1 || norm_type == SPLAT_NORM_L2;
}

inline int size_of(int dtype) { return dtype == SPLAT_F32 ? 4 : dtype == SPLAT_F64 ? 8 : 2; }

// A buffer of float32 or float64 values that is there.
inline bool aligned(const void* p, bool f64) { return p && reinterpret_cast<uintptr_t>(p) % (f64 ? 8 : 4) == 0; }

// A buffer of a call: its first byte's address, doubled, with whether the call writes it in the lowest bit (addresses
// have fewer than 63 bits), and the address behind its last byte.
struct Range {
    uint64_t begin, end;
};

inline Range range_of(const void* p, unsigned long long bytes, bool written) {
    const uint64_t at = reinterpret_cast<uintptr_t>(p);
    return {at << 1 | (written ? 1u : 0u), at + bytes};
}

// No range that is written overlaps another one. Sorts them.
inline bool apart(Range* s, int count) {
    std::sort(s, s + count, [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uint64_t to[2] = {0, 0};  // where the ranges so far end that are read, that are written
    for (int i = 0; i < count; ++i) {
        const uint64_t begin = s[i].begin >> 1;
        const bool written = s[i].begin & 1;
        if (begin < to[1] || (written && begin < to[0])) return false;
        to[written] = std::max(to[written], s[i].end);
    }
    return true;
}

inline long long chunks_of(const void* src, long long n, int dtype) {
    const uintptr_t head = reinterpret_cast<uintptr_t>(src) & (kVecBytes - 1);
    return (static_cast<long long>(head) + n * size_of(dtype) + kChunkBytes - 1) / kChunkBytes;
}

// Fills the table from tensor `from` on, skipping empty ones; returns the first tensor that did not fit. The list's
// chunks fit 32 bits (checked by the entry points).
template <int CAP>
int fill(Table<CAP>& t, int from, int count, const void* const* src, void* const* dst, const long long* n,
         const unsigned char* dtypes) {
    t.count = 0;
    long long chunks = 0;
    int i = from;
    for (; i < count && t.count < CAP; ++i) {
        if (n[i] == 0) continue;
        t.src[t.count] = src[i];
        t.dst[t.count] = dst ? dst[i] : nullptr;
        t.n[t.count] = n[i];
        t.dtype[t.count] = dtypes[i];
        t.first_chunk[t.count++] = static_cast<uint32_t>(chunks);
        chunks += chunks_of(src[i], n[i], dtypes[i]);
    }
    t.chunks = static_cast<uint32_t>(chunks);
    return i;
}

// The statement with NORM a constant for the norm's code.
#define SPLAT_FOR_NORM(norm_type, NORM, ...)                                  \
    do {                                                                      \
        if ((norm_type) == SPLAT_NORM_L2) {                                   \
            constexpr int NORM = SPLAT_NORM_L2;                               \
            __VA_ARGS__;                                                      \
        } else if ((norm_type) == SPLAT_NORM_L1) {                            \
            constexpr int NORM = SPLAT_NORM_L1;                               \
            __VA_ARGS__;                                                      \
        } else {                                                              \
            constexpr int NORM = SPLAT_NORM_INF;                              \
            __VA_ARGS__;                                                      \
        }                                                                     \
    } while (0)

// A list whose norm takes one launch (also an empty one).
inline bool is_small(int count, const void* const* grads, const long long* n, const unsigned char* dtypes) {
    if (count > kSmallTensors) return false;
    long long chunks = 0;
    for (int i = 0; i < count; ++i)
        if (n[i] > 0) chunks += chunks_of(grads[i], n[i], dtypes[i]);
    return chunks <= kSmallChunks;
}

enum class Again { kNo, kInPlace, kAll };

// The norm of a list that is not small, stored as `c` says (grad_norm.cu). Arguments already checked. The kernel that
// uses it can be launched as a dependent. again: it reads all of the list again, is to find the end in the L2, and takes
// its factor with block_factor(), for which a list of middling length leaves the partials in `c`.
int enqueue_norm(int count, const void* const* grads, const long long* n, const unsigned char* dtypes, int norm_type,
                 double* partials, Clip& c, Again again, cudaStream_t stream);

}  // namespace gradnorm
}  // namespace splat
