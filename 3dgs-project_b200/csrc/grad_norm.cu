// grad_norm.cu - the global norm over a list of gradient tensors, and the tensors scaled by the clip factor.
//
//   norm = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|, over every element of every tensor
//   out  = g * min(1, max_norm / (norm + 1e-6))
// The tensors (float32, bfloat16, float16 or float64, mixed) are described by a table passed by value and cut into
// chunks of 16 KiB from the 16-byte boundary at or before their first element, so that all but the first and the last
// 16 bytes of a tensor move as 16-byte vectors wherever it starts.
//
// The norm reads everything once and is bound by HBM: 102 us for the 708 MB of 3M Gaussians' gradients (6.9 TB/s, 1.06
// of the measured copy rate; with lines that leave the L2 first, as a call that reads on wants them, 105). Squares are
// added in float64, which keeps float32's whole range (a square of 1e-25 or 1e25 leaves it) and every bit of the result;
// it costs a conversion and a float64 multiply-add an element, hidden behind the loads at 32 registers and all 64 warps
// of an SM (46 registers, for looking the next chunk up while this one loads, cost 1% on 3M Gaussians and 13% on a ragged
// 16-bit list). Teams take every teams-th chunk: neighbouring chunks a team, with one search for the tensor, took 109 us.
// A list of 300 16-bit tensors (91 MB) takes 23 us, with 64% of the issue slots busy: the 32 elements that a thread adds
// of a chunk carry the search and the chunk's geometry, and a conversion each. Which of these costs what is not known.
//
// Clipping reads the gradients again, since the factor needs all of them: 1M Gaussians (236 MB) clipped into other
// buffers move 3 x 236 MB less the 64 MiB that the norm's pass leaves in the L2 and take 111.3 us (644 MB in 98 us would
// be the copy rate); where it leaves nothing there in particular 114.5.
#include <algorithm>
#include <memory>
#include <new>

#include "grad_norm.cuh"

namespace splat {
namespace gradnorm {

constexpr int kNormThreads = 512;
constexpr int kNormBlocks = 4;  // per SM: all its threads
// What the norm's pass leaves in the L2 for a second one: 64 MiB of its 126 MB (32 MiB: 113.2 us for the 1M Gaussians
// above, 96 MiB: 111.6, 64 MiB: 111.3). Those lines have the normal priority and the ones before them leave first. Lines
// of the highest priority serve the second pass no better (111.7; the dense step of 3M Gaussians 854 us against 858), and
// stay when the call is over: every later pass over 80 MB took 20 us where it takes 16.5, until gigabytes had gone by.
constexpr uint32_t kKeepChunks = 4096;
// Lists of up to 2048 chunks (32 MiB) leave the partials to the blocks that scale or step, each of which reduces them
// for itself: one launch less, 3 us of the host's time, and on the device 6.5 against 7.4 us for clipping 20 thousand
// 3D Gaussians' gradients and 31.9 against 32.6 for the step of 100 thousand (1444 chunks). Longer lists have too many
// blocks for that: the lean step of 1M Gaussians (14408 chunks) takes 214 us so and 207 after k_norm_finish. Between
// these two lengths nothing was measured.
constexpr long long kDirectChunks = 2048;
constexpr int kScaleThreads = kTeam;
// Out of place a block scales one chunk: a resident grid that loops took 84 us where this takes 72 (1M Gaussians, 236 MB
// read and written). In place most calls find a factor of 1 and end there, and blocks that only end cost time too: with
// 8 chunks a block the call over 3M Gaussians takes 105 us when nothing changes and 343 when something does; with 1 it
// was 19 us slower when nothing changes, with 32 the scaling took 235 us instead of 225.
constexpr unsigned int kScaleChunksInPlace = 8;
constexpr unsigned int kScaleBlocks = 8;  // per SM, that a short list is spread over all the same

__device__ __forceinline__ float scaled(float g, double f) { return g * static_cast<float>(f); }
__device__ __forceinline__ double scaled(double g, double f) { return g * f; }
// The product in float32, rounded once more to the tensor's type.
__device__ __forceinline__ __nv_bfloat16 scaled(__nv_bfloat16 g, double f) {
    return __float2bfloat16_rn(__bfloat162float(g) * static_cast<float>(f));
}
__device__ __forceinline__ __half scaled(__half g, double f) {
    return __float2half_rn(__half2float(g) * static_cast<float>(f));
}

template <int CAP, int NORM>
__global__ void __launch_bounds__(kNormThreads)
    k_norm_partials(const __grid_constant__ Table<CAP> t, double* partials, uint32_t keep) {
    release_dependents();  // once every block has started, the next kernels' launches overlap this one's work
    constexpr int kTeams = kNormThreads / kTeam;
    double acc = accumulate_table<CAP, NORM>(t, blockIdx.x * kTeams + threadIdx.x / kTeam, gridDim.x * kTeams,
                                             threadIdx.x % kTeam, keep);
    acc = block_total<kNormThreads, NORM>(acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// One warp reduces the partials, for a norm alone or a long list.
__global__ void __launch_bounds__(32) k_norm_finish(const double* partials, int count, int norm_type, Clip c) {
    release_dependents();
    wait_for_primary();
    const double norm = rounded_norm(warp_total(partials, count, norm_type), norm_type, c.norm_f64);
    if (threadIdx.x == 0) store_norm(c, norm);
}

// Writes the tensor's scaled chunk; src and dst are the same, or do not overlap.
template <typename T>
__device__ __forceinline__ void scale_chunk(const T* src, T* dst, long long n, uint32_t chunk, int thread, double f) {
    constexpr int V = Span<T>::V;
    const Span<T> s(src, n, chunk);
    const bool vec = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & (kVecBytes - 1)) == 0;
    const T* base = src - s.head;
    T* out = dst - s.head;
    const uint64_t policy = l2_policy(Evict::kFirst);  // what the norm's pass kept is done with
    if (s.whole() && vec) {
        Vec<T> x[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) x[k].raw = load_hinted(base + s.element(k, thread), policy);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[k].v[j] = scaled(x[k].v[j], f);
            *reinterpret_cast<uint4*>(out + s.element(k, thread)) = x[k].raw;
        }
    } else {
        for (int k = 0; k < kUnroll; ++k) {
            const long long e = s.element(k, thread);
            if (e >= s.head && e + V <= s.end) {
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
                    if (e + j >= s.head && e + j < s.end) out[e + j] = scaled(base[e + j], f);
            }
        }
    }
}

// Scales the table's chunks team, team + teams, ... counted from the last one: the norm's pass kept the end of the list
// in the L2.
template <int CAP>
__device__ __forceinline__ void scale_table(const Table<CAP>& t, uint32_t team, uint32_t teams, int thread, double f) {
    for (uint32_t i = team; i < t.chunks; i += teams) {
        const uint32_t c = t.chunks - 1 - i;
        const int k = tensor_of(t, c);
        const uint32_t chunk = c - t.first_chunk[k];
        const void* src = t.src[k];
        void* dst = t.dst[k];
        switch (t.dtype[k]) {
            case SPLAT_F32:
                scale_chunk(static_cast<const float*>(src), static_cast<float*>(dst), t.n[k], chunk, thread, f);
                break;
            case SPLAT_BF16:
                scale_chunk(static_cast<const __nv_bfloat16*>(src), static_cast<__nv_bfloat16*>(dst), t.n[k], chunk,
                            thread, f);
                break;
            case SPLAT_F16:
                scale_chunk(static_cast<const __half*>(src), static_cast<__half*>(dst), t.n[k], chunk, thread, f);
                break;
            default:
                scale_chunk(static_cast<const double*>(src), static_cast<double*>(dst), t.n[k], chunk, thread, f);
                break;
        }
    }
}

template <int CAP>
__global__ void __launch_bounds__(kScaleThreads)
    k_clip_scale(const __grid_constant__ Table<CAP> t, const __grid_constant__ Clip c, int in_place) {
    const double f = block_factor(c);
    if (in_place && f == 1.0) return;  // x * 1 is x, NaN and infinities too
    scale_table(t, blockIdx.x, gridDim.x, threadIdx.x, f);
}

// Norm, and scaling when `clip`, of a small list in one launch of one cluster.
template <int CAP, int NORM>
__global__ void __launch_bounds__(kSmallThreads)
    k_norm_small(const __grid_constant__ Table<CAP> t, const __grid_constant__ Clip c, int clip, int in_place) {
    const double norm = cluster_norm<CAP, NORM>(t, c.norm_f64);
    if (blockIdx.x == 0 && threadIdx.x == 0) store_norm(c, norm);
    if (!clip) return;
    const double f = factor_of(norm, c.max_norm);
    if (in_place && f == 1.0) return;
    constexpr int kTeams = kSmallThreads / kTeam;
    scale_table(t, blockIdx.x * kTeams + threadIdx.x / kTeam, kSmallCluster * kTeams, threadIdx.x % kTeam, f);
}

template <int CAP>
int norm_of(int count, const void* const* grads, const long long* n, const unsigned char* dtypes, int norm_type,
            double* partials, Clip& c, Again again, cudaStream_t st) {
    Table<CAP> t;
    int used = 0;
    long long chunks = 0;
    for (int i = 0; i < count;) {
        i = fill(t, i, count, grads, nullptr, n, dtypes);
        if (t.count == 0) break;
        constexpr unsigned int kTeams = kNormThreads / kTeam;
        const unsigned int grid = std::min((t.chunks + kTeams - 1) / kTeams,
                                           static_cast<unsigned int>(std::min(kNormBlocks * sm_count(), kMaxPartials)));
        SPLAT_FOR_NORM(norm_type, NORM,
                       (k_norm_partials<CAP, NORM>
                        <<<grid, kNormThreads, 0, st>>>(t, partials + used, again == Again::kAll ? kKeepChunks : 0u)));
        note_launch();
        used += static_cast<int>(grid);
        chunks += t.chunks;
        SPLAT_TRY(check_launch("gradient norm"));
    }
    if (again != Again::kNo && chunks <= kDirectChunks) {
        c.partials = partials;
        c.count = used;
        c.norm_type = norm_type;
        return SPLAT_OK;
    }
    SPLAT_CUDA(launch(k_norm_finish, 1, 32, st, used > 0, 1, static_cast<const double*>(partials), used, norm_type, c));
    note_launch();
    return check_launch("gradient norm");
}

// Runs the statement with CAP the table that the list fits best (a launch copies all of its table; 29 KB cost 3 us of
// the host's time).
#define SPLAT_FOR_TABLE(count, CAP, ...)      \
    do {                                      \
        if ((count) <= 16) {                  \
            constexpr int CAP = 16;           \
            __VA_ARGS__;                      \
        } else if ((count) <= 64) {           \
            constexpr int CAP = 64;           \
            __VA_ARGS__;                      \
        } else if ((count) <= 256) {          \
            constexpr int CAP = 256;          \
            __VA_ARGS__;                      \
        } else {                              \
            constexpr int CAP = kTableMax;    \
            __VA_ARGS__;                      \
        }                                     \
    } while (0)

int enqueue_norm(int count, const void* const* grads, const long long* n, const unsigned char* dtypes, int norm_type,
                 double* partials, Clip& c, Again again, cudaStream_t st) {
    SPLAT_FOR_TABLE(count, CAP, return norm_of<CAP>(count, grads, n, dtypes, norm_type, partials, c, again, st));
}

// One launch for a list that fits one small table.
template <int CAP>
int small(int count, const void* const* grads, void* const* outs, const long long* n, const unsigned char* dtypes,
          int norm_type, const Clip& c, int in_place, cudaStream_t st) {
    Table<CAP> t;
    fill(t, 0, count, grads, outs, n, dtypes);
    cudaError_t e = cudaSuccess;
    SPLAT_FOR_NORM(norm_type, NORM,
                   e = launch(k_norm_small<CAP, NORM>, kSmallCluster, kSmallThreads, st, false, kSmallCluster, t, c,
                              outs != nullptr ? 1 : 0, in_place));
    SPLAT_CUDA(e);
    note_launch();
    return check_launch("gradient norm");
}

int run_small(int count, const void* const* grads, void* const* outs, const long long* n, const unsigned char* dtypes,
              int norm_type, const Clip& c, int in_place, cudaStream_t st) {
    return count <= 16 ? small<16>(count, grads, outs, n, dtypes, norm_type, c, in_place, st)
                       : small<kSmallTensors>(count, grads, outs, n, dtypes, norm_type, c, in_place, st);
}

template <int CAP>
int scale_all(int count, const void* const* grads, void* const* outs, const long long* n, const unsigned char* dtypes,
              const Clip& c, int in_place, bool dependent, cudaStream_t st) {
    Table<CAP> t;
    for (int i = 0; i < count;) {
        i = fill(t, i, count, grads, outs, n, dtypes);
        if (t.count == 0) break;
        unsigned int grid = t.chunks;
        if (in_place) grid = std::max(div_up(grid, kScaleChunksInPlace), std::min(grid, kScaleBlocks * sm_count()));
        grid = std::min(grid, 0x7fffffffu);
        SPLAT_CUDA(launch(k_clip_scale<CAP>, grid, kScaleThreads, st, dependent, 1, t, c, in_place));
        dependent = false;
        note_launch();
        SPLAT_TRY(check_launch("splat_grad_clip"));
    }
    return SPLAT_OK;
}

int enqueue_scaling(int count, const void* const* grads, void* const* outs, const long long* n,
                    const unsigned char* dtypes, const Clip& c, int in_place, bool dependent, cudaStream_t st) {
    SPLAT_FOR_TABLE(count, CAP, return scale_all<CAP>(count, grads, outs, n, dtypes, c, in_place, dependent, st));
}

int check_list(const char* what, int count, const void* const* grads, const long long* n,
               const unsigned char* dtypes, int norm_f64) {
    SPLAT_REQUIRE(count >= 0, "%s: negative count", what);
    SPLAT_REQUIRE(count == 0 || (grads && n && dtypes), "%s: the list of tensors is missing", what);
    long long chunks = 0;
    for (int i = 0; i < count; ++i) {
        SPLAT_REQUIRE(n[i] >= 0, "%s: tensor %d has negative size", what, i);
        SPLAT_REQUIRE(dtypes[i] <= SPLAT_F64, "%s: tensor %d has an unknown type", what, i);
        // 32 TiB
        SPLAT_REQUIRE(n[i] <= (1ll << 45) / size_of(dtypes[i]), "%s: tensor %d has %lld elements", what, i, n[i]);
        SPLAT_REQUIRE(dtypes[i] != SPLAT_F64 || norm_f64, "%s: tensor %d is float64, the norm is not", what, i);
        if (n[i] == 0) continue;
        SPLAT_REQUIRE(grads[i], "%s: tensor %d has a null buffer", what, i);
        SPLAT_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % size_of(dtypes[i]) == 0,
                      "%s: tensor %d is not aligned to its type", what, i);
        chunks += chunks_of(grads[i], n[i], dtypes[i]);
        // No device holds as much, but a list may name a tensor many times. A kernel's chunk index, raised by less than
        // 2^31 at a time, stays in 32 bits so, and every launch has its place in the workspace.
        SPLAT_REQUIRE(chunks < (1ll << 31), "%s: the tensors have more than 32 TiB together", what);
    }
    return SPLAT_OK;
}

// What is written overlaps nothing else: the outputs one another, (out of place) any input, or the norm.
int check_overlap(int count, const void* const* grads, void* const* outs, const long long* n,
                  const unsigned char* dtypes, bool in_place, const Clip& c, bool given) {
    std::unique_ptr<Range[]> s(new (std::nothrow) Range[2 * static_cast<size_t>(count) + 1]);
    SPLAT_REQUIRE(s, "splat_grad_clip: out of host memory");
    int k = 0;
    s[k++] = range_of(c.norm, c.norm_f64 ? 8 : 4, !given);
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const auto bytes = static_cast<unsigned long long>(n[i]) * size_of(dtypes[i]);
        s[k++] = range_of(outs[i], bytes, true);
        if (!in_place) s[k++] = range_of(grads[i], bytes, false);
    }
    SPLAT_REQUIRE(apart(s.get(), k), "splat_grad_clip: a tensor that is written overlaps another one of the call");
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
    SPLAT_REQUIRE(gradnorm::aligned(norm, norm_is_f64), "splat_grad_norm: the norm's buffer is missing or not aligned");
    SPLAT_REQUIRE(gradnorm::aligned(workspace, true) && workspace_bytes >= gradnorm::partial_bytes(count),
                  "splat_grad_norm: workspace too small or not aligned");
    gradnorm::Clip c{norm, 0.0, norm_is_f64};
    const cudaStream_t st = as_stream(stream);
    if (gradnorm::is_small(count, grads, n, dtypes))
        return gradnorm::run_small(count, grads, nullptr, n, dtypes, norm_type, c, 0, st);
    return gradnorm::enqueue_norm(count, grads, n, dtypes, norm_type, static_cast<double*>(workspace), c,
                                  gradnorm::Again::kNo, st);
}

int splat_grad_clip(int count, const void* const* grads, void* const* outs, const long long* n,
                    const unsigned char* dtypes, int norm_type, double max_norm, void* norm, int norm_is_f64,
                    void* workspace, size_t workspace_bytes, void* stream) {
    SPLAT_TRY(gradnorm::check_list("splat_grad_clip", count, grads, n, dtypes, norm_is_f64));
    SPLAT_REQUIRE(norm_type == SPLAT_NORM_GIVEN || gradnorm::known_norm(norm_type),
                  "splat_grad_clip: unknown norm type %d", norm_type);
    SPLAT_REQUIRE(max_norm >= 0.0, "splat_grad_clip: max_norm must not be negative");
    SPLAT_REQUIRE(gradnorm::aligned(norm, norm_is_f64), "splat_grad_clip: the norm's buffer is missing or not aligned");
    const bool given = norm_type == SPLAT_NORM_GIVEN;
    SPLAT_REQUIRE(given || (gradnorm::aligned(workspace, true) && workspace_bytes >= gradnorm::partial_bytes(count)),
                  "splat_grad_clip: workspace too small or not aligned");
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
    gradnorm::Clip c{norm, max_norm, norm_is_f64};
    SPLAT_TRY(gradnorm::check_overlap(count, grads, outs, n, dtypes, same > 0, c, given));
    const cudaStream_t st = as_stream(stream);
    if (!given) {
        // the norm of a list without elements (0) is still the call's
        if (same + other == 0) return gradnorm::run_small(0, grads, nullptr, n, dtypes, norm_type, c, 0, st);
        if (gradnorm::is_small(count, grads, n, dtypes))
            return gradnorm::run_small(count, grads, outs, n, dtypes, norm_type, c, same > 0, st);
        SPLAT_TRY(gradnorm::enqueue_norm(count, grads, n, dtypes, norm_type, static_cast<double*>(workspace), c,
                                         same ? gradnorm::Again::kInPlace : gradnorm::Again::kAll, st));
    }
    return gradnorm::enqueue_scaling(count, grads, outs, n, dtypes, c, same > 0, !given, st);
}

}  // extern "C"
