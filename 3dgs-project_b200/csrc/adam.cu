// adam.cu - fused Adam over all parameter groups in one launch.
//
// Per element, the update of Faster-GS's adam_step_cu / adam_step_sparse_cu<false>
// (cluster/patches/fastergs_lean_adam.patch:88-130):
//   m = beta1 (m - g) + g;  v = beta2 (v - g^2) + g^2
//   p -= lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// Groups (means, scales, rotations, opacities, sh0, sh_rest) are described by a table passed by value;
// each 256-thread block owns a contiguous run of one group and streams it with 16-byte accesses when
// the group's buffers allow, so a step reads 4 and writes 3 floats per element and nothing else.
// k_adam_lean adds the two options of the reference's lean Adam (adam_step_sparse_cu<LOWP>, same patch):
// a per-primitive visibility mask and bfloat16 moments written with stochastic rounding.
// Both kernels have a clipped form that multiplies each gradient by the clip factor of the global gradient norm
// (grad_norm.cuh) as it is read, so that clipping costs the norm's read of the gradients and nothing else.
#include <algorithm>

#include "adam_math.cuh"
#include "common.cuh"
#include "grad_norm.cuh"

namespace splat {
namespace adam {

constexpr int kThreads = 256;
constexpr int kVec = 4;
constexpr int kPerBlock = kThreads * kVec * 4;  // 4096 elements per block
static_assert(kThreads == gradnorm::kTeam, "the small kernels split a block into teams of one tile");

constexpr int kSmallParts = kPerBlock / (kThreads * kVec);

using GradTable = gradnorm::Table<SPLAT_ADAM_MAX_GROUPS>;

struct Group {
    float* param;
    const float* grad;
    float* exp_avg;
    float* exp_avg_sq;
    long long n;
    float step_size;       // lr / (1 - beta1^t)
    float bc2_sqrt_rcp;    // 1 / sqrt(1 - beta2^t)
    long long first_block;  // prefix of blocks over the groups
    int vec;               // all four buffers 16-byte aligned
};

struct Table {
    Group g[SPLAT_ADAM_MAX_GROUPS];
    int count;
    float beta1, beta2, eps;
};

// The gradient as the clipped step sees it: one product, rounded as the scaling kernel rounds it.
template <bool kClip>
__device__ __forceinline__ float clipped(float g, float factor) {
    return kClip ? __fmul_rn(g, factor) : g;
}

template <bool kClip>
__device__ __forceinline__ void upd(float& p, float g, float& m, float& v, const Group& G, const Table& t,
                                    float factor) {
    adam_element(p, clipped<kClip>(g, factor), m, v, G.step_size, G.bc2_sqrt_rcp, t.beta1, t.beta2, t.eps);
}

// One tile of kIters x 1024 elements from `base` on, by kThreads threads.
template <bool kClip, int kIters = kPerBlock / (kThreads * kVec)>
__device__ __forceinline__ void adam_tile(const Group& G, const Table& t, long long base, int thread, float f) {
    if (G.vec) {
#pragma unroll
        for (int k = 0; k < kIters; ++k) {
            const long long e = base + (static_cast<long long>(k) * kThreads + thread) * kVec;
            if (e + kVec <= G.n) {
                float4 p = *reinterpret_cast<const float4*>(G.param + e);
                const float4 g = __ldg(reinterpret_cast<const float4*>(G.grad + e));
                float4 m = *reinterpret_cast<const float4*>(G.exp_avg + e);
                float4 v = *reinterpret_cast<const float4*>(G.exp_avg_sq + e);
                upd<kClip>(p.x, g.x, m.x, v.x, G, t, f);
                upd<kClip>(p.y, g.y, m.y, v.y, G, t, f);
                upd<kClip>(p.z, g.z, m.z, v.z, G, t, f);
                upd<kClip>(p.w, g.w, m.w, v.w, G, t, f);
                *reinterpret_cast<float4*>(G.param + e) = p;
                *reinterpret_cast<float4*>(G.exp_avg + e) = m;
                *reinterpret_cast<float4*>(G.exp_avg_sq + e) = v;
            } else {
                for (long long j = e; j < G.n; ++j)
                    upd<kClip>(G.param[j], G.grad[j], G.exp_avg[j], G.exp_avg_sq[j], G, t, f);
            }
        }
    } else {
        for (long long e = base + thread; e < base + kIters * kThreads * kVec && e < G.n; e += kThreads)
            upd<kClip>(G.param[e], G.grad[e], G.exp_avg[e], G.exp_avg_sq[e], G, t, f);
    }
}

// The group that tile `tile` of the launch belongs to.
template <typename T>
__device__ __forceinline__ int group_of(const T& t, long long tile) {
    int gi = 0;
#pragma unroll 1
    while (gi + 1 < t.count && tile >= t.g[gi + 1].first_block) ++gi;
    return gi;
}

__global__ void __launch_bounds__(kThreads) k_adam(Table t) {
    const Group& G = t.g[group_of(t, blockIdx.x)];
    adam_tile<false>(G, t, (static_cast<long long>(blockIdx.x) - G.first_block) * kPerBlock, threadIdx.x, 1.f);
}

// The clipped step: k_adam with the factor, after the norm's kernels. It and they are bound by HBM: 3M Gaussians move
// 4.96 GB in the step and 0.71 GB in the norm's pass, less the 64 MiB that this pass leaves in the L2 for the tiles taken
// first here, and take 846 us (105 of them the norm's), 5.6 GB at 6.6 TB/s. A resident grid whose blocks loop over
// tiles took 935 us: blocks in step with one another load and store in turn.
__global__ void __launch_bounds__(kThreads, 5)
    k_adam_clipped(const __grid_constant__ Table t, const __grid_constant__ gradnorm::Clip c) {
    const long long tile = gridDim.x - 1u - blockIdx.x;
    const Group& G = t.g[group_of(t, tile)];
    const float f = static_cast<float>(gradnorm::block_factor(c));
    adam_tile<true>(G, t, (tile - G.first_block) * kPerBlock, threadIdx.x, f);
}

// The clipped step of a small model in one launch: every cluster takes the norm of all gradients for itself, then its
// share of the tiles. 4096 2D Gaussians take 5.9 us, 3.5 of which are the norm; by whole tiles, on fewer SMs, 9.2.
template <int NORM>
__global__ void __launch_bounds__(gradnorm::kSmallThreads)
    k_adam_small(const __grid_constant__ Table t, const __grid_constant__ GradTable grads,
                 const __grid_constant__ gradnorm::Clip c, long long tiles) {
    const double norm = gradnorm::cluster_norm<SPLAT_ADAM_MAX_GROUPS, NORM>(grads, 0);
    if (blockIdx.x == 0 && threadIdx.x == 0) gradnorm::store_norm(c, norm);
    const float f = static_cast<float>(gradnorm::factor_of(norm, c.max_norm));
    // A quarter of a tile at a time: one vector a thread, as many blocks as that takes.
    constexpr int kTeams = gradnorm::kSmallThreads / kThreads;
    for (long long q = static_cast<long long>(blockIdx.x) * kTeams + threadIdx.x / kThreads; q < kSmallParts * tiles;
         q += static_cast<long long>(gridDim.x) * kTeams) {
        const long long tile = q / kSmallParts;
        const Group& G = t.g[group_of(t, tile)];
        const long long base = (tile - G.first_block) * kPerBlock + (q % kSmallParts) * (kThreads * kVec);
        if (base < G.n) adam_tile<true, 1>(G, t, base, threadIdx.x % kThreads, f);
    }
}

// ---- lean Adam: visibility mask and bfloat16 moments with stochastic rounding ----

struct LeanGroup {
    float* param;
    const float* grad;
    void* exp_avg;
    void* exp_avg_sq;
    long long n;
    float step_size;
    float bc2_sqrt_rcp;
    long long first_block;
    int features;
    uint32_t magic;  // ceil(2^32 / features)
    int lowp;
    int vec;  // 16-byte (fp32 moments) / 8-byte (bf16 moments) accesses possible, features at most kMaxFeatures
};

struct LeanTable {
    LeanGroup g[SPLAT_ADAM_MAX_GROUPS];
    int count;
    float beta1, beta2, eps;
    uint32_t seed;
    const int32_t* visibility;  // may be null
};

// lowbias32 (C. Wellons, "hash prospector", 2018): a 32-bit integer hash with two multiply-xorshift rounds.
__device__ __forceinline__ uint32_t lowbias32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    x ^= x >> 16;
    return x;
}

__device__ __forceinline__ float bf16_to_float(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }

// Stochastic rounding to bfloat16 of a result of float32 arithmetic: uniform noise in the 16 bits that are dropped, then
// truncation. NaN stays NaN: arithmetic gives it as 0x7FFFFFFF, where the noise would carry through the exponent into the
// sign and leave -0, so it is cut to 0x7FFF0000, the largest of all values as a signed integer. One minimum an element
// costs the step of 1M Gaussians with bfloat16 SH moments 0.5%; a comparison and a choice take 2%, a branch 5%.
__device__ __forceinline__ uint16_t float_to_bf16_sr(float f, uint32_t rnd) {
    const uint32_t bits = static_cast<uint32_t>(min(__float_as_int(f), 0x7FFF0000));
    return static_cast<uint16_t>((bits + (rnd & 0xFFFFu)) >> 16);
}

// The primitive that element i of the group belongs to: a 32-bit division where the group's element count allows
// (every group of a scene below 2^32 elements), a 64-bit one otherwise.
__device__ __forceinline__ long long primitive_of(const LeanGroup& G, long long i) {
    if (G.n <= 0xFFFFFFFFll) return static_cast<uint32_t>(i) / static_cast<uint32_t>(G.features);
    return i / G.features;
}

template <bool kLowp, bool kClip>
__device__ __forceinline__ void lean_one(const LeanGroup& G, const LeanTable& t, long long i, float f) {
    if (t.visibility && t.visibility[primitive_of(G, i)] == 0) return;
    const float g = clipped<kClip>(G.grad[i], f);
    float m, v;
    if (kLowp) {
        m = bf16_to_float(static_cast<const uint16_t*>(G.exp_avg)[i]);
        v = bf16_to_float(static_cast<const uint16_t*>(G.exp_avg_sq)[i]);
    } else {
        m = static_cast<const float*>(G.exp_avg)[i];
        v = static_cast<const float*>(G.exp_avg_sq)[i];
    }
    adam_element(G.param[i], g, m, v, G.step_size, G.bc2_sqrt_rcp, t.beta1, t.beta2, t.eps);
    if (kLowp) {
        const uint32_t r1 = lowbias32(static_cast<uint32_t>(i) ^ t.seed);
        const uint32_t r2 = lowbias32(r1);
        static_cast<uint16_t*>(G.exp_avg)[i] = float_to_bf16_sr(m, r1);
        static_cast<uint16_t*>(G.exp_avg_sq)[i] = float_to_bf16_sr(v, r2);
    } else {
        static_cast<float*>(G.exp_avg)[i] = m;
        static_cast<float*>(G.exp_avg_sq)[i] = v;
    }
}

// Finds the primitives of a tile's elements with one division a tile: an element's offset from the first element of
// the tile's first primitive is below 2^16 (features at most kMaxFeatures), where a multiplication by 2^32 / features,
// rounded up, divides exactly.
constexpr int kMaxFeatures = 32768;

struct TilePrimitives {
    const int32_t* visibility;  // of the tile's first primitive
    uint32_t first;             // elements of that primitive before the tile
    uint32_t features, magic;

    __device__ __forceinline__ TilePrimitives(const LeanGroup& G, const int32_t* vis, long long base) {
        const long long prim = primitive_of(G, base);
        visibility = vis + prim;
        features = static_cast<uint32_t>(G.features);
        first = static_cast<uint32_t>(base - prim * G.features);
        magic = G.magic;
    }

    // Which of the four elements from offset `o` of the tile on are of visible primitives (bit k: element o + k). All
    // four exist.
    __device__ __forceinline__ unsigned mask(uint32_t o) const {
        if (features == 1) {
            unsigned m = 0u;
#pragma unroll
            for (int k = 0; k < kVec; ++k) m |= static_cast<unsigned>(visibility[o + k] != 0) << k;
            return m;
        }
        const uint32_t x = first + o, p = __umulhi(x, magic);
        const uint32_t left = (p + 1u) * features - x;  // elements of primitive p from x on
        unsigned m = visibility[p] != 0 ? (1u << min(left, 4u)) - 1u : 0u;
        if (left < 4u) {
            // elements left ... 3 are of the next primitive, or with 2 features of the next two
            const uint32_t more = min(left + features, 4u);
            if (visibility[p + 1u] != 0) m |= ((1u << more) - 1u) & ~((1u << left) - 1u);
            if (more < 4u && visibility[p + 2u] != 0) m |= 0xFu & ~((1u << more) - 1u);
        }
        return m;
    }
};
static_assert(kMaxFeatures + kPerBlock <= 65536, "TilePrimitives divides offsets below 2^16");

// Four consecutive elements from e, read and written with vector accesses.
template <bool kLowp, bool kClip>
struct LeanFour {
    float4 p, g, m4{}, v4{};  // m4, v4: float32 moments
    uint2 mb{}, vb{};         // bfloat16 moments

    __device__ __forceinline__ void load(const LeanGroup& G, long long e) {
        p = *reinterpret_cast<const float4*>(G.param + e);
        g = __ldg(reinterpret_cast<const float4*>(G.grad + e));
        if (kLowp) {
            mb = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(G.exp_avg) + e);
            vb = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(G.exp_avg_sq) + e);
        } else {
            m4 = *reinterpret_cast<const float4*>(static_cast<const float*>(G.exp_avg) + e);
            v4 = *reinterpret_cast<const float4*>(static_cast<const float*>(G.exp_avg_sq) + e);
        }
    }

    // Updates and stores them; `mask` from TilePrimitives (non-zero): elements of primitives that are not visible keep
    // their parameter and moments.
    __device__ __forceinline__ void update(const LeanGroup& G, const LeanTable& t, long long e, unsigned mask, float f) {
        float pv[kVec] = {p.x, p.y, p.z, p.w};
        const float gv[kVec] = {g.x, g.y, g.z, g.w};
        float mv[kVec] = {m4.x, m4.y, m4.z, m4.w}, vv[kVec] = {v4.x, v4.y, v4.z, v4.w};
        uint32_t mo[2] = {mb.x, mb.y}, vo[2] = {vb.x, vb.y};
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            if (!((mask >> k) & 1u)) continue;
            const int sh = 16 * (k & 1);
            if (kLowp) {
                mv[k] = bf16_to_float(static_cast<uint16_t>(mo[k >> 1] >> sh));
                vv[k] = bf16_to_float(static_cast<uint16_t>(vo[k >> 1] >> sh));
            }
            adam_element(pv[k], clipped<kClip>(gv[k], f), mv[k], vv[k], G.step_size, G.bc2_sqrt_rcp, t.beta1, t.beta2,
                         t.eps);
            if (kLowp) {
                const uint32_t r1 = lowbias32(static_cast<uint32_t>(e + k) ^ t.seed);
                const uint32_t r2 = lowbias32(r1);
                mo[k >> 1] = (mo[k >> 1] & ~(0xFFFFu << sh)) | (static_cast<uint32_t>(float_to_bf16_sr(mv[k], r1)) << sh);
                vo[k >> 1] = (vo[k >> 1] & ~(0xFFFFu << sh)) | (static_cast<uint32_t>(float_to_bf16_sr(vv[k], r2)) << sh);
            }
        }
        *reinterpret_cast<float4*>(G.param + e) = make_float4(pv[0], pv[1], pv[2], pv[3]);
        if (kLowp) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(G.exp_avg) + e) = make_uint2(mo[0], mo[1]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(G.exp_avg_sq) + e) = make_uint2(vo[0], vo[1]);
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(G.exp_avg) + e) = make_float4(mv[0], mv[1], mv[2], mv[3]);
            *reinterpret_cast<float4*>(static_cast<float*>(G.exp_avg_sq) + e) = make_float4(vv[0], vv[1], vv[2], vv[3]);
        }
    }
};

constexpr int kLeanIters = kPerBlock / (kThreads * kVec);
constexpr int kLeanList = 32 * kLeanIters;  // groups of four elements that a warp looks at in a tile

// One tile, by kThreads threads whose warps each have kLeanList entries of shared memory at `list`. With a mask, a
// warp first collects its groups of four that have a visible element (the visibility of all of them is loaded before
// any is used) and then deals them to its lanes in order: the update is dozens of instructions an element, which the
// lanes of groups without one would sit through. Measured on 3M Gaussians with bfloat16 SH moments, against each thread
// updating its own groups: 51% visible at random 574 us (611), visible in long runs 404 (405), without a mask, where
// nothing is collected, 590 (615). On 1M: 10% visible at random 108 (130), 90% 221 (219), all 224 (224); the collecting
// costs up to 0.4 us where it saves nothing, which shows below 256 Gaussians (2.3 us against 2.0 for four). Lanes that
// keep their own groups where dealing saves no round took 220 at 90% and 1% longer everywhere else. Not unrolled: two
// groups in flight a thread took 638 us at random on 3M.
template <bool kLowp, bool kClip, bool kMasked, int kIters>
__device__ __forceinline__ void lean_block(const LeanGroup& G, const LeanTable& t, long long base, int thread,
                                           uint16_t* list, float f) {
    if (!G.vec) {
        for (long long e = base + thread; e < base + kIters * kThreads * kVec && e < G.n; e += kThreads)
            lean_one<kLowp, kClip>(G, t, e, f);
        return;
    }
    if (kMasked) {
        unsigned mask[kIters];
        const TilePrimitives prims(G, t.visibility, base);
#pragma unroll
        for (int k = 0; k < kIters; ++k) {
            const uint32_t o = static_cast<uint32_t>(k * kThreads + thread) * kVec;
            mask[k] = base + o + kVec <= G.n ? prims.mask(o) : 0u;
        }
        const int lane = thread & 31;
        int count = 0;
#pragma unroll
        for (int k = 0; k < kIters; ++k) {
            const unsigned some = __ballot_sync(kFullMask, mask[k] != 0u);
            if (mask[k])
                list[count + __popc(some & ((1u << lane) - 1u))] =
                    static_cast<uint16_t>((k * kThreads + thread) << kVec | mask[k]);
            count += __popc(some);
        }
        __syncwarp();
#pragma unroll 1
        for (int j = lane; j < count; j += 32) {
            const unsigned a = list[j];
            const long long e = base + static_cast<long long>(a >> kVec) * kVec;
            LeanFour<kLowp, kClip> x;
            x.load(G, e);
            x.update(G, t, e, a & ((1u << kVec) - 1u), f);
        }
        __syncwarp();  // the list is read before a next tile fills it
    }
#pragma unroll
    for (int k = 0; k < kIters; ++k) {
        const long long e = base + (static_cast<long long>(k) * kThreads + thread) * kVec;
        if (e + kVec <= G.n) {
            if (!kMasked) {
                LeanFour<kLowp, kClip> x;
                x.load(G, e);
                x.update(G, t, e, (1u << kVec) - 1u, f);
            }
        } else {
            for (long long j = e; j < G.n; ++j) lean_one<kLowp, kClip>(G, t, j, f);
        }
    }
}

// Part `part` (of kIters x 1024 elements) of a tile; without one, all of it.
template <bool kClip, bool kMasked, int kIters = kLeanIters>
__device__ __forceinline__ void lean_tile(const LeanTable& t, long long tile, int thread, uint16_t* list, float f,
                                          int part = 0) {
    const LeanGroup& G = t.g[group_of(t, tile)];
    const long long base = (tile - G.first_block) * kPerBlock + part * (kIters * kThreads * kVec);
    if (base >= G.n) return;
    if (G.lowp)
        lean_block<true, kClip, kMasked, kIters>(G, t, base, thread, list, f);
    else
        lean_block<false, kClip, kMasked, kIters>(G, t, base, thread, list, f);
}

// kMasked: there is a visibility mask.
template <bool kMasked>
__global__ void __launch_bounds__(kThreads) k_adam_lean(const __grid_constant__ LeanTable t) {
    __shared__ uint16_t s_list[kThreads / 32][kLeanList];
    lean_tile<false, kMasked>(t, blockIdx.x, threadIdx.x, s_list[threadIdx.x / 32], 1.f);
}

// As k_adam_clipped. 1M Gaussians of which 35% are visible, at random: 171 us after the norm's 35, 753 MB from and to
// HBM, more than the visible elements' 370 MB because rows of 12 to 180 bytes share their 32-byte sectors. 62% of the
// issue slots are busy beside 4.5 TB/s, and loads ahead of the update made it slower.
// With the mask six blocks an SM are faster than five (206 us against 219, the norm included in both), without it slower
// (3M Gaussians in float32: this kernel alone 773 us against 733).
template <bool kMasked>
__global__ void __launch_bounds__(kThreads, kMasked ? 6 : 1)
    k_adam_lean_clipped(const __grid_constant__ LeanTable t, const __grid_constant__ gradnorm::Clip c) {
    __shared__ uint16_t s_list[kThreads / 32][kLeanList];
    const float f = static_cast<float>(gradnorm::block_factor(c));
    lean_tile<true, kMasked>(t, gridDim.x - 1u - blockIdx.x, threadIdx.x, s_list[threadIdx.x / 32], f);
}

// As k_adam_small.
template <int NORM, bool kMasked>
__global__ void __launch_bounds__(gradnorm::kSmallThreads)
    k_adam_lean_small(const __grid_constant__ LeanTable t, const __grid_constant__ GradTable grads,
                      const __grid_constant__ gradnorm::Clip c, long long tiles) {
    __shared__ uint16_t s_list[gradnorm::kSmallThreads / 32][kLeanList];
    const double norm = gradnorm::cluster_norm<SPLAT_ADAM_MAX_GROUPS, NORM>(grads, 0);
    if (blockIdx.x == 0 && threadIdx.x == 0) gradnorm::store_norm(c, norm);
    const float f = static_cast<float>(gradnorm::factor_of(norm, c.max_norm));
    constexpr int kTeams = gradnorm::kSmallThreads / kThreads;
    for (long long q = static_cast<long long>(blockIdx.x) * kTeams + threadIdx.x / kThreads; q < kSmallParts * tiles;
         q += static_cast<long long>(gridDim.x) * kTeams)
        lean_tile<true, kMasked, 1>(t, q / kSmallParts, threadIdx.x % kThreads, s_list[threadIdx.x / 32], f,
                                    static_cast<int>(q % kSmallParts));
}

}  // namespace adam
}  // namespace splat

using namespace splat;

namespace {

// The reference wrapper's host arithmetic (fastergs_lean_adam.patch:162-164): in double, rounded once to float.
void bias_corrections(double lr, double beta1, double beta2, int step, float& step_size, float& bc2_sqrt_rcp) {
    adam_bias_corrections(lr, beta1, beta2, step, step_size, bc2_sqrt_rcp);
}

// The kernel's table for `count` groups; *blocks is 0 when every group is empty.
int build_table(const char* what, int count, const adam_group* groups, int step, double beta1, double beta2, double eps,
                adam::Table& t, long long* total_blocks) {
    SPLAT_REQUIRE(count >= 0 && count <= SPLAT_ADAM_MAX_GROUPS, "%s: %d groups (at most %d)", what, count,
                  SPLAT_ADAM_MAX_GROUPS);
    SPLAT_REQUIRE(step >= 1, "%s: step must be >= 1", what);
    t.beta1 = static_cast<float>(beta1);
    t.beta2 = static_cast<float>(beta2);
    t.eps = static_cast<float>(eps);
    long long blocks = 0;
    int k = 0;
    for (int i = 0; i < count; ++i) {
        const adam_group& g = groups[i];
        SPLAT_REQUIRE(g.n >= 0, "%s: group %d has negative size", what, i);
        if (g.n == 0) continue;
        SPLAT_REQUIRE(g.param && g.grad && g.exp_avg && g.exp_avg_sq, "%s: group %d has a null buffer", what, i);
        adam::Group& G = t.g[k++];
        G.param = g.param;
        G.grad = g.grad;
        G.exp_avg = g.exp_avg;
        G.exp_avg_sq = g.exp_avg_sq;
        G.n = g.n;
        bias_corrections(g.lr, beta1, beta2, step, G.step_size, G.bc2_sqrt_rcp);
        G.first_block = blocks;
        G.vec = ((reinterpret_cast<uintptr_t>(g.param) | reinterpret_cast<uintptr_t>(g.grad) |
                  reinterpret_cast<uintptr_t>(g.exp_avg) | reinterpret_cast<uintptr_t>(g.exp_avg_sq)) & 15u) == 0;
        blocks += (g.n + adam::kPerBlock - 1) / adam::kPerBlock;
    }
    t.count = k;
    SPLAT_REQUIRE(blocks < (1ll << 31), "%s: too many elements", what);
    *total_blocks = blocks;
    return SPLAT_OK;
}

int build_lean_table(const char* what, int count, const adam_lean_group* groups, int step, double beta1, double beta2,
                     double eps, const int32_t* visibility, long long n_primitives, adam::LeanTable& t,
                     long long* total_blocks) {
    SPLAT_REQUIRE(count >= 0 && count <= SPLAT_ADAM_MAX_GROUPS, "%s: %d groups (at most %d)", what, count,
                  SPLAT_ADAM_MAX_GROUPS);
    SPLAT_REQUIRE(step >= 1, "%s: step must be >= 1", what);
    t.beta1 = static_cast<float>(beta1);
    t.beta2 = static_cast<float>(beta2);
    t.eps = static_cast<float>(eps);
    t.seed = 0x9E3779B9u * static_cast<uint32_t>(step) + 0x85EBCA6Bu;
    t.visibility = visibility;
    long long blocks = 0;
    int k = 0;
    for (int i = 0; i < count; ++i) {
        const adam_lean_group& g = groups[i];
        SPLAT_REQUIRE(g.n >= 0 && (g.n == 0 || g.features >= 1), "%s: group %d has a bad size", what, i);
        if (g.n == 0) continue;  // rows of no elements (features 0) or no rows
        SPLAT_REQUIRE(g.param && g.grad && g.exp_avg && g.exp_avg_sq, "%s: group %d has a null buffer", what, i);
        SPLAT_REQUIRE(!visibility || g.n == static_cast<long long>(g.features) * n_primitives,
                      "%s: group %d has %lld elements, not %d x %lld primitives", what, i, g.n, g.features,
                      n_primitives);
        adam::LeanGroup& G = t.g[k++];
        G.param = g.param;
        G.grad = g.grad;
        G.exp_avg = g.exp_avg;
        G.exp_avg_sq = g.exp_avg_sq;
        G.n = g.n;
        bias_corrections(g.lr, beta1, beta2, step, G.step_size, G.bc2_sqrt_rcp);
        G.first_block = blocks;
        G.features = g.features;
        G.magic = static_cast<uint32_t>(((1ull << 32) + g.features - 1) / g.features);
        G.lowp = g.lowp_moments != 0;
        const uintptr_t moment_align = G.lowp ? 7u : 15u;
        G.vec = ((reinterpret_cast<uintptr_t>(g.param) | reinterpret_cast<uintptr_t>(g.grad)) & 15u) == 0 &&
                ((reinterpret_cast<uintptr_t>(g.exp_avg) | reinterpret_cast<uintptr_t>(g.exp_avg_sq)) & moment_align) == 0 &&
                (!visibility || g.features <= adam::kMaxFeatures);
        blocks += (g.n + adam::kPerBlock - 1) / adam::kPerBlock;
    }
    t.count = k;
    SPLAT_REQUIRE(blocks < (1ll << 31), "%s: too many elements", what);
    *total_blocks = blocks;
    return SPLAT_OK;
}

struct Grads {
    const void* grad[SPLAT_ADAM_MAX_GROUPS];
    long long n[SPLAT_ADAM_MAX_GROUPS];
    unsigned char dtype[SPLAT_ADAM_MAX_GROUPS];
};

unsigned long long moment_bytes(const adam_group&) { return 4; }
unsigned long long moment_bytes(const adam_lean_group& g) { return g.lowp_moments ? 2 : 4; }

// What a clipped step writes overlaps nothing else of it: in a step of one launch some clusters still read the gradients
// for the norm while others write.
template <typename G>
int check_overlap(const char* what, int count, const G* groups, const float* norm, bool given) {
    gradnorm::Range s[4 * SPLAT_ADAM_MAX_GROUPS + 1];
    int k = 0;
    s[k++] = gradnorm::range_of(norm, sizeof(float), !given);
    for (int i = 0; i < count; ++i) {
        const G& g = groups[i];
        if (g.n == 0) continue;
        const auto n = static_cast<unsigned long long>(g.n);
        s[k++] = gradnorm::range_of(g.param, 4 * n, true);
        s[k++] = gradnorm::range_of(g.grad, 4 * n, false);
        s[k++] = gradnorm::range_of(g.exp_avg, moment_bytes(g) * n, true);
        s[k++] = gradnorm::range_of(g.exp_avg_sq, moment_bytes(g) * n, true);
    }
    SPLAT_REQUIRE(gradnorm::apart(s, k), "%s: a buffer that is written overlaps another one of the call", what);
    return SPLAT_OK;
}

// A clipped step: the norm's kernel and the update's, or for a small model one kernel that does both.
template <typename G, typename T>
int clipped_step(const char* what, int count, const G* groups, const T& table, long long blocks,
                 void (*update)(T, gradnorm::Clip),
                 void (*const (&small)[3])(T, adam::GradTable, gradnorm::Clip, long long), int norm_type,
                 double max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    const bool given = norm_type == SPLAT_NORM_GIVEN;
    SPLAT_REQUIRE(given || gradnorm::known_norm(norm_type), "%s: unknown norm type %d", what, norm_type);
    SPLAT_REQUIRE(max_norm >= 0.0, "%s: max_norm must not be negative", what);
    SPLAT_REQUIRE(gradnorm::aligned(norm, false), "%s: the norm's buffer is missing or not aligned", what);
    SPLAT_REQUIRE(
        given || (gradnorm::aligned(workspace, true) && workspace_bytes >= splat_grad_workspace_size(count)),
        "%s: workspace too small or not aligned", what);
    SPLAT_TRY(check_overlap(what, count, groups, norm, given));
    if (blocks == 0)  // the norm of nothing is the call's all the same
        return given ? SPLAT_OK
                     : splat_grad_norm(0, nullptr, nullptr, nullptr, norm_type, norm, 0, workspace, workspace_bytes,
                                       stream);
    const cudaStream_t st = as_stream(stream);
    gradnorm::Clip c{norm, max_norm, 0};
    if (!given) {
        Grads list{};  // dtype 0: SPLAT_F32
        for (int i = 0; i < count; ++i) {
            list.grad[i] = groups[i].grad;
            list.n[i] = groups[i].n;
        }
        if (gradnorm::is_small(count, list.grad, list.n, list.dtype)) {
            adam::GradTable grads;
            gradnorm::fill(grads, 0, count, list.grad, nullptr, list.n, list.dtype);
            constexpr int kTilesPerCluster =
                gradnorm::kSmallCluster * (gradnorm::kSmallThreads / adam::kThreads);
            const long long clusters =
                std::min<long long>((adam::kSmallParts * blocks + kTilesPerCluster - 1) / kTilesPerCluster, 8);
            cudaError_t e = cudaSuccess;
            SPLAT_TIMED_LAUNCH("k_adam", st,
                               (e = gradnorm::launch(small[norm_type],
                                                     static_cast<unsigned int>(clusters * gradnorm::kSmallCluster),
                                                     gradnorm::kSmallThreads, st, false, gradnorm::kSmallCluster, table,
                                                     grads, c, blocks)));
            SPLAT_CUDA(e);
            note_launch();
            return check_launch(what);
        }
        SPLAT_TRY(gradnorm::enqueue_norm(count, list.grad, list.n, list.dtype, norm_type,
                                         static_cast<double*>(workspace), c, gradnorm::Again::kAll, st));
    }
    cudaError_t e = cudaSuccess;
    SPLAT_TIMED_LAUNCH("k_adam", st,
                       (e = gradnorm::launch(update, static_cast<unsigned int>(blocks), adam::kThreads, st, !given, 1,
                                             table, c)));
    SPLAT_CUDA(e);
    note_launch();
    return check_launch(what);
}

}  // namespace

extern "C" {

int adam_step_multi(int count, const adam_group* groups, int step, double beta1, double beta2, double eps,
                    void* stream) {
    adam::Table t{};
    long long blocks = 0;
    SPLAT_TRY(build_table("adam_step_multi", count, groups, step, beta1, beta2, eps, t, &blocks));
    if (blocks == 0) return SPLAT_OK;
    SPLAT_TIMED_LAUNCH("k_adam", as_stream(stream),
                       (adam::k_adam<<<static_cast<unsigned int>(blocks), adam::kThreads, 0, as_stream(stream)>>>(t)));
    note_launch();
    return check_launch("adam_step_multi");
}

int adam_step_multi_lean(int count, const adam_lean_group* groups, int step, double beta1, double beta2,
                         double eps, const int32_t* visibility, long long n_primitives, void* stream) {
    adam::LeanTable t{};
    long long blocks = 0;
    SPLAT_TRY(build_lean_table("adam_step_multi_lean", count, groups, step, beta1, beta2, eps, visibility, n_primitives,
                               t, &blocks));
    if (blocks == 0) return SPLAT_OK;
    const auto kernel = visibility ? adam::k_adam_lean<true> : adam::k_adam_lean<false>;
    kernel<<<static_cast<unsigned int>(blocks), adam::kThreads, 0, as_stream(stream)>>>(t);
    note_launch();
    return check_launch("adam_step_multi_lean");
}

int adam_step_multi_clipped(int count, const adam_group* groups, int step, double beta1, double beta2, double eps,
                            int norm_type, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                            void* stream) {
    static void (*const small[3])(adam::Table, adam::GradTable, gradnorm::Clip, long long) = {
        adam::k_adam_small<SPLAT_NORM_INF>, adam::k_adam_small<SPLAT_NORM_L1>, adam::k_adam_small<SPLAT_NORM_L2>};
    adam::Table t{};
    long long blocks = 0;
    SPLAT_TRY(build_table("adam_step_multi_clipped", count, groups, step, beta1, beta2, eps, t, &blocks));
    return clipped_step("adam_step_multi_clipped", count, groups, t, blocks, adam::k_adam_clipped, small, norm_type,
                        max_norm, norm, workspace, workspace_bytes, stream);
}

int adam_step_multi_lean_clipped(int count, const adam_lean_group* groups, int step, double beta1, double beta2,
                                 double eps, const int32_t* visibility, long long n_primitives, int norm_type,
                                 double max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    using Small = void (*)(adam::LeanTable, adam::GradTable, gradnorm::Clip, long long);
    static const Small small[2][3] = {
        {adam::k_adam_lean_small<SPLAT_NORM_INF, false>, adam::k_adam_lean_small<SPLAT_NORM_L1, false>,
         adam::k_adam_lean_small<SPLAT_NORM_L2, false>},
        {adam::k_adam_lean_small<SPLAT_NORM_INF, true>, adam::k_adam_lean_small<SPLAT_NORM_L1, true>,
         adam::k_adam_lean_small<SPLAT_NORM_L2, true>}};
    const bool masked = visibility != nullptr;
    adam::LeanTable t{};
    long long blocks = 0;
    SPLAT_TRY(build_lean_table("adam_step_multi_lean_clipped", count, groups, step, beta1, beta2, eps, visibility,
                               n_primitives, t, &blocks));
    const auto update = masked ? adam::k_adam_lean_clipped<true> : adam::k_adam_lean_clipped<false>;
    return clipped_step("adam_step_multi_lean_clipped", count, groups, t, blocks, update, small[masked], norm_type,
                        max_norm, norm, workspace, workspace_bytes, stream);
}

}  // extern "C"
