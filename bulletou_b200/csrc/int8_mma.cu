// The 8-bit product on the 5th-generation tensor cores (sm_100a):
// tcgen05.mma.kind::i8, 8-bit operands from shared memory, 32-bit integer sums
// in TMEM, so that every order of summation gives the same bits.
//
// Both operands are rows of k (K-major): a stage holds 128 bytes of k of each
// row of the tile, loaded by TMA with 128-byte swizzle, and takes four MMAs of
// 32 k.  Rows and k beyond the matrices are filled with zeros by the TMA.
//
// int8_pair_kernel, for large products: two CTAs of a cluster share a 256 x 256
// tile (cta_group::2).  Each loads 128 rows of q and 128 of w -- half of what
// two single CTAs would load for the same products, and what L2 can deliver
// per SM is the limit of a 128 x 256 tile.  Persistent; the 512 TMEM columns
// hold two accumulators, so a tile's epilogue runs under the next tile's MMAs.
// 16384 x 4096 x 4096: 165 us, 3.3 POP/s, the tensor pipe busy in 94 % of the
// cycles at the clock that the power limit leaves.  Where k is short the epilogue
// is the bound, by the shared memory that it shares with the operands: results
// staged as they are stored and fetched from there by TMA, with eight warps for
// them and five stages: 8192 x 1024 x 4096 with bf16 results 33 us and f32 43, where
// four warps that staged f32 and stored it themselves took 43 and 47 (lanes
// that store their own rows 44 and 74).  Six stages and four such warps take 35
// and 47; for many tiles of long k they are ahead by 4 %.
//
// int8_tile_kernel, where there are too few 256 x 256 tiles for the SMs: one
// 128 x 64 tile for each CTA, with k cut over a cluster of up to four CTAs where
// that is long; the partial integer sums meet through distributed shared memory.
// Bound by latency: 8 x 1536 x 2048 takes 5.8 us, of which 0.2 us for each 128 of
// k (an MMA takes 64 cycles to issue whatever its N, and a wait between) and 3.4
// us for the launch, the first load and the epilogue.  Meeting in a cluster costs
// about 2 us, so k is cut from 16 blocks of 128 on.
//
// Every wait on an mbarrier is bounded (2 s); where one runs out the CTA's
// remaining results are NaN.  No multicast loads.
#include <algorithm>

#include "int8_linear.cuh"
#include "tensor_core.cuh"
#include "token_launch.cuh"

namespace bou {
namespace {

constexpr int kTileM = 128;                 // rows of q for each CTA (MMA M of one CTA)
constexpr int kTileN = 64;                  // rows of w for a tile of one CTA
constexpr int kTileK = 128;                 // bytes of k in a stage: one swizzle atom
constexpr uint32_t kABytes = kTileM * kTileK;
constexpr int kStagePad = 4;                // floats between staged rows: 16-byte accesses without bank conflicts

// Instruction descriptor, kind::i8: D s32 [4,6) = 2, A s8 [7,10) = 1, B s8
// [10,13) = 1, both K-major, N >> 3 [17,23), M >> 4 [24,29).
constexpr uint32_t int8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n) >> 3 << 17) |
           (static_cast<uint32_t>(m) >> 4 << 24);
}

// K-major with 128-byte swizzle: groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t k_major_desc(uint32_t addr) { return smem_desc(addr, 16u, 1024u); }

template <int kGroup>
__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kGroup == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

__device__ __forceinline__ void commit_one(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Arrives on the barrier at this offset in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// The load's bytes are counted on the barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// The results of 32 columns of a lane's row.
__device__ __forceinline__ void results(const uint32_t* sum, float row_scale, const float* col_scale, const float* col_bias,
                                        float* v) {
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
        const float4 s = *reinterpret_cast<const float4*>(col_scale + c), b = *reinterpret_cast<const float4*>(col_bias + c);
        v[c] = int8_result(static_cast<int>(sum[c]), row_scale, s.x, b.x);
        v[c + 1] = int8_result(static_cast<int>(sum[c + 1]), row_scale, s.y, b.y);
        v[c + 2] = int8_result(static_cast<int>(sum[c + 2]), row_scale, s.z, b.z);
        v[c + 3] = int8_result(static_cast<int>(sum[c + 3]), row_scale, s.w, b.w);
    }
}

// A warp writes 32 rows x 32 columns, one row in each lane: through shared
// memory, so that the global stores cover whole rows of the block.
template <typename Out>
__device__ __forceinline__ void store_block(float* stage, const float* v, const ProductArgs& a, int row0, int col0,
                                            bool vector_ok) {
    constexpr int kCols = 32, kPitch = kCols + kStagePad;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < kCols; c += 4)
        *reinterpret_cast<float4*>(stage + lane * kPitch + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
    __syncwarp();
    Out* const out = static_cast<Out*>(a.out);
    if (vector_ok && col0 + kCols <= a.n) {
        constexpr int kVec = 16 / sizeof(Out);       // values of a 16-byte store
        constexpr int kLanes = kCols / kVec;         // lanes of a row
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 32 / kLanes) {
            const int r = r0 + lane / kLanes, c = lane % kLanes * kVec;
            if (row0 + r >= a.m) continue;
            const float* src = stage + r * kPitch + c;
            uint4 packed;
            if constexpr (sizeof(Out) == 4) {
                packed = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t* p = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(src[2 * i], src[2 * i + 1]);
                    p[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
            }
            *reinterpret_cast<uint4*>(out + static_cast<size_t>(row0 + r) * a.out_stride + col0 + c) = packed;
        }
    } else if (col0 + lane < a.n) {
        Out* at = out + static_cast<size_t>(row0) * a.out_stride + col0 + lane;
        const int rows = a.m - row0;
#pragma unroll
        for (int r = 0; r < 32; ++r, at += a.out_stride)
            if (r < rows) *at = from_f32<Out>(stage[r * kPitch + lane]);
    }
    __syncwarp();
}

// ------------------------------------------------------------------ one tile for each CTA
// kDeep, where every CTA has an SM to itself: all of the shared memory, so that 1
// KB of k of the tile is on the way at once (512 x 512 x 512: 5.9 us, 6.8 without);
// otherwise 96 KB, for two CTAs.
template <bool kDeep>
struct TileShape {
    static constexpr uint32_t kStageBytes = kABytes + kTileN * kTileK;
    static constexpr int kStages = kDeep ? 192 * 1024 / kStageBytes : 96 * 1024 / kStageBytes;
    // after the last MMA the stages hold the partial sums and the staged rows
    static constexpr uint32_t kStagingAt = kTileN * kTileM * 4;
    static constexpr int kThreads = 128;
    static constexpr uint32_t kSmem = kStages * kStageBytes + 2 * kTileN * 4 + 256 + 1024;
    static_assert(kStagingAt + 4 * 32 * (32 + kStagePad) * 4 <= kStages * kStageBytes);
};

// `splits` CTAs of a cluster share a tile and cut k; the grid is their tiles,
// the columns' tiles first.
template <bool kDeep, typename Out>
__global__ void __launch_bounds__(128) int8_tile_kernel(const __grid_constant__ CUtensorMap map_q,
                                                        const __grid_constant__ CUtensorMap map_w, const ProductArgs a,
                                                        int splits, int box_rows, bool vector_ok, bool weights_ready) {
    using S = TileShape<kDeep>;
    extern __shared__ uint8_t raw[];
    const uint32_t raw_addr = smem_u32(raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;  // swizzle atoms
    uint8_t* const stages = raw + (base - raw_addr);
    float* const staging = reinterpret_cast<float*>(stages + S::kStagingAt);
    float* const col_scale = reinterpret_cast<float*>(stages + S::kStages * S::kStageBytes);
    float* const col_bias = col_scale + kTileN;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(col_bias + kTileN);  // full, empty, done
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S::kStages + 1);
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages, done = empty + 8 * S::kStages;
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

    const int rank = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = blockIdx.x / splits;
    const int tiles_n = (a.n + kTileN - 1) / kTileN;
    const int row0 = tile / tiles_n * kTileM, col0 = tile % tiles_n * kTileN;
    const int blocks = (a.k + kTileK - 1) / kTileK;
    const int share = (blocks + splits - 1) / splits;
    const int k0 = min(blocks, rank * share), count = min(blocks, k0 + share) - k0;
    const uint32_t stage_bytes = box_rows * kTileK + kTileN * kTileK;  // what a stage's loads bring

    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(static_cast<uint32_t>(kTileN))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = uniform(*tmem_slot);

    bool good = true;
    if (warp == 0 || warp == 2) {
        // One warp loads w, another q, since a load takes its time to issue.  The first
        // weights come while the rows are still being quantised.
        const bool rows = warp == 2;
        if (rows || !weights_ready) wait_for_previous();
        for (int i = 0; i < count && good; ++i) {
            const int s = i % S::kStages;
            good = i < S::kStages || mbar_wait(empty + 8 * s, (i / S::kStages - 1) & 1);
            if (good && elect_one()) {
                const uint32_t stage = base + s * S::kStageBytes;
                if (rows) {
                    tma_load_2d(stage, &map_q, (k0 + i) * kTileK, row0, full + 8 * s);
                } else {
                    mbar_expect_tx(full + 8 * s, stage_bytes);
                    tma_load_2d(stage + kABytes, &map_w, (k0 + i) * kTileK, col0, full + 8 * s);
                }
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        for (int i = 0; i < count && good; ++i) {
            const int s = i % S::kStages;
            good = mbar_wait(full + 8 * s, (i / S::kStages) & 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (good && elect_one()) {
                const uint64_t qd = k_major_desc(base + s * S::kStageBytes);
                const uint64_t wd = k_major_desc(base + s * S::kStageBytes + kABytes);
#pragma unroll
                for (int j = 0; j < kTileK / 32; ++j)  // (a descriptor counts in 16 bytes)
                    mma_i8<1>(tmem, qd + 2 * j, wd + 2 * j, int8_idesc(kTileM, kTileN), (i | j) != 0 ? 1u : 0u);
                if (i + S::kStages < count) commit_one(empty + 8 * s);  // the stage is loaded again
                if (i + 1 == count) commit_one(done);
            }
            __syncwarp();
        }
    } else {
        for (int c = lane; c < kTileN; c += 32) {
            const bool in = col0 + c < a.n;
            col_scale[c] = in ? a.w_scales[col0 + c] : 0.0f;
            col_bias[c] = in && a.bias != nullptr ? a.bias[col0 + c] : 0.0f;
        }
    }
    __syncwarp();
    wait_for_previous();  // the rows' scales
    const int own_row = row0 + warp * 32 + lane;
    const float own_scale = splits == 1 && own_row < a.m ? a.scales[own_row] : 0.0f;
    good = count == 0 || mbar_wait(done, 0);
    __syncthreads();  // the columns' scales
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float* const stage = staging + warp * 32 * (32 + kStagePad);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    if (splits == 1) {
        const float row_scale = good ? own_scale : NAN;
#pragma unroll 1
        for (int c0 = 0; c0 < kTileN && col0 + c0 < a.n; c0 += 32) {
            uint32_t sum[32];
            float v[32];
            tmem_ld32(lanes + c0, sum);
            if (count == 0)
#pragma unroll
                for (int c = 0; c < 32; ++c) sum[c] = 0;
            results(sum, row_scale, col_scale + c0, col_bias + c0, v);
            store_block<Out>(stage, v, a, row0 + warp * 32, col0 + c0, vector_ok);
        }
    } else {
        // partial sums as [column][row], over the stages that are no longer needed
        int* const part = reinterpret_cast<int*>(stages);
#pragma unroll 1
        for (int c0 = 0; c0 < kTileN; c0 += 32) {
            uint32_t sum[32];
            tmem_ld32(lanes + c0, sum);
#pragma unroll
            for (int c = 0; c < 32; ++c) part[(c0 + c) * kTileM + warp * 32 + lane] = count > 0 ? static_cast<int>(sum[c]) : 0;
        }
        int* const failed = reinterpret_cast<int*>(tmem_slot + 1);
        if (tid == 0) *failed = 0;
        __syncthreads();
        if (!good) *failed = 1;
        cluster_sync();
        // the tile's 4 row groups x kTileN / 32 column groups, dealt out over the cluster's warps
        const uint32_t mine = smem_u32(part), flag = smem_u32(failed);
        for (int job = rank * 4 + warp; job < 4 * (kTileN / 32); job += 4 * splits) {
            const int group = job & 3, c0 = (job >> 2) * 32;
            const int row = row0 + group * 32 + lane;
            if (row0 + group * 32 >= a.m || col0 + c0 >= a.n) continue;
            uint32_t sum[32] = {};
            bool broken = false;
            for (int r = 0; r < splits; ++r) {
                const uint32_t from = map_rank(mine, r);
                broken |= ld_cluster(map_rank(flag, r)) != 0;
#pragma unroll
                for (int c = 0; c < 32; ++c) sum[c] += ld_cluster(from + ((c0 + c) * kTileM + group * 32 + lane) * 4);
            }
            const float row_scale = row < a.m ? (broken ? NAN : a.scales[row]) : 0.0f;
            float v[32];
            results(sum, row_scale, col_scale + c0, col_bias + c0, v);
            store_block<Out>(stage, v, a, row0 + group * 32, col0 + c0, vector_ok);
        }
        cluster_sync();  // no CTA leaves while another reads its sums
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (!good && tid == 0)  // copies in flight end before the memory is given back
        for (int s = 0; s < min(count, S::kStages); ++s) mbar_wait(full + 8 * s, ((count - 1 - s) / S::kStages) & 1);
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(kTileN))
                     : "memory");
}

// ------------------------------------------------------------------ a pair of CTAs on 256 x 256 tiles
// The lane's row of a block that leaves by TMA, columns h .. h + 31: 16-byte units
// in the 128-byte swizzle, which keeps 8 lanes of a store on different banks.
template <typename Out>
__device__ __forceinline__ void stage_row(uint8_t* stage, int h, const float* v) {
    constexpr int kVec = 16 / sizeof(Out);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 32; c += kVec) {
        uint4 unit;
        if constexpr (sizeof(Out) == 4) {
            unit = make_uint4(__float_as_uint(v[c]), __float_as_uint(v[c + 1]), __float_as_uint(v[c + 2]), __float_as_uint(v[c + 3]));
        } else {
            uint32_t* const p = reinterpret_cast<uint32_t*>(&unit);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[c + 2 * i], v[c + 2 * i + 1]);
                p[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
        *reinterpret_cast<uint4*>(stage + lane * 128 + (((h + c) / kVec) ^ (lane & 7)) * 16) = unit;
    }
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n cp.async.bulk.commit_group;" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(x), "r"(y), "r"(src)
        : "memory");
}
__device__ __forceinline__ void wait_for_stores_to_be_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

constexpr int kPairN = 256;
constexpr uint32_t kPairStageBytes = 2 * kABytes;  // 128 rows of q, 128 rows of w
constexpr uint32_t kWarpStaging = 5 * 1024;        // of an epilogue warp: 32 rows of 128 bytes, or of 32 + kStagePad floats
constexpr int kGroupM = 8;                         // tiles of rows that run next to one another, for L2
// kManyLong, for tiles of long k that come one after the other: as many stages as
// fit, and the four epilogue warps that the MMAs hide; otherwise eight.
template <bool kManyLong>
struct PairShape {
    static constexpr int kStages = kManyLong ? 6 : 5;
    static constexpr int kEpilogueWarps = kManyLong ? 4 : 8;  // for each quarter of the TMEM lanes one, or two with half of the columns each
    static constexpr int kWarpCols = kPairN * 4 / kEpilogueWarps;
    static constexpr int kThreads = 64 + 32 * kEpilogueWarps;  // TMA, MMA, epilogue
    static constexpr uint32_t kSmem = kStages * kPairStageBytes + kEpilogueWarps * kWarpStaging + 2 * kPairN * 4 + 256 + 1024;
};

template <bool kManyLong, typename Out>
__global__ void __launch_bounds__(PairShape<kManyLong>::kThreads, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_out, const ProductArgs a, bool out_by_tma) {
    using S = PairShape<kManyLong>;
    constexpr int kPairStages = S::kStages, kEpilogueWarps = S::kEpilogueWarps, kWarpCols = S::kWarpCols;
    extern __shared__ uint8_t raw[];
    const uint32_t raw_addr = smem_u32(raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* const stages = raw + (base - raw_addr);
    uint8_t* const staging = stages + kPairStages * kPairStageBytes;
    float* const col_scale = reinterpret_cast<float*>(staging + kEpilogueWarps * kWarpStaging);
    float* const col_bias = col_scale + kPairN;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(col_bias + kPairN);
    const uint32_t full = smem_u32(bars), empty = full + 8 * kPairStages, tile_full = empty + 8 * kPairStages,
                   tile_empty = tile_full + 16;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kPairStages + 4);
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    const uint32_t rank = cluster_rank();

    if (tid == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tile_full + 8 * b, 1);
            mbar_init(tile_empty + 8 * b, 2 * kEpilogueWarps);  // of both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(2u * kPairN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = uniform(*tmem_slot);
    wait_for_previous();

    const int tiles_m = (a.m + 2 * kTileM - 1) / (2 * kTileM), tiles_n = (a.n + kPairN - 1) / kPairN;
    const int tiles = tiles_m * tiles_n;
    const int blocks = (a.k + kTileK - 1) / kTileK;
    auto place = [&](int t, int& row0, int& col0) {
        const int group = t / (kGroupM * tiles_n);
        const int first = group * kGroupM, height = min(kGroupM, tiles_m - first);
        const int in = t - group * kGroupM * tiles_n;
        row0 = (first + in % height) * 2 * kTileM + static_cast<int>(rank) * kTileM;
        col0 = in / height * kPairN;
    };
    const int first_tile = blockIdx.x >> 1, step = gridDim.x >> 1;

    bool good = true;
    if (warp == 0) {
        int i = 0;
        for (int t = first_tile; t < tiles && good; t += step) {
            int row0, col0;
            place(t, row0, col0);
            for (int kb = 0; kb < blocks && good; ++kb, ++i) {
                const int s = i % kPairStages;
                good = i < kPairStages || mbar_wait(empty + 8 * s, (i / kPairStages - 1) & 1);
                if (good && elect_one()) {
                    if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * kPairStageBytes);
                    const uint32_t bar = map_rank(full + 8 * s, 0), dst = base + s * kPairStageBytes;
                    tma_load_pair(dst, &map_q, kb * kTileK, row0, bar);
                    tma_load_pair(dst + kABytes, &map_w, kb * kTileK, col0 + static_cast<int>(rank) * kTileM, bar);
                }
                __syncwarp();
            }
        }
        // without a failure every copy was consumed; after one the last of each stage is waited for
        if (!good && rank == 0)
            for (int j = max(0, i - kPairStages); j < i; ++j) mbar_wait(full + 8 * (j % kPairStages), (j / kPairStages) & 1);
    } else if (warp == 1 && rank == 0) {
        int i = 0;
        for (int t = first_tile, n = 0; t < tiles && good; t += step, ++n) {
            const int b = n & 1;
            good = n < 2 || mbar_wait(tile_empty + 8 * b, (n / 2 - 1) & 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int kb = 0; kb < blocks && good; ++kb, ++i) {
                const int s = i % kPairStages;
                good = mbar_wait(full + 8 * s, (i / kPairStages) & 1);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (good && elect_one()) {
                    const uint64_t qd = k_major_desc(base + s * kPairStageBytes);
                    const uint64_t wd = k_major_desc(base + s * kPairStageBytes + kABytes);
#pragma unroll
                    for (int j = 0; j < kTileK / 32; ++j)  // (a descriptor counts in 16 bytes)
                        mma_i8<2>(tmem + b * kPairN, qd + 2 * j, wd + 2 * j, int8_idesc(2 * kTileM, kPairN),
                                  (kb | j) != 0 ? 1u : 0u);
                    commit_pair(empty + 8 * s);
                    if (kb + 1 == blocks) commit_pair(tile_full + 8 * b);
                }
                __syncwarp();
            }
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3;  // the TMEM lanes this warp may read
        const int first_col = (warp - 2) / 4 * kWarpCols;
        uint8_t* const stage = staging + (warp - 2) * kWarpStaging;
        const uint32_t stage_address = smem_u32(stage);
        constexpr int kBlockCols = 128 / sizeof(Out);  // a block that leaves by TMA: 32 rows of 128 bytes
        for (int t = first_tile, n = 0; t < tiles; t += step, ++n) {
            const int b = n & 1;
            int row0, col0;
            place(t, row0, col0);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");  // the last tile's scales are read
            for (int c = tid - 64; c < kPairN; c += 32 * kEpilogueWarps) {
                const bool in = col0 + c < a.n;
                col_scale[c] = in ? a.w_scales[col0 + c] : 0.0f;
                col_bias[c] = in && a.bias != nullptr ? a.bias[col0 + c] : 0.0f;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");
            const int row = row0 + quarter * 32 + lane;
            const float own_scale = row < a.m ? a.scales[row] : 0.0f;
            good = good && mbar_wait(tile_full + 8 * b, (n / 2) & 1);
            good = __all_sync(0xffffffffu, good);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float row_scale = good ? own_scale : NAN;
            const uint32_t lanes = tmem + b * kPairN + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int c0 = first_col; c0 < first_col + kWarpCols && col0 + c0 < a.n; c0 += kBlockCols) {
                uint32_t sum[32];
                float v[32];
                wait_for_stores_to_be_read();  // of the block before
                __syncwarp();
                // a TMA store writes whole 16-byte units, so the last columns go by it only where they fill theirs
                if (!out_by_tma || (col0 + c0 + kBlockCols > a.n && a.n % (16 / sizeof(Out)) != 0)) {
#pragma unroll 1
                    for (int h = 0; h < kBlockCols && col0 + c0 + h < a.n; h += 32) {
                        tmem_ld32(lanes + c0 + h, sum);
                        results(sum, row_scale, col_scale + c0 + h, col_bias + c0 + h, v);
                        store_block<Out>(reinterpret_cast<float*>(stage), v, a, row0 + quarter * 32, col0 + c0 + h, out_by_tma);
                    }
                    continue;
                }
#pragma unroll
                for (int h = 0; h < kBlockCols; h += 32) {
                    tmem_ld32(lanes + c0 + h, sum);
                    results(sum, row_scale, col_scale + c0 + h, col_bias + c0 + h, v);
                    stage_row<Out>(stage, h, v);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0 && row0 + quarter * 32 < a.m) tma_store_2d(&map_out, stage_address, col0 + c0, row0 + quarter * 32);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 map_rank(tile_empty + 8 * b, 0))
                             : "memory");
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync();  // neither CTA leaves while the other's copies, MMAs or arrivals reach it
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * kPairN) : "memory");
}

// ------------------------------------------------------------------ host
// rows x k bytes in boxes of box_rows x 128 bytes.  (With k = 0 nothing is
// loaded, but a map has no empty dimension.)
int operand_map(CUtensorMap* map, const int8_t* data, int rows, int k, size_t stride, int box_rows) {
    const EncodeTiled fn = encode_tiled();
    if (fn == nullptr) return fail_message("cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(std::max(k, 1)), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
    const cuuint32_t box[2] = {kTileK, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estride[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(data), dims, strides, box, estride,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail_messagef("cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return 0;
}

// The results in blocks of 32 rows x 128 bytes; the rows and 16-byte units beyond are not written.
template <typename Out>
int result_map(CUtensorMap* map, const ProductArgs& a) {
    const EncodeTiled fn = encode_tiled();
    if (fn == nullptr) return fail_message("cuTensorMapEncodeTiled is unavailable");
    const size_t stride = a.m > 1 ? a.out_stride * sizeof(Out) : (a.n * sizeof(Out) + 15) / 16 * 16;  // of one row: any
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.n), static_cast<cuuint64_t>(a.m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
    const cuuint32_t box[2] = {128 / sizeof(Out), 32};
    const cuuint32_t estride[2] = {1, 1};
    const CUresult r = fn(map, sizeof(Out) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.out, dims,
                          strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail_messagef("cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return 0;
}

template <bool kDeep, typename Out>
int launch_tiles(BulletOuCudaCppContext* ctx, const ProductArgs& a, int64_t tiles, int splits, bool vector_ok, bool early, bool weights_ready) {
    using S = TileShape<kDeep>;
    CUtensorMap q, w;
    // few rows are loaded as they are: the rest of the tile is what the stage
    // held before and reaches no result
    const int box_rows = std::min(kTileM, (a.m + 7) / 8 * 8);
    if (operand_map(&q, a.q, a.m, a.k, a.q_stride, box_rows) != 0 || operand_map(&w, a.w, a.n, a.k, a.w_stride, kTileN) != 0)
        return -1;
    const LaunchShape shape{dim3(static_cast<unsigned>(tiles * splits)), S::kThreads, S::kSmem, splits, early};
    return launch_kernel(ctx, "int8 product launch", int8_tile_kernel<kDeep, Out>, shape, q, w, a, splits, box_rows, vector_ok, weights_ready);
}

template <typename Out>
int launch_tiles(BulletOuCudaCppContext* ctx, const ProductArgs& a, bool vector_ok, bool early, bool weights_ready) {
    const int64_t tiles = static_cast<int64_t>((a.m + kTileM - 1) / kTileM) * ((a.n + kTileN - 1) / kTileN);
    const int blocks = (a.k + kTileK - 1) / kTileK;
    int splits = 1;
    while (splits < 4 && tiles * splits * 2 <= ctx->sm_count && blocks >= 16 * splits) splits *= 2;
    if (tiles * splits > INT32_MAX) return fail_messagef("int8 product: %d x %d results are too many", a.m, a.n);
    return tiles * splits <= ctx->sm_count ? launch_tiles<true, Out>(ctx, a, tiles, splits, vector_ok, early, weights_ready)
                                           : launch_tiles<false, Out>(ctx, a, tiles, splits, vector_ok, early, weights_ready);
}

template <bool kManyLong, typename Out>
int launch_pairs(BulletOuCudaCppContext* ctx, const ProductArgs& a, int tiles, bool vector_ok, bool early) {
    CUtensorMap q, w, out{};
    if (operand_map(&q, a.q, a.m, a.k, a.q_stride, kTileM) != 0 || operand_map(&w, a.w, a.n, a.k, a.w_stride, kTileM) != 0)
        return -1;
    if (vector_ok && result_map<Out>(&out, a) != 0) return -1;
    const LaunchShape shape{dim3(2 * std::min(tiles, ctx->sm_count / 2)), PairShape<kManyLong>::kThreads, PairShape<kManyLong>::kSmem, 2, early};
    return launch_kernel(ctx, "int8 product launch", int8_pair_kernel<kManyLong, Out>, shape, q, w, out, a, vector_ok);
}

template <typename Out>
int launch_typed(BulletOuCudaCppContext* ctx, const ProductArgs& a, bool early, bool weights_ready) {
    const bool vector_ok = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && (a.m <= 1 || a.out_stride * sizeof(Out) % 16 == 0);
    // Single tiles while they all run at once, two on an SM: 512 x 4096 x 4096 (256 of
    // them) takes 15 us, in pairs 18; 8192 x 640 x 256 (256) 6.0 and 9.0.  Beyond,
    // pairs, unless most of their columns are empty: 16384 x 2560 x 256 (512) takes
    // 13 us in pairs, 17 singly, but 65536 x 640 x 64 16 and 10.  Without inner columns
    // there is no MMA whose end a pair could wait for; a single tile takes its sums as zeros.
    const int64_t pairs = static_cast<int64_t>((a.m + 255) / 256) * ((a.n + 255) / 256);
    const int64_t singles = static_cast<int64_t>((a.m + 127) / 128) * ((a.n + 63) / 64);
    if (a.k > 0 && a.n > 64 && singles > 2 * ctx->sm_count && pairs <= INT32_MAX)
        // 16384 x 4096 x 4096 takes 197 us with six stages, 206 with five; 4096 x 8192 x
        // 2048 (two tiles for each pair) 67 and 66, 8192 x 1024 x 4096 44 and 41
        return a.k >= 2048 && pairs >= 4 * ctx->sm_count / 2 ? launch_pairs<true, Out>(ctx, a, static_cast<int>(pairs), vector_ok, early)
                                                             : launch_pairs<false, Out>(ctx, a, static_cast<int>(pairs), vector_ok, early);
    return launch_tiles<Out>(ctx, a, vector_ok, early, weights_ready);
}

}  // namespace

int launch_int8_mma(BulletOuCudaCppContext* ctx, const ProductArgs& a, int out_type, bool after_quantise, bool weights_ready) {
    return out_type == BULLETOU_B200_TYPE_F32 ? launch_typed<float>(ctx, a, after_quantise, weights_ready)
                                              : launch_typed<__nv_bfloat16>(ctx, a, after_quantise, weights_ready);
}

}  // namespace bou
