// NVFP4 block-scaled matmul for sm_100a: E2M1 operands, one E4M3 scale per 16 elements along K, fp32 accumulation:
//     D[m,n] = round( alpha * sum_k (a[m,k] * sa[m,k/16]) * (b[n,k] * sb[n,k/16]) )
// The products and the scaling happen in the tensor core (tcgen05.mma.kind::mxf4nvf4.block_scale.block16); the scales
// sit in TMEM next to the accumulator, in the order of the tiled scale layout: per 128 rows x 4 blocks (one MMA of 64
// elements along K) a 512-byte block [row % 32][row / 32][4 bytes].
//
//   nvfp4_pack_scales_kernel  scales by rows -> tiled; for a grouped problem also the row-tile table: tiles start at a
//                             group's first row, so their scale blocks do too.
//   nvfp4_pair_kernel         CTA pairs (cta_group::2), tile 256 x 256: prompts.  Tensor-bound.
//   nvfp4_few_kernel          (nvfp4_few.cuh) weights on the M axis, up to 128 rows of A on the N axis: HBM-bound.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx_gemm_pair.cuh"
#include "nvfp4_quantize.cuh"

namespace cb200 {

constexpr int kNvStageK = 256;   // elements along K per stage: 128 bytes per row, four MMAs, four scale words

struct NvParams {
    uint32_t m, n, k;
    uint32_t num_k_blocks;         // stages: ceil(k / 256)
    uint32_t words;                // scale words of 64 elements: ceil(k / 64)
    uint32_t band_rows;            // tile rows per band of the tile order (mx_tile_coords)
    uint32_t sfb_blocks;           // 128-row scale blocks of B per group: ceil(n / 128)
    uint32_t d_type;               // 0 fp32, 1 bf16, 2 fp16
    const uint8_t* sfa;            // tiled scales of A, one block per 128 rows of a row tile
    const uint8_t* sfb;            // tiled scales of B
    const float* alpha;            // [1] or [groups], or nullptr
    void* d;
    unsigned* status;
    const int4* table;             // grouped: [row tile] = (first row, one past the group's last row, group, 0)
    const uint32_t* num_row_tiles; // grouped: entries of the table
    uint32_t tma_store;            // pair kernel: D has a tensor map
};

// Instruction descriptor of kind::mxf4nvf4 with E4M3 scales (bit 23 = 0); with 16-element blocks an MMA uses all four
// bytes of a scale column, the byte selectors stay 0.
__host__ __device__ constexpr uint32_t make_idesc_nv(uint32_t m, uint32_t n)
{
    return (kFmtMxf4E2M1 << 7) | (kFmtMxf4E2M1 << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int kCtaGroup>
__device__ __forceinline__ void umma_nv(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                        uint32_t accumulate, uint32_t sfa, uint32_t sfb)
{
    if constexpr (kCtaGroup == 1) {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t"
            "}\n" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
            : "memory");
    } else {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t"
            "}\n" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
            : "memory");
    }
}

// ---------------------------------------------------------------- scales by rows -> tiled, row-tile table

struct NvPackParams {
    const uint8_t* in;         // [batch][rows][blocks]
    uint8_t* out;              // [batch][row blocks][words][512]
    uint32_t rows, blocks, words;
    uint64_t in_batch, out_batch;
    // grouped A (group_list != nullptr; one batch): out block tile * (tile_rows / 128) + i holds rows
    // [first row of the tile + 128 i, ...) of the tile's group
    const void* group_list;
    uint32_t list_i32, list_prefix, groups, tile_rows;
    int4* table;
    uint32_t* num_row_tiles;
};

constexpr int kNvPackThreads = 256;

// A group's rows [begin, end), clamped to `rows` and never decreasing, and its first row tile, in shared memory:
// s_end[g], s_tile[g] (s_tile[groups] = number of tiles).  All threads of the CTA take part.
__device__ __forceinline__ void nv_group_tiles(const NvPackParams& p, uint32_t* s_end, uint32_t* s_tile)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        int64_t prev = 0;       // end of the groups before this batch of 32
        uint32_t tiles = 0;
        for (uint32_t g0 = 0; g0 < p.groups; g0 += 32) {
            const uint32_t g = g0 + lane;
            int64_t v = 0;
            if (g < p.groups) {
                v = p.list_i32 ? static_cast<int64_t>(static_cast<const int32_t*>(p.group_list)[g])
                               : static_cast<const int64_t*>(p.group_list)[g];
            }
            if (!p.list_prefix) {
                v = v < 0 ? 0 : (v < static_cast<int64_t>(p.rows) ? v : static_cast<int64_t>(p.rows));
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int64_t below = __shfl_up_sync(0xffffffffu, v, off);
                    v += lane >= static_cast<uint32_t>(off) ? below : 0;
                }
                v += prev;
            } else {  // a running maximum: a prefix sum that falls leaves an empty group
                v = v > prev ? v : prev;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int64_t below = __shfl_up_sync(0xffffffffu, v, off);
                    v = lane >= static_cast<uint32_t>(off) && below > v ? below : v;
                }
            }
            const uint32_t end = v < static_cast<int64_t>(p.rows) ? static_cast<uint32_t>(v) : p.rows;
            uint32_t begin = __shfl_up_sync(0xffffffffu, end, 1);
            begin = lane == 0 ? static_cast<uint32_t>(prev) : begin;
            uint32_t count = g < p.groups ? (end - begin + p.tile_rows - 1) / p.tile_rows : 0u;
            const uint32_t own = count;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t below = __shfl_up_sync(0xffffffffu, count, off);
                count += lane >= static_cast<uint32_t>(off) ? below : 0u;
            }
            if (g < p.groups) {
                s_end[g] = end;
                s_tile[g] = tiles + count - own;
            }
            // (lanes past the last group repeat its end, so lane 31 always carries on)
            prev = __shfl_sync(0xffffffffu, end, p.groups - g0 >= 32 ? 31 : static_cast<int>(p.groups - g0 - 1));
            tiles += __shfl_sync(0xffffffffu, count, 31);
        }
        if (lane == 0) {
            s_tile[p.groups] = tiles;
        }
    }
    __syncthreads();
}

// blockIdx.y walks the batch.  A thread moves four words (64 elements each) of one row: 16 bytes in, four 4-byte
// stores 512 bytes apart out.
__global__ void __launch_bounds__(kNvPackThreads)
nvfp4_pack_scales_kernel(const NvPackParams p)
{
    __shared__ uint32_t s_end[kMaxGroups];
    __shared__ uint32_t s_tile[kMaxGroups + 1];
    grid_launch_dependents();
    const uint8_t* in = p.in + blockIdx.y * p.in_batch;
    uint8_t* out = p.out + blockIdx.y * p.out_batch;
    const bool grouped = p.group_list != nullptr;
    uint32_t row_blocks = (p.rows + 127u) / 128u;
    const uint32_t per_tile = grouped ? p.tile_rows / 128u : 1u;
    if (grouped) {
        nv_group_tiles(p, s_end, s_tile);
        row_blocks = s_tile[p.groups] * per_tile;
        if (blockIdx.x == 0) {
            for (uint32_t g = threadIdx.x; g < p.groups; g += kNvPackThreads) {
                const uint32_t begin = g == 0 ? 0u : s_end[g - 1];
                for (uint32_t t = s_tile[g]; t < s_tile[g + 1]; ++t) {
                    p.table[t] = make_int4(static_cast<int>(begin + (t - s_tile[g]) * p.tile_rows),
                                           static_cast<int>(s_end[g]), static_cast<int>(g), 0);
                }
            }
            if (threadIdx.x == 0) {
                *p.num_row_tiles = s_tile[p.groups];
            }
        }
    }
    const uint32_t quads = (p.words + 3) / 4;
    const uint64_t items = static_cast<uint64_t>(row_blocks) * 128u * quads;
    const bool vec = (p.blocks & 15u) == 0 && (reinterpret_cast<uintptr_t>(in) & 15u) == 0;
    for (uint64_t i = blockIdx.x * static_cast<uint64_t>(kNvPackThreads) + threadIdx.x; i < items;
         i += static_cast<uint64_t>(gridDim.x) * kNvPackThreads) {
        const uint32_t prow = static_cast<uint32_t>(i / quads);
        const uint32_t quad = static_cast<uint32_t>(i - static_cast<uint64_t>(prow) * quads);
        uint32_t row = prow, end = p.rows;
        if (grouped) {
            const uint32_t tile = prow / p.tile_rows;
            uint32_t lo = 0, hi = p.groups - 1;  // the group whose tiles hold this one: last g with s_tile[g] <= tile
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) / 2;
                if (s_tile[mid] <= tile) {
                    lo = mid;
                } else {
                    hi = mid - 1;
                }
            }
            row = (lo == 0 ? 0u : s_end[lo - 1]) + (prow - s_tile[lo] * p.tile_rows);
            end = s_end[lo];
        }
        if (row >= end) {
            continue;  // rows that are never stored may have any scale
        }
        const uint8_t* src = in + static_cast<uint64_t>(row) * p.blocks + quad * 16;
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (vec) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            w[0] = v.x;
            w[1] = v.y;
            w[2] = v.z;
            w[3] = v.w;
        } else {
#pragma unroll
            for (uint32_t b = 0; b < 16; ++b) {
                if (quad * 16 + b < p.blocks) {
                    w[b / 4] |= static_cast<uint32_t>(src[b]) << (8 * (b % 4));
                }
            }
        }
        uint8_t* dst = out + nvfp4_tiled_offset(prow, quad * 16, p.words);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (quad * 4 + j < p.words) {
                *reinterpret_cast<uint32_t*>(dst + j * 512) = w[j];
            }
        }
    }
}

// ---------------------------------------------------------------- CTA pairs, 256 x 256 tiles

constexpr int kNvPairStages = 5;
constexpr int kNvPairCopiers = 4;
constexpr int kNvPairEpiWarps = 16;
// warps: 0 operand producer, 1 MMA issuer, 2 scale producer, 3-6 scale copiers, 7-22 epilogue
constexpr int kNvPairThreads = (3 + kNvPairCopiers + kNvPairEpiWarps) * 32;

struct NvPairSmem {
    static constexpr int kABytes = kBlockM * kBlockKBytes;          // 16 KB: this CTA's 128 rows of A
    static constexpr int kBBytes = (kMxBlockN / 2) * kBlockKBytes;  // 16 KB: this CTA's half of B
    static constexpr int kSfBytes = 3 * 2048;                       // four words each of A, B block 0, B block 1
    static constexpr int kStageBytes = kABytes + kBBytes + kSfBytes;
    static constexpr int kRingBytes = kNvPairStages * kStageBytes;
    static constexpr int kBarriers = 3 * kNvPairStages + 2;
    // D leaves through a slab per epilogue warp: 32 rows x 64 bytes for a TMA store (64-byte swizzle, so slabs start on
    // 512-byte boundaries), or, where D's rows do not start on 16-byte boundaries, 32 rows 17 words apart (an odd
    // number: rows fall on different banks)
    static constexpr int kSlabBytes = 2048;
    static constexpr int kOddSlabBytes = 32 * 17 * 4;
    static constexpr int kSlabOffset = kRingBytes;
    static constexpr int kBarrierOffset = kSlabOffset + kNvPairEpiWarps * kOddSlabBytes;
    static constexpr int kTotalBytes = 1024 + kBarrierOffset + kBarriers * 8 + 16;
};
static_assert(NvPairSmem::kTotalBytes <= 227 * 1024, "shared memory budget");
static_assert(NvPairSmem::kStageBytes % 1024 == 0, "swizzled tiles start on 1 KB boundaries");
static_assert(NvPairSmem::kBarrierOffset % 8 == 0 && NvPairSmem::kSlabBytes <= NvPairSmem::kOddSlabBytes, "slabs");

// One row's `kCount` accumulator columns (fp32 bit patterns) starting at col, times alpha, to D.
template <int kCount>
__device__ __forceinline__ void nv_store_row(const NvParams& p, const uint32_t (&r)[kCount], uint32_t row, uint32_t col,
                                             float alpha)
{
    const uint64_t at = static_cast<uint64_t>(row) * p.n + col;
    const bool whole = col + kCount <= p.n;
    if (p.d_type == 0) {
        float* d = static_cast<float*>(p.d) + at;
        if (whole && (p.n & 3u) == 0) {
#pragma unroll
            for (int v = 0; v < kCount / 4; ++v) {
                reinterpret_cast<float4*>(d)[v] =
                    make_float4(__uint_as_float(r[4 * v]) * alpha, __uint_as_float(r[4 * v + 1]) * alpha,
                                __uint_as_float(r[4 * v + 2]) * alpha, __uint_as_float(r[4 * v + 3]) * alpha);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                if (col + i < p.n) {
                    d[i] = __uint_as_float(r[i]) * alpha;
                }
            }
        }
        return;
    }
    const bool f16 = p.d_type == 2;
    uint16_t* d = static_cast<uint16_t*>(p.d) + at;
    uint32_t packed[kCount / 2];
#pragma unroll
    for (int i = 0; i < kCount / 2; ++i) {
        packed[i] = pack_out2(__uint_as_float(r[2 * i]) * alpha, __uint_as_float(r[2 * i + 1]) * alpha, f16);
    }
    if (whole && (p.n & 7u) == 0) {
#pragma unroll
        for (int v = 0; v < kCount / 8; ++v) {
            reinterpret_cast<uint4*>(d)[v] =
                make_uint4(packed[4 * v], packed[4 * v + 1], packed[4 * v + 2], packed[4 * v + 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCount / 2; ++i) {
            if (col + 2 * i < p.n) {
                d[2 * i] = static_cast<uint16_t>(packed[i]);
            }
            if (col + 2 * i + 1 < p.n) {
                d[2 * i + 1] = static_cast<uint16_t>(packed[i] >> 16);
            }
        }
    }
}

// The same for a whole warp (lane = row, rows row0 + lane < row_end), every store instruction covering 32 consecutive
// columns of one row: for rows of D that start anywhere.  One row per lane there means 32 two-byte pieces of 32 rows per
// instruction (4111 x 515 x 7168: 61 us, against 24 us this way).  All lanes take part.
__device__ __forceinline__ void nv_store_rows_staged(const NvParams& p, const uint32_t (&r)[32], uint32_t* slab,
                                                     uint32_t row0, uint32_t row_end, uint32_t col, float alpha,
                                                     uint32_t lane)
{
    const uint32_t rows = row0 >= row_end ? 0u : (row_end - row0 < 32u ? row_end - row0 : 32u);
    if (p.d_type == 0) {
        for (uint32_t h = 0; h < 2; ++h) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                slab[lane * 17 + i] = __float_as_uint(__uint_as_float(h == 0 ? r[i] : r[16 + i]) * alpha);
            }
            __syncwarp();
            const uint32_t c = col + h * 16 + (lane & 15u);  // two rows per step
            for (uint32_t q = lane >> 4; q < rows; q += 2) {
                if (c < p.n) {
                    static_cast<uint32_t*>(p.d)[static_cast<uint64_t>(row0 + q) * p.n + c] = slab[q * 17 + (lane & 15u)];
                }
            }
        }
        return;
    }
    const bool f16 = p.d_type == 2;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        slab[lane * 17 + i] = pack_out2(__uint_as_float(r[2 * i]) * alpha, __uint_as_float(r[2 * i + 1]) * alpha, f16);
    }
    __syncwarp();
    const uint16_t* half = reinterpret_cast<const uint16_t*>(slab) + lane;
    if (col + lane < p.n) {
        uint16_t* d = static_cast<uint16_t*>(p.d) + static_cast<uint64_t>(row0) * p.n + col + lane;
#pragma unroll 8
        for (uint32_t q = 0; q < rows; ++q) {
            d[static_cast<uint64_t>(q) * p.n] = half[q * 34];
        }
    }
}

// A warp's 32 rows x 64 bytes of D (kCount columns from r, times alpha) by one TMA store.  Every store instruction of the
// row-per-lane form above touches 32 rows, 16 bytes each; 256 x 256 tiles took 1.8 us longer that way, and the last one 3.6.
// The slab's previous store has been read (the caller waits).  All lanes take part; the rows are all to be stored.
template <int kCount>
__device__ __forceinline__ void nv_tma_store(const NvParams& p, const CUtensorMap* tmap_d, const uint32_t* r, uint8_t* slab,
                                             uint32_t row0, uint32_t col, float alpha, uint32_t lane)
{
    uint8_t* row = slab + lane * 64;
    const uint32_t swizzle = (lane >> 1) & 3u;
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kCount == 16) {
                w[i] = __float_as_uint(__uint_as_float(r[4 * c + i]) * alpha);
            } else {
                w[i] = pack_out2(__uint_as_float(r[8 * c + 2 * i]) * alpha, __uint_as_float(r[8 * c + 2 * i + 1]) * alpha,
                                 p.d_type == 2);
            }
        }
        *reinterpret_cast<uint4*>(row + ((c ^ swizzle) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_2d(tmap_d, smem_u32(slab), static_cast<int32_t>(col * (64 / kCount)), static_cast<int32_t>(row0));
        tma_store_commit();
    }
}

// The lane that issues a warp's stores waits until they have read the slab; then the warp may write it again.
__device__ __forceinline__ void nv_slab_free(uint32_t lane)
{
    if (lane == 0) {
        tma_store_wait_read<0>();
    }
    __syncwarp();
}

// tmap_b: {row bytes, n, groups}, boxes of 128 rows; tmap_sfa / tmap_sfb: the tiled scales as {256, 2 * words, row
// blocks}, boxes of {256, 8, 1} = four words; words past the last read as zero; tmap_d: D as bytes, boxes of
// 64 bytes x 32 rows (p.tma_store).
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNvPairThreads, 1)
nvfp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ CUtensorMap tmap_sfa, const __grid_constant__ CUtensorMap tmap_sfb,
                  const __grid_constant__ CUtensorMap tmap_d, const NvParams p)
{
    using S = NvPairSmem;
    constexpr int kStages = kNvPairStages;
    constexpr uint32_t kAccCols = kMxBlockN;
    constexpr uint32_t kSfSlot = 48;  // one scale slot: A 16 columns, B 32
    constexpr uint32_t kTmemCols = 512;
    static_assert(kAccCols + kStages * kSfSlot <= kTmemCols, "TMEM budget");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t* smem = smem_raw + pad;
    const uint32_t ring = raw_addr + pad;
    uint64_t* s_bars = reinterpret_cast<uint64_t*>(smem + S::kBarrierOffset);
    const uint32_t bar_full = smem_u32(s_bars);               // leader: operands and scales of both CTAs landed
    const uint32_t bar_empty = bar_full + kStages * 8;        // both: the stage's MMAs completed
    const uint32_t bar_sf_full = bar_empty + kStages * 8;     // leader: scales copied into both TMEMs
    const uint32_t bar_tmem_full = bar_sf_full + kStages * 8; // both: accumulator complete
    const uint32_t bar_tmem_empty = bar_tmem_full + 8;        // leader: accumulator read by both epilogues
    uint32_t* s_tmem_ptr = reinterpret_cast<uint32_t*>(s_bars + S::kBarriers);
    volatile uint32_t* s_abort = s_tmem_ptr + 1;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta_rank = cluster_ctarank();  // 0 = leader
    const uint32_t pair = blockIdx.x >> 1;
    const uint32_t num_pairs = gridDim.x >> 1;
    const bool grouped = p.table != nullptr;

    if (threadIdx.x == 0) {
        *s_abort = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
            mbar_init(bar_sf_full + s * 8, kNvPairCopiers);
        }
        mbar_init(bar_tmem_full, 1);
        mbar_init(bar_tmem_empty, 2 * kNvPairEpiWarps);
        fence_mbar_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        prefetch_tmap(&tmap_sfa);
        prefetch_tmap(&tmap_sfb);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(s_tmem_ptr), kTmemCols);
        tmem_relinquish<2>();
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are initialised and their TMEM allocated before any cross-CTA signal
    tcgen05_fence_after();
    const uint32_t tmem_base = *s_tmem_ptr;
    grid_launch_dependents();
    grid_dependency_wait();  // the packed scales, the table and the operands of the kernels before

    const uint32_t m_tiles = grouped ? *p.num_row_tiles : (p.m + 2 * kBlockM - 1) / (2 * kBlockM);
    const uint32_t n_tiles = (p.n + kMxBlockN - 1) / kMxBlockN;
    const uint32_t total_tiles = m_tiles * n_tiles;
    const uint32_t num_kb = p.num_k_blocks;
    auto row_tile = [&](uint32_t mt, int32_t& row0, int32_t& row_end, int32_t& group) {
        if (grouped) {
            const int4 e = __ldg(p.table + mt);
            row0 = e.x;
            row_end = e.y;
            group = e.z;
        } else {
            row0 = static_cast<int32_t>(mt) * 2 * kBlockM;
            row_end = static_cast<int32_t>(p.m);
            group = 0;
        }
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- operand producer (both CTAs)
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                uint32_t mt, nt;
                mx_tile_coords(idx, m_tiles, n_tiles, p.band_rows, mt, nt);
                int32_t tile_row0, row_end, group;
                row_tile(mt, tile_row0, row_end, group);
                const int32_t row0 = tile_row0 + static_cast<int32_t>(cta_rank * kBlockM);
                const int32_t col0 = static_cast<int32_t>(nt * kMxBlockN + cta_rank * (kMxBlockN / 2));
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_empty + stage * 8, phase ^ 1, s_abort, p.status, kDevTimeoutProducer);
                    if (!ok) {
                        break;
                    }
                    const uint32_t sa = ring + stage * S::kStageBytes;
                    const int32_t k0 = static_cast<int32_t>(kb) * kBlockKBytes;
                    if (cta_rank == 0) {  // both CTAs' tiles and scale blocks
                        mbar_expect_tx(bar_full + stage * 8, 2 * S::kStageBytes);
                    }
                    const uint32_t full = map_to_cta(bar_full + stage * 8, 0);  // the leader's barrier
                    tma_load_2d_pair(sa, &tmap_a, full, k0, row0);
                    tma_load_3d_pair(sa + S::kABytes, &tmap_b, full, k0, col0, group);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------------------------------------------------------- scale producer (both CTAs)
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                uint32_t mt, nt;
                mx_tile_coords(idx, m_tiles, n_tiles, p.band_rows, mt, nt);
                int32_t tile_row0, row_end, group;
                row_tile(mt, tile_row0, row_end, group);
                const int32_t block_a = static_cast<int32_t>(2 * mt + cta_rank);
                const int32_t block_b = group * static_cast<int32_t>(p.sfb_blocks) + static_cast<int32_t>(2 * nt);
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_empty + stage * 8, phase ^ 1, s_abort, p.status, kDevTimeoutProducer);
                    if (!ok) {
                        break;
                    }
                    const uint32_t ssf = ring + stage * S::kStageBytes + S::kABytes + S::kBBytes;
                    const uint32_t full = map_to_cta(bar_full + stage * 8, 0);
                    const int32_t w2 = static_cast<int32_t>(kb * 8);  // rows of 256 bytes, two per word
                    // (a block past the last, of A or of B, reads zeros or another group's scales: its rows and
                    // columns are not stored)
                    tma_load_3d_pair(ssf, &tmap_sfa, full, 0, w2, block_a);
                    tma_load_3d_pair(ssf + 2048, &tmap_sfb, full, 0, w2, block_b);
                    tma_load_3d_pair(ssf + 4096, &tmap_sfb, full, 0, w2, block_b + 1);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer (leader CTA only)
        if (lane == 0 && cta_rank == 0) {
            constexpr uint32_t idesc = make_idesc_nv(2 * kBlockM, kMxBlockN);
            uint32_t stage = 0, phase = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                ok = mbar_wait(bar_tmem_empty, acc_phase ^ 1, s_abort, p.status, kDevTimeoutMmaTmem);
                if (!ok) {
                    break;
                }
                tcgen05_fence_after();
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    // (the copiers waited for "full" before they copied, and their commit orders this thread behind it)
                    ok = mbar_wait(bar_sf_full + stage * 8, phase, s_abort, p.status, kDevTimeoutMma);
                    if (!ok) {
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t sa = ring + stage * S::kStageBytes;
                    const uint32_t sb = sa + S::kABytes;
                    const uint32_t t_sfa = tmem_base + kAccCols + stage * kSfSlot;
                    const uint32_t t_sfb = t_sfa + 16;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint64_t da = make_smem_desc_sw128(sa + j * 32, 16, 1024);
                        const uint64_t db = make_smem_desc_sw128(sb + j * 32, 16, 1024);
                        umma_nv<2>(tmem_base, da, db, idesc, (kb | j) != 0 ? 1u : 0u, t_sfa + j * 4, t_sfb + j * 8);
                    }
                    umma_commit_pair(bar_empty + stage * 8, 0x3);  // frees the stage and its TMEM slot in both CTAs
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) {
                    break;
                }
                umma_commit_pair(bar_tmem_full, 0x3);
                acc_phase ^= 1;
            }
        }
        __syncwarp();
    } else if (warp < 3 + kNvPairCopiers) {
        // ---------------------------------------------------------------- scale copiers (leader CTA only)
        // Copier w moves word w of the three scale blocks.  Slot `stage` is free when the stage's "full" barrier
        // fires: the MMAs that read it completed before the producers were allowed to refill the stage.
        const uint32_t w = warp - 3;
        if (lane == 0 && cta_rank == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_full + stage * 8, phase, s_abort, p.status, kDevTimeoutConvert);
                    if (!ok) {
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t ssf = ring + stage * S::kStageBytes + S::kABytes + S::kBBytes + w * 512;
                    const uint32_t t_sfa = tmem_base + kAccCols + stage * kSfSlot;
                    const uint32_t t_sfb = t_sfa + 16 + w * 8;
                    tmem_cp_32x128b_warpx4_pair(t_sfa + w * 4, make_smem_desc_noswizzle(ssf, 16, 128));
                    tmem_cp_32x128b_warpx4_pair(t_sfb, make_smem_desc_noswizzle(ssf + 2048, 16, 128));
                    tmem_cp_32x128b_warpx4_pair(t_sfb + 4, make_smem_desc_noswizzle(ssf + 4096, 16, 128));
                    umma_commit<2>(bar_sf_full + stage * 8);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- epilogue: sixteen warps per CTA
        const uint32_t quad = warp & 3;                           // TMEM lane quarter this warp may read
        const uint32_t part = (warp - 3 - kNvPairCopiers) >> 2;   // which 64 columns of the tile's 256
        const bool staged = (p.n & (p.d_type == 0 ? 3u : 7u)) != 0;
        uint8_t* slab = smem + S::kSlabOffset +
                        (warp - 3 - kNvPairCopiers) * (staged ? S::kOddSlabBytes : S::kSlabBytes);
        uint32_t acc_phase = 0;
        bool ok = true;
        for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
            uint32_t mt, nt;
            mx_tile_coords(idx, m_tiles, n_tiles, p.band_rows, mt, nt);
            int32_t tile_row0, row_end, group;
            row_tile(mt, tile_row0, row_end, group);
            const float alpha = p.alpha != nullptr ? __ldg(p.alpha + group) : 1.0f;
            ok = mbar_wait(bar_tmem_full, acc_phase, s_abort, p.status, kDevTimeoutEpilogue);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                break;
            }
            tcgen05_fence_after();
            const uint32_t taddr = tmem_base + part * 64 + ((quad * 32u) << 16);
            uint32_t r[2][32];
            tmem_ld_32x32b_x32(taddr, r[0]);
            tmem_ld_32x32b_x32(taddr + 32, r[1]);
            tmem_ld_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_cluster(bar_tmem_empty, 0);  // this warp's share is in registers
            }
            acc_phase ^= 1;
            const uint32_t row0 = static_cast<uint32_t>(tile_row0) + cta_rank * kBlockM + quad * 32, row = row0 + lane;
            const uint32_t col = nt * kMxBlockN + part * 64;
            if (col >= p.n || row0 >= static_cast<uint32_t>(row_end)) {
                continue;
            }
            if (staged) {
                uint32_t* words = reinterpret_cast<uint32_t*>(slab);
                nv_store_rows_staged(p, r[0], words, row0, static_cast<uint32_t>(row_end), col, alpha, lane);
                if (col + 32 < p.n) {
                    nv_store_rows_staged(p, r[1], words, row0, static_cast<uint32_t>(row_end), col + 32, alpha, lane);
                }
            } else if (p.tma_store && row0 + 32 <= static_cast<uint32_t>(row_end)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (p.d_type == 0) {
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            if (col + h * 32 + f * 16 < p.n) {
                                nv_slab_free(lane);
                                nv_tma_store<16>(p, &tmap_d, r[h] + f * 16, slab, row0, col + h * 32 + f * 16, alpha, lane);
                            }
                        }
                    } else if (col + h * 32 < p.n) {
                        nv_slab_free(lane);
                        nv_tma_store<32>(p, &tmap_d, r[h], slab, row0, col + h * 32, alpha, lane);
                    }
                }
            } else if (row < static_cast<uint32_t>(row_end)) {
                nv_store_row<32>(p, r[0], row, col, alpha);
                if (col + 32 < p.n) {
                    nv_store_row<32>(p, r[1], row, col + 32, alpha);
                }
            }
        }
        if (lane == 0) {
            tma_store_wait_all<0>();
        }
    }

    // Every thread of both CTAs gets here (all waits are bounded).  The cluster barrier keeps either CTA's shared
    // memory and barriers alive until its peer has stopped signalling them.
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc<2>(tmem_base, kTmemCols);
    }
}

}  // namespace cb200
