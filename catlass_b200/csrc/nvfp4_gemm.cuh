// NVFP4 block-scaled matmul for sm_100a: E2M1 operands, one E4M3 scale per 16 elements along K, fp32 accumulation:
//     D[m,n] = round( alpha * sum_k (a[m,k] * sa[m,k/16]) * (b[n,k] * sb[n,k/16]) )
// The products and the scaling happen in the tensor core (tcgen05.mma.kind::mxf4nvf4.block_scale.block16); the scales
// sit in TMEM next to the accumulator, in the order of the tiled scale layout: per 128 rows x 4 blocks (one MMA of 64
// elements along K) a 512-byte block [row % 32][row / 32][4 bytes].
//
//   nvfp4_pack_scales_kernel  scales by rows -> tiled; for a grouped problem also the row-tile table: tiles start at a
//                             group's first row, so their scale blocks do too.
//   nvfp4_pair_kernel         CTA pairs (cta_group::2): 256 weight rows on the M axis, up to 256 rows of A on the N axis.
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
    uint32_t tile_x;               // pair kernel, dense: rows of A per tile, 128, 192 or 256
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

// blockIdx.y walks the batch.  A warp works on one 128-row block and four words (256 elements) of it: a lane reads 16 bytes
// of each of its four rows lane, lane + 32, lane + 64 and lane + 96, whose words lie next to each other in the output, so
// that every store instruction writes 512 contiguous bytes.  (8192 rows of 7168, 16 groups: 6.3 us; with a lane per
// 16 bytes of one row and four-byte stores 11.6.)
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
    const bool vec = (p.blocks & 15u) == 0 && (reinterpret_cast<uintptr_t>(in) & 15u) == 0;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * (kNvPackThreads / 32);
    const uint32_t warp_id = blockIdx.x * (kNvPackThreads / 32) + (threadIdx.x >> 5);
    const uint32_t step_blocks = warps / quads, step_quads = warps % quads;
    uint32_t block = warp_id / quads, quad = warp_id % quads;
    while (block < row_blocks) {
        uint32_t row0 = block * 128u, end = p.rows;
        if (grouped) {
            const uint32_t tile = block / per_tile;
            uint32_t lo = 0, hi = p.groups - 1;  // the group whose tiles hold this one: last g with s_tile[g] <= tile
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) / 2;
                if (s_tile[mid] <= tile) {
                    lo = mid;
                } else {
                    hi = mid - 1;
                }
            }
            row0 = (lo == 0 ? 0u : s_end[lo - 1]) + (block - s_tile[lo] * per_tile) * 128u;
            end = s_end[lo];
        }
        uint32_t w[4][4];  // [word][row group]
#pragma unroll
        for (uint32_t g = 0; g < 4; ++g) {
            const uint32_t row = row0 + g * 32 + lane;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (row < end) {  // (rows that are never stored may have any scale)
                const uint8_t* src = in + static_cast<uint64_t>(row) * p.blocks + quad * 16;
                if (vec) {
                    v = *reinterpret_cast<const uint4*>(src);
                } else {
                    uint32_t x[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (uint32_t b = 0; b < 16; ++b) {
                        if (quad * 16 + b < p.blocks) {
                            x[b / 4] |= static_cast<uint32_t>(src[b]) << (8 * (b % 4));
                        }
                    }
                    v = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            w[0][g] = v.x;
            w[1][g] = v.y;
            w[2][g] = v.z;
            w[3][g] = v.w;
        }
        uint8_t* dst = out + (static_cast<uint64_t>(block) * p.words + quad * 4) * 512 + lane * 16;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (quad * 4 + j < p.words) {
                *reinterpret_cast<uint4*>(dst + j * 512) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
            }
        }
        block += step_blocks;
        quad += step_quads;
        if (quad >= quads) {
            quad -= quads;
            ++block;
        }
    }
}

// ---------------------------------------------------------------- CTA pairs
//
// The problem lies transposed on the tensor core: a tile is 256 WEIGHT rows (the M axis; CTA r of the pair owns rows
// [128 r, 128 r + 128) and their accumulator lanes) and up to 256 rows of A (the N axis, in steps of 32).  A group's last
// rows then cost what they are: an MMA of N columns takes N/256 of a full one and reads N/256 of A, where rows of A on the
// M axis would be padded to 256.  And a warp that stores a row of D writes 32 neighbouring columns.
//
// The single threads of the pipeline are picked by elect.sync: the compiler then knows that one thread runs their loops and
// keeps what tcgen05 and TMA instructions take in uniform registers.  With lane == 0 instead, issuing them set the pace of
// small tiles (128 x 4096 x 4096: 10.7 us against 8.7).
//
// Per stage (256 along K) a CTA takes in its weights 16 KB, half of the tile's rows of A (up to 16 KB) and the scale blocks
// of its weight rows (2 KB) and of all rows of A (2 x 2 KB), and the tensor core reads 16 + 16 + 6 KB of it: 76 KB through
// a shared memory of 128 bytes a clock are 608 clocks, against 512 of MMAs.  Measured with a full tile: ~720 a
// stage, and ~1.5 us between tiles for handing the one accumulator over (256 columns and the scale slots fill TMEM).
// 8192^3: 4.9 PFLOP/s in a burst, 4.2 under the power cap; grouped, 32768 rows of 64 experts, n 4096, k 7168: 494 us.
constexpr int kNvPairStages = 5;
constexpr int kNvPairCopiers = 4;
constexpr int kNvPairEpiWarps = 16;
constexpr uint32_t kNvTileW = 256;  // weight rows per tile
constexpr uint32_t kNvTileX = 256;  // rows of A per tile
// warps: 0 operand producer, 1 MMA issuer, 2 scale producer, 3-6 scale copiers, 7-22 epilogue
constexpr int kNvPairThreads = (3 + kNvPairCopiers + kNvPairEpiWarps) * 32;

struct NvPairSmem {
    static constexpr int kWBytes = 128 * kBlockKBytes;   // this CTA's 128 weight rows
    static constexpr int kXBytes = 128 * kBlockKBytes;   // its half of the rows of A
    static constexpr int kSfBytes = 3 * 2048;            // four words each of the weights and of A's two blocks
    static constexpr int kStageBytes = kWBytes + kXBytes + kSfBytes;
    static constexpr int kRingBytes = kNvPairStages * kStageBytes;
    // 32 rows of D x 64 bytes (fp32: 16 x 128) per epilogue warp, on their way out by TMA stores
    static constexpr int kSlabBytes = 2048;
    static constexpr int kBarrierOffset = kRingBytes + kNvPairEpiWarps * kSlabBytes;
    static constexpr int kBarriers = 3 * kNvPairStages + 2;
    static constexpr int kTotalBytes = 1024 + kBarrierOffset + kBarriers * 8 + 16;
};
static_assert(NvPairSmem::kTotalBytes <= 227 * 1024, "shared memory budget");
static_assert(NvPairSmem::kStageBytes % 1024 == 0, "swizzled tiles start on 1 KB boundaries");

// One warp's share of an accumulator whose lanes are columns of D: 32 columns (lane = column) of rows row0 .. row0 + rows,
// r[i] being row i.  Every store instruction writes 32 neighbouring columns.
template <int kCount>
__device__ __forceinline__ void nv_store_columns(const NvParams& p, const uint32_t (&r)[kCount], uint32_t row0,
                                                 uint32_t rows, uint32_t col, float alpha)
{
    const uint64_t at = static_cast<uint64_t>(row0) * p.n + col;
    if (col >= p.n) {
        return;
    }
    if (p.d_type == 0) {
        float* d = static_cast<float*>(p.d) + at;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if (static_cast<uint32_t>(i) < rows) {
                *d = __uint_as_float(r[i]) * alpha;
            }
            d += p.n;
        }
    } else {
        uint16_t* d = static_cast<uint16_t*>(p.d) + at;
        const bool f16 = p.d_type == 2;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if (static_cast<uint32_t>(i) < rows) {
                *d = pack_out1(__uint_as_float(r[i]) * alpha, f16);
            }
            d += p.n;
        }
    }
}

// The same 32 columns of kCount whole rows through a slab and one TMA store (every thread writes its column, two bytes at a
// time: 32 lanes, 64 neighbouring bytes).  The slab's previous store is waited for.  All lanes take part.
template <int kCount>
__device__ __forceinline__ void nv_tma_store_columns(const NvParams& p, const CUtensorMap* tmap_d, const uint32_t* r,
                                                     uint8_t* slab, uint32_t row0, uint32_t col0, float alpha,
                                                     uint32_t lane)
{
    if (lane == 0) {
        tma_store_wait_read<0>();
    }
    __syncwarp();
    constexpr uint32_t kElem = 64 / kCount;  // 32 rows of two-byte, 16 of four-byte elements
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
        const float v = __uint_as_float(r[i]) * alpha;
        if constexpr (kElem == 4) {
            reinterpret_cast<float*>(slab)[i * 32 + lane] = v;
        } else {
            reinterpret_cast<uint16_t*>(slab)[i * 32 + lane] = pack_out1(v, p.d_type == 2);
        }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_2d(tmap_d, smem_u32(slab), static_cast<int32_t>(col0 * kElem), static_cast<int32_t>(row0));
        tma_store_commit();
    }
}

// Rows of A as a tensor {row bytes, m}, boxes of 16, 32, 64 and 128 rows.  A tile's share of a CTA is one box, the smallest
// that holds it: a TMA instruction costs its thread ~65 ns, and eight boxes of 16 rows a stage set the kernel's pace (0.59
// us a stage instead of 0.38).
struct NvRowMaps {
    CUtensorMap box[4];
};

// tmap_w: {row bytes, n, groups}, boxes of 128 rows; tmap_sfw / tmap_sfx: the tiled scales as {256, 2 * words, row blocks},
// boxes of {256, 8, 1} = four words; words past the last read as zero; tmap_d: D as bytes, boxes of 64 bytes x 32 rows, fp32
// 128 x 16 (p.tma_store).
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNvPairThreads, 1)
nvfp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ NvRowMaps tmap_x,
                  const __grid_constant__ CUtensorMap tmap_sfw, const __grid_constant__ CUtensorMap tmap_sfx,
                  const __grid_constant__ CUtensorMap tmap_d, const NvParams p)
{
    using S = NvPairSmem;
    constexpr int kStages = kNvPairStages;
    constexpr uint32_t kAccCols = kNvTileX;
    constexpr uint32_t kSfSlot = 48;  // one scale slot: weights 16 columns, rows of A 32
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
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x.box[3]);
        prefetch_tmap(&tmap_sfw);
        prefetch_tmap(&tmap_sfx);
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

    const uint32_t m_tiles = grouped ? *p.num_row_tiles : (p.m + p.tile_x - 1) / p.tile_x;
    const uint32_t n_tiles = (p.n + kNvTileW - 1) / kNvTileW;
    const uint32_t total_tiles = m_tiles * n_tiles;
    const uint32_t num_kb = p.num_k_blocks;
    struct Tile {
        uint32_t mt, nt;    // row tile of A, weight tile
        uint32_t row0;      // first row of A
        uint32_t rows;      // rows of A to store, 1 .. 256
        uint32_t cols;      // ... padded to a multiple of 32: columns of the MMA
        uint32_t block_x;   // the scale block of the first row, and the row's place in it (0, or 64 with 192-row tiles)
        uint32_t shift;
        uint32_t group;
    };
    auto get = [&](uint32_t idx) {
        Tile t;
        mx_tile_coords(idx, m_tiles, n_tiles, p.band_rows, t.mt, t.nt);
        uint32_t end;
        if (grouped) {
            const int4 e = __ldg(p.table + t.mt);
            t.row0 = static_cast<uint32_t>(e.x);
            end = static_cast<uint32_t>(e.y);
            t.group = static_cast<uint32_t>(e.z);
            t.block_x = 2 * t.mt;
            t.shift = 0;
        } else {
            t.row0 = t.mt * p.tile_x;
            end = p.m;
            t.group = 0;
            t.block_x = t.row0 / 128;
            t.shift = t.row0 % 128;
        }
        const uint32_t most = grouped ? kNvTileX : p.tile_x;
        t.rows = end - t.row0 < most ? end - t.row0 : most;
        t.cols = (t.rows + 31u) & ~31u;
        return t;
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- operand producer (both CTAs)
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                const Tile t = get(idx);
                const uint32_t half = t.cols / 2;                          // this CTA's rows of A: 16 .. 128
                const uint32_t which = half <= 16 ? 0u : (half <= 32 ? 1u : (half <= 64 ? 2u : 3u));
                const uint32_t x_bytes = (16u << which) * kBlockKBytes;
                const uint32_t x0 = t.row0 + cta_rank * half;
                const uint32_t w0 = t.nt * kNvTileW + cta_rank * 128;
                const uint32_t sf_x = t.shift + t.cols > 128 ? 4096u : 2048u;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_empty + stage * 8, phase ^ 1, s_abort, p.status, kDevTimeoutProducer);
                    if (!ok) {
                        break;
                    }
                    const uint32_t sw = ring + stage * S::kStageBytes;
                    const uint32_t sx = sw + S::kWBytes;
                    const int32_t k0 = static_cast<int32_t>(kb) * kBlockKBytes;
                    if (cta_rank == 0) {  // both CTAs' tiles and scale blocks
                        mbar_expect_tx(bar_full + stage * 8, 2 * (S::kWBytes + x_bytes + 2048 + sf_x));
                    }
                    const uint32_t full = map_to_cta(bar_full + stage * 8, 0);  // the leader's barrier
                    tma_load_3d_pair(sw, &tmap_w, full, k0, static_cast<int32_t>(w0), static_cast<int32_t>(t.group));
                    tma_load_2d_pair(sx, &tmap_x.box[which], full, k0, static_cast<int32_t>(x0));
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
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                const Tile t = get(idx);
                const int32_t block_w = static_cast<int32_t>(t.group * p.sfb_blocks + 2 * t.nt + cta_rank);
                const int32_t block_x = static_cast<int32_t>(t.block_x);
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_empty + stage * 8, phase ^ 1, s_abort, p.status, kDevTimeoutProducer);
                    if (!ok) {
                        break;
                    }
                    const uint32_t ssf = ring + stage * S::kStageBytes + S::kWBytes + S::kXBytes;
                    const uint32_t full = map_to_cta(bar_full + stage * 8, 0);
                    const int32_t w2 = static_cast<int32_t>(kb * 8);  // rows of 256 bytes, two per word
                    // (a block past the last, of A or of the weights, reads zeros or another group's scales: its rows
                    // and columns are not stored)
                    tma_load_3d_pair(ssf, &tmap_sfw, full, 0, w2, block_w);
                    tma_load_3d_pair(ssf + 2048, &tmap_sfx, full, 0, w2, block_x);
                    if (t.shift + t.cols > 128) {
                        tma_load_3d_pair(ssf + 4096, &tmap_sfx, full, 0, w2, block_x + 1);
                    }
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
        if (cta_rank == 0 && elect_one()) {
            uint32_t stage = 0, phase = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                const Tile t = get(idx);
                const uint32_t idesc = make_idesc_nv(kNvTileW, t.cols);
                const uint32_t skip = t.shift / 32;  // scale columns of rows in front of the tile
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
                    const uint32_t sw = ring + stage * S::kStageBytes;
                    const uint32_t sx = sw + S::kWBytes;
                    const uint32_t t_sfw = tmem_base + kAccCols + stage * kSfSlot;
                    const uint32_t t_sfx = t_sfw + 16 + skip;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint64_t dw = make_smem_desc_sw128(sw + j * 32, 16, 1024);
                        const uint64_t dx = make_smem_desc_sw128(sx + j * 32, 16, 1024);
                        umma_nv<2>(tmem_base, dw, dx, idesc, (kb | j) != 0 ? 1u : 0u, t_sfw + j * 4, t_sfx + j * 8);
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
        // Copier w moves word w of the scale blocks.  Slot `stage` is free when the stage's "full" barrier fires: the
        // MMAs that read it completed before the producers were allowed to refill the stage.
        const uint32_t w = warp - 3;
        if (cta_rank == 0 && elect_one()) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
                const Tile t = get(idx);
                const bool two = t.shift + t.cols > 128;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = mbar_wait(bar_full + stage * 8, phase, s_abort, p.status, kDevTimeoutConvert);
                    if (!ok) {
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t ssf = ring + stage * S::kStageBytes + S::kWBytes + S::kXBytes + w * 512;
                    const uint32_t t_sfw = tmem_base + kAccCols + stage * kSfSlot;
                    const uint32_t t_sfx = t_sfw + 16 + w * 8;
                    tmem_cp_32x128b_warpx4_pair(t_sfw + w * 4, make_smem_desc_noswizzle(ssf, 16, 128));
                    tmem_cp_32x128b_warpx4_pair(t_sfx, make_smem_desc_noswizzle(ssf + 2048, 16, 128));
                    if (two) {
                        tmem_cp_32x128b_warpx4_pair(t_sfx + 4, make_smem_desc_noswizzle(ssf + 4096, 16, 128));
                    }
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
        const uint32_t part = (warp - 3 - kNvPairCopiers) >> 2;   // which 64 rows of A
        uint8_t* slab = smem + S::kRingBytes + (warp - 3 - kNvPairCopiers) * S::kSlabBytes;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (uint32_t idx = pair; ok && idx < total_tiles; idx += num_pairs) {
            const Tile t = get(idx);
            const float alpha = p.alpha != nullptr ? __ldg(p.alpha + t.group) : 1.0f;
            ok = mbar_wait(bar_tmem_full, acc_phase, s_abort, p.status, kDevTimeoutEpilogue);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                break;
            }
            tcgen05_fence_after();
            const uint32_t first = part * 64;
            const uint32_t rows = t.rows > first ? t.rows - first : 0u;  // of this warp's 64
            const uint32_t taddr = tmem_base + first + ((quad * 32u) << 16);
            uint32_t r[2][32];
            if (rows != 0) {
                tmem_ld_32x32b_x32(taddr, r[0]);
                tmem_ld_32x32b_x32(taddr + 32, r[1]);
                tmem_ld_wait();
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_cluster(bar_tmem_empty, 0);  // this warp's share is in registers
            }
            acc_phase ^= 1;
            const uint32_t col0 = t.nt * kNvTileW + cta_rank * 128 + quad * 32;
            if (col0 >= p.n) {
                continue;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t row0 = t.row0 + first + h * 32;
                if (p.tma_store && rows >= h * 32 + 32u) {
                    if (p.d_type == 0) {
                        nv_tma_store_columns<16>(p, &tmap_d, r[h], slab, row0, col0, alpha, lane);
                        nv_tma_store_columns<16>(p, &tmap_d, r[h] + 16, slab, row0 + 16, col0, alpha, lane);
                    } else {
                        nv_tma_store_columns<32>(p, &tmap_d, r[h], slab, row0, col0, alpha, lane);
                    }
                } else if (rows > h * 32u) {
                    nv_store_columns<32>(p, r[h], row0, rows - h * 32, col0 + lane, alpha);
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
