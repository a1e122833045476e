// NVFP4 matmul for few rows of A per weight matrix: a serving step, dense or grouped (a few rows per expert).
//
// The problem lies transposed on the tensor core: 128 weight rows on the M axis / TMEM lanes, the tile's rows of A
// (padded to 16, at most 128) on the N axis, so that every weight byte is read once and nothing of the 128 lanes is
// wasted.  A persistent CTA walks (row tile, 128-column block) items; HBM-bound on the weights and their scales
// (9/16 byte per weight).  With few items the K range of an item is split over the CTAs of a cluster: their fp32
// partial sums go to the first CTA's shared memory and are added in rank order, the same bits on every run.
// 256 rows of 64 experts, n 4096, k 7168: 154 - 163 us (weights 1.06 GB: the HBM copy rate); 16 x 14336 x 4096: 9.5 us; 16 x
// 4096 x 14336, four CTAs per tile: 10.8.  Weights arrive as fast as HBM gives them; a call of its own costs ~4 us, a row of A
// 45 ns.
//   warp 0  producer: weights and rows of A (tensor maps), both scale blocks (bulk copies)
//   warp 1  MMA issuer        warps 2-5  scale copiers, one per word of a stage: smem -> TMEM
//   warps 6-9  epilogue, under the next item's MMAs (two accumulators)
#pragma once

#include "nvfp4_gemm.cuh"

namespace cb200 {

constexpr int kNvFewThreads = 320;
constexpr uint32_t kNvFewCopiers = 4;
constexpr int kNvFewEpiThreads = 128;
constexpr int kNvFewMaxStages = 8;
constexpr uint32_t kNvFewWBytes = 128 * kBlockKBytes;              // 16 KB of weights per stage
constexpr uint32_t kNvFewFixedBytes = kNvFewWBytes + 2 * 2048;     // plus both scale blocks
constexpr uint32_t kNvFewSmemBudget = 226u * 1024u;

struct NvFewParams {
    NvParams g;
    uint32_t mt;       // rows of A a stage has room for: 16, 32, 64 or 128, at least min(m, 128)
    uint32_t stages;
    uint32_t splits;   // CTAs of a cluster along K (1, 2, 4, 8); > 1 only when every cluster has one item at most
};

__host__ __device__ inline uint32_t nv_few_stage_bytes(uint32_t mt)
{
    return kNvFewFixedBytes + mt * kBlockKBytes;
}
// partial sums [splits - 1][mt][128] fp32 behind the ring
__host__ __device__ inline uint32_t nv_few_partial_bytes(uint32_t mt, uint32_t splits)
{
    return (splits - 1) * mt * 128u * 4u;
}
__host__ __device__ inline uint32_t nv_few_smem_bytes(uint32_t mt, uint32_t stages, uint32_t splits)
{
    return 1024 + stages * nv_few_stage_bytes(mt) + nv_few_partial_bytes(mt, splits) + (3 * kNvFewMaxStages + 5) * 8 + 16;
}

// tmap_w: {row bytes, n, groups}, boxes of 128 rows; tmap_x: {row bytes, m}, boxes of 16 rows.
__global__ void __launch_bounds__(kNvFewThreads, 1)
nvfp4_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                 const NvFewParams fp)
{
    const NvParams& p = fp.g;
    constexpr uint32_t kAccCols = 128;                // columns between the two accumulators
    constexpr uint32_t kSfBase = 2 * kAccCols;
    constexpr uint32_t kSfSlot = 32;                  // weights 16 columns, rows of A 16
    constexpr uint32_t kTmemCols = 512;
    static_assert(kSfBase + kNvFewMaxStages * kSfSlot <= kTmemCols, "TMEM budget");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t* smem = smem_raw + pad;
    const uint32_t ring = raw_addr + pad;
    const uint32_t stage_bytes = nv_few_stage_bytes(fp.mt);
    float* s_partials = reinterpret_cast<float*>(smem + fp.stages * stage_bytes);
    uint64_t* s_bars = reinterpret_cast<uint64_t*>(smem + fp.stages * stage_bytes + nv_few_partial_bytes(fp.mt, fp.splits));
    const uint32_t bar_full = smem_u32(s_bars);
    const uint32_t bar_empty = bar_full + kNvFewMaxStages * 8;
    const uint32_t bar_sf_full = bar_empty + kNvFewMaxStages * 8;
    const uint32_t bar_tmem_full = bar_sf_full + kNvFewMaxStages * 8;
    const uint32_t bar_tmem_empty = bar_tmem_full + 2 * 8;
    const uint32_t bar_partials = bar_tmem_empty + 2 * 8;  // first CTA: the other CTAs' sums have landed
    uint32_t* s_tmem_ptr = reinterpret_cast<uint32_t*>(s_bars + 3 * kNvFewMaxStages + 5);
    volatile uint32_t* s_abort = s_tmem_ptr + 1;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t split = fp.splits > 1 ? cluster_ctarank() : 0u;
    const uint32_t first_item = blockIdx.x / fp.splits;
    const uint32_t item_step = gridDim.x / fp.splits;
    const bool grouped = p.table != nullptr;

    if (threadIdx.x == 0) {
        *s_abort = 0;
        for (uint32_t s = 0; s < fp.stages; ++s) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
            mbar_init(bar_sf_full + s * 8, kNvFewCopiers);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tmem_full + a * 8, 1);
            mbar_init(bar_tmem_empty + a * 8, 4);
        }
        mbar_init(bar_partials, fp.splits > 1 ? (fp.splits - 1) * kNvFewEpiThreads : 1);
        fence_mbar_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(s_tmem_ptr), kTmemCols);
        tmem_relinquish<1>();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *s_tmem_ptr;
    if (fp.splits > 1) {
        cluster_sync();  // the first CTA's barrier exists before any other CTA can arrive on it
    }
    grid_launch_dependents();
    grid_dependency_wait();

    const uint32_t m_tiles = grouped ? *p.num_row_tiles : (p.m + 127u) / 128u;
    const uint32_t n_tiles = p.sfb_blocks;
    const uint32_t items = m_tiles * n_tiles;
    // this CTA's stages of K
    const uint32_t kb_per = (p.num_k_blocks + fp.splits - 1) / fp.splits;
    const uint32_t kb_begin = split * kb_per < p.num_k_blocks ? split * kb_per : p.num_k_blocks;
    const uint32_t kb_end = kb_begin + kb_per < p.num_k_blocks ? kb_begin + kb_per : p.num_k_blocks;
    // item -> row tile and column block, the column block fastest: the CTAs at work share a group's rows
    struct Item {
        uint32_t nt, mt;
        int32_t row0, rows, group;
    };
    auto get = [&](uint32_t idx) {
        Item it;
        it.mt = idx / n_tiles;
        it.nt = idx - it.mt * n_tiles;
        if (grouped) {
            const int4 e = __ldg(p.table + it.mt);
            it.row0 = e.x;
            it.rows = e.y - e.x < 128 ? e.y - e.x : 128;  // (never more than fp.mt: a tile's rows are at most m)
            it.group = e.z;
        } else {
            it.row0 = static_cast<int32_t>(it.mt * 128);
            it.rows = p.m - it.mt * 128 < 128 ? static_cast<int32_t>(p.m - it.mt * 128) : 128;
            it.group = 0;
        }
        return it;
    };
    // scale words of stage kb: all four but for the last
    auto words_of = [&](uint32_t kb) { return p.words - kb * 4 < 4 ? p.words - kb * 4 : 4u; };

    if (warp == 0) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = first_item; ok && idx < items; idx += item_step) {
                const Item it = get(idx);
                const uint32_t boxes = (static_cast<uint32_t>(it.rows) + 15u) / 16u;
                const uint8_t* sfw = p.sfb + (static_cast<uint64_t>(it.group) * p.sfb_blocks + it.nt) * p.words * 512;
                const uint8_t* sfx = p.sfa + static_cast<uint64_t>(it.mt) * p.words * 512;
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    ok = mbar_wait(bar_empty + stage * 8, phase ^ 1, s_abort, p.status, kDevTimeoutProducer);
                    if (!ok) {
                        break;
                    }
                    const uint32_t full = bar_full + stage * 8;
                    const uint32_t sw = ring + stage * stage_bytes;
                    const uint32_t ssf = sw + kNvFewWBytes;
                    const uint32_t sx = sw + kNvFewFixedBytes;
                    const int32_t k0 = static_cast<int32_t>(kb) * kBlockKBytes;
                    const uint32_t sf_bytes = words_of(kb) * 512;
                    mbar_expect_tx(full, kNvFewWBytes + boxes * 16 * kBlockKBytes + 2 * sf_bytes);
                    tma_load_3d(sw, &tmap_w, full, k0, static_cast<int32_t>(it.nt) * 128, it.group);
                    bulk_load(ssf, sfw + static_cast<uint64_t>(kb) * 2048, sf_bytes, full);
                    for (uint32_t b = 0; b < boxes; ++b) {
                        tma_load_2d(sx + b * 16 * kBlockKBytes, &tmap_x, full, k0, it.row0 + static_cast<int32_t>(b) * 16);
                    }
                    bulk_load(ssf + 2048, sfx + static_cast<uint64_t>(kb) * 2048, sf_bytes, full);
                    if (++stage == fp.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t idx = first_item; ok && idx < items; idx += item_step) {
                const Item it = get(idx);
                const uint32_t idesc = make_idesc_nv(128, (static_cast<uint32_t>(it.rows) + 15u) & ~15u);
                ok = mbar_wait(bar_tmem_empty + acc * 8, acc_phase ^ 1, s_abort, p.status, kDevTimeoutMmaTmem);
                if (!ok) {
                    break;
                }
                tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + acc * kAccCols;
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    ok = mbar_wait(bar_sf_full + stage * 8, phase, s_abort, p.status, kDevTimeoutMma);
                    if (!ok) {
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t sw = ring + stage * stage_bytes;
                    const uint32_t sx = sw + kNvFewFixedBytes;
                    const uint32_t t_sfw = tmem_base + kSfBase + stage * kSfSlot;
                    const uint32_t words = words_of(kb);
                    for (uint32_t j = 0; j < words; ++j) {
                        umma_nv<1>(tmem_d, make_smem_desc_sw128(sw + j * 32, 16, 1024),
                                   make_smem_desc_sw128(sx + j * 32, 16, 1024), idesc,
                                   kb != kb_begin || j != 0 ? 1u : 0u, t_sfw + j * 4, t_sfw + 16 + j * 4);
                    }
                    umma_commit<1>(bar_empty + stage * 8);
                    if (++stage == fp.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) {
                    break;
                }
                umma_commit<1>(bar_tmem_full + acc * 8);
                acc ^= 1;
                acc_phase ^= acc == 0 ? 1u : 0u;
            }
        }
        __syncwarp();
    } else if (warp < 2 + kNvFewCopiers) {
        // Copier w moves word w of the weights' scales to columns [4w, 4w + 4) of the stage's slot and that of A's to 16
        // columns behind.  (A stage's last words may be missing: then there is nothing to move, the arrival stays.)
        if (elect_one()) {
            const uint32_t w = warp - 2;
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t idx = first_item; ok && idx < items; idx += item_step) {
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    ok = mbar_wait(bar_full + stage * 8, phase, s_abort, p.status, kDevTimeoutConvert);
                    if (!ok) {
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t ssf = ring + stage * stage_bytes + kNvFewWBytes + w * 512;
                    const uint32_t slot = tmem_base + kSfBase + stage * kSfSlot + w * 4;
                    if (w < words_of(kb)) {
                        tmem_cp_32x128b_warpx4(slot, make_smem_desc_noswizzle(ssf, 16, 128));
                        tmem_cp_32x128b_warpx4(slot + 16, make_smem_desc_noswizzle(ssf + 2048, 16, 128));
                    }
                    umma_commit<1>(bar_sf_full + stage * 8);
                    if (++stage == fp.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        const uint32_t quad = warp & 3;
        const uint32_t lane_row = quad * 32 + lane;  // weight row inside the block = TMEM lane
        uint32_t acc = 0, acc_phase = 0;
        bool ok = true;
        for (uint32_t idx = first_item; idx < items; idx += item_step) {
            const Item it = get(idx);
            const uint32_t rows = static_cast<uint32_t>(it.rows);
            const uint32_t chunks = (rows + 15u) / 16u;
            const float alpha = p.alpha != nullptr ? __ldg(p.alpha + it.group) : 1.0f;
            const bool have = kb_begin < kb_end;  // a CTA without stages of K contributes zeros
            ok = mbar_wait(bar_tmem_full + acc * 8, acc_phase, s_abort, p.status, kDevTimeoutEpilogue);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok && fp.splits == 1) {
                break;
            }
            tcgen05_fence_after();
            const uint32_t taddr = tmem_base + acc * kAccCols + ((quad * 32u) << 16);
            const uint32_t col = it.nt * 128 + lane_row;
            if (fp.splits > 1 && split != 0) {
                // [token][lane] in the first CTA: 32 lanes write 128 contiguous bytes
                const uint32_t local = smem_u32(s_partials) + ((split - 1) * fp.mt * 128 + lane_row) * 4;
                uint32_t remote;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(0u));
                for (uint32_t c = 0; c < chunks; ++c) {
                    uint32_t r[16];
                    if (ok && have) {
                        tmem_ld_32x32b_x16(taddr + c * 16, r);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            r[i] = 0;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote + (c * 16 + i) * 512), "r"(r[i])
                                     : "memory");
                    }
                }
                mbar_arrive_cluster(bar_partials, 0);  // release: this thread's stores are visible to the waiter
            } else {
                bool sums = true;
                if (fp.splits > 1) {
                    // (a CTA that timed out still arrives, with zeros)
                    sums = mbar_wait_cluster(bar_partials, 0, s_abort, p.status, kDevTimeoutPeerCta);
                    sums = __all_sync(0xffffffffu, sums);
                }
                for (uint32_t c = 0; c < chunks && ok && sums; ++c) {
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(taddr + c * 16, r);
                    tmem_ld_wait();
                    for (uint32_t s = 1; s < fp.splits; ++s) {  // (sixteen reads of a peer's sums in flight)
                        const float* sums_of = s_partials + ((s - 1) * fp.mt + c * 16) * 128 + lane_row;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            r[i] = __float_as_uint(__uint_as_float(r[i]) + sums_of[i * 128]);
                        }
                    }
                    nv_store_columns<16>(p, r, static_cast<uint32_t>(it.row0) + c * 16, rows - c * 16, col, alpha);
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar_tmem_empty + acc * 8);
            }
            acc ^= 1;
            acc_phase ^= acc == 0 ? 1u : 0u;
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (fp.splits > 1) {
        cluster_sync();  // nobody's shared memory goes away while a peer may still write to it
    }
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc<1>(tmem_base, kTmemCols);
    }
}

}  // namespace cb200
