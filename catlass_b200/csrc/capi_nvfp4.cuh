// C-ABI entry points of the NVFP4 matmuls, dense and grouped.  (Part of capi.cu's translation unit; uses its helpers.)
#pragma once

namespace {

struct NvProblem {
    uint32_t m, n, k;
    uint32_t group_count;  // 0 = dense
    uint32_t group_list_type, group_list_kind;
    uint32_t scale_a_layout, scale_b_layout, d_type;
    const void* a;
    const void* b;
    const void* group_list;
    const void* scale_a;
    const void* scale_b;
    const float* alpha;
    void* d;
    void* workspace;
    uint64_t workspace_bytes;
    uint32_t block_num, flags;
};

struct NvPlan {
    bool few;                // nvfp4_few_kernel, else nvfp4_pair_kernel
    bool pack_a, pack_b;
    uint32_t tile_rows;      // rows per row tile: 128 (few) or 256
    uint32_t max_tiles;      // row tiles at most
    uint32_t sfa_blocks;     // 128-row scale blocks of A: a row tile's own, or those of all rows of a dense problem
    uint32_t words, sfb_blocks, matrices;
    uint64_t table_bytes, sfa_bytes, sfb_bytes;
    uint64_t total() const { return table_bytes + sfa_bytes + sfb_bytes; }
};

uint32_t nv_few_rows(const NvProblem& q)  // rows of A a stage has room for
{
    uint32_t mt = 16;
    while (mt < q.m && mt < 128u) {
        mt *= 2;
    }
    return mt;
}

// CTAs of a cluster along K: as many as leave every cluster at most one item and every CTA two stages, with partial sums
// of 64 KB at most.
uint32_t nv_few_splits(uint32_t mt, uint64_t items, uint32_t stages, uint32_t ctas)
{
    uint32_t splits = 1;
    while (splits < 8u && items * splits * 2u <= ctas && stages >= 4u * splits &&
           nv_few_partial_bytes(mt, splits * 2u) <= 64u * 1024u) {
        splits *= 2;
    }
    return splits;
}

// Which kernel.  nvfp4_few_kernel reads weights faster (128-row tiles, a deeper ring) and can split K, but every row of A
// costs it more.  Measured, few / pair, us.  Grouped, rows per group on average (64 groups, n 4096, k 7168): 4: 163 / 182, 32:
// 174 / 191, 64: 185 / 197, 128: 241 / 223; (128 groups, n 1024, k 2048): 16: 35 / 45, 64: 42 / 48, 256: 88 / 71.
// Dense, m x n x k: 16 x 14336 x 4096: 9.5 / 12.1, 128 x: 13.2 / 12.8; 16 x 4096 x 4096: 6.2 / 8.2, 128 x: 11.6 / 8.9; 16 x 4096 x
// 14336: 10.8 / 21.0, 128 x: 20.5 / 22.4.  The model below is fitted to those (ns): a call, the rows of A, and the stages of
// the longest CTA or the weights' way from memory.
bool nv_use_few(const NvProblem& q)
{
    const long v = dev_knob("CB200_NV_FEW", -1);
    if (v >= 0) {
        return v != 0;
    }
    if (q.group_count != 0) {
        return q.m / q.group_count <= 64u;
    }
    if (q.m > 128u) {
        return false;
    }
    constexpr uint64_t kSms = 148;
    const uint32_t stages = (q.k + kNvStageK - 1u) / kNvStageK;
    const uint64_t items = (q.n + 127u) / 128u, tiles = (q.n + kNvTileW - 1u) / kNvTileW;
    const uint64_t splits = nv_few_splits(nv_few_rows(q), items, stages, kSms);
    const uint64_t weights = static_cast<uint64_t>(q.n) * q.k * 9u / 16u;  // bytes
    const uint64_t few_stages = 330ull * ((stages + splits - 1) / splits) * ((items * splits + kSms - 1) / kSms);
    const uint64_t pair_stages = 290ull * stages * ((tiles + kSms / 2 - 1) / (kSms / 2));
    const uint64_t few_bytes = weights / 5500u, pair_bytes = weights / 4200u;
    const uint64_t few = 3800ull + 45ull * q.m + (few_stages > few_bytes ? few_stages : few_bytes);
    const uint64_t pair = 4000ull + 10ull * q.m + (pair_stages > pair_bytes ? pair_stages : pair_bytes);
    return few <= pair;
}

int plan_nv(const NvProblem& q, NvPlan* plan)
{
    *plan = NvPlan{};
    if (q.flags != 0 || !is_float_type(q.d_type) || q.scale_a_layout > CB200_NVFP4_SCALES_TILED ||
        q.scale_b_layout > CB200_NVFP4_SCALES_TILED) {
        return CB200_INVALID;
    }
    if (q.group_count != 0 &&
        (q.group_count > static_cast<uint32_t>(kMaxGroups) ||
         (q.group_list_type != CB200_GROUP_LIST_INT64 && q.group_list_type != CB200_GROUP_LIST_INT32) ||
         (q.group_list_kind != CB200_GROUP_LIST_SIZES && q.group_list_kind != CB200_GROUP_LIST_PREFIX_SUMS))) {
        return CB200_INVALID;
    }
    if (q.m == 0 || q.n == 0) {
        return CB200_SUCCESS;
    }
    if (q.a == nullptr || q.b == nullptr || q.scale_a == nullptr || q.scale_b == nullptr || q.d == nullptr || q.k == 0 ||
        q.k % 32u != 0 || q.m > 0x7fffff00u || q.n > 0x7fffff00u || q.k > 0x7fffff00u || !aligned16(q.a) ||
        !aligned16(q.b) || !aligned16(q.scale_a) || !aligned16(q.scale_b) || !aligned_to(q.alpha, 4)) {
        return CB200_INVALID;
    }
    if (q.group_count != 0 && (q.group_list == nullptr ||
                               !aligned_to(q.group_list, q.group_list_type == CB200_GROUP_LIST_INT64 ? 8 : 4))) {
        return CB200_INVALID;
    }
    const uint64_t elem = float_bytes(q.d_type);
    if (!aligned_to(q.d, elem) || (q.n % (16u / elem) == 0 && !aligned16(q.d))) {
        return CB200_INVALID;  // 16-byte vector stores
    }
    plan->few = nv_use_few(q);
    plan->tile_rows = plan->few ? 128u : 256u;
    plan->matrices = q.group_count == 0 ? 1u : q.group_count;
    plan->max_tiles = (q.m + plan->tile_rows - 1u) / plan->tile_rows + q.group_count;
    plan->words = (q.k + 63u) / 64u;
    plan->sfb_blocks = (q.n + 127u) / 128u;
    if (static_cast<uint64_t>(plan->sfb_blocks) * plan->matrices > 0x7fffffffu ||
        static_cast<uint64_t>(plan->max_tiles) * 2u * plan->sfb_blocks > 0x7fffffffu) {
        return CB200_INVALID;  // tile and block numbers are 32-bit
    }
    plan->pack_a = q.group_count != 0 || q.scale_a_layout == CB200_NVFP4_SCALES_ROWS;
    plan->pack_b = q.scale_b_layout == CB200_NVFP4_SCALES_ROWS;
    plan->table_bytes = q.group_count == 0 ? 0 : align256(static_cast<uint64_t>(plan->max_tiles) * 16u + 16u);
    plan->sfa_blocks = q.group_count != 0 ? plan->max_tiles * (plan->tile_rows / 128u) : (q.m + 127u) / 128u;
    plan->sfa_bytes = plan->pack_a ? static_cast<uint64_t>(plan->sfa_blocks) * plan->words * 512u : 0;
    plan->sfb_bytes = plan->pack_b ? static_cast<uint64_t>(plan->sfb_blocks) * plan->matrices * plan->words * 512u : 0;
    return CB200_SUCCESS;
}

// A tiled scale array as {256, 2 * words, row blocks}: boxes of four words of one block.
int encode_nv_scales(CUtensorMap* map, const void* base, uint32_t words, uint64_t row_blocks)
{
    const uint64_t dims[3] = {256, 2ull * words, row_blocks};
    const uint64_t strides[2] = {256, 512ull * words};
    const uint32_t box[3] = {256, 8, 1};
    return encode_tmap_u8(map, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

int encode_nv_weights(CUtensorMap* map, const NvProblem& q, const NvPlan& plan)
{
    const uint64_t row_bytes = q.k / 2u;
    const uint64_t dims[3] = {row_bytes, q.n, plan.matrices};
    const uint64_t strides[2] = {row_bytes, static_cast<uint64_t>(q.n) * row_bytes};
    const uint32_t box[3] = {kBlockKBytes, 128, 1};
    return encode_tmap_u8(map, q.b, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int encode_nv_rows(CUtensorMap* map, const NvProblem& q, uint32_t box_rows)
{
    const uint64_t row_bytes = q.k / 2u;
    const uint64_t dims[2] = {row_bytes, q.m};
    const uint64_t strides[1] = {row_bytes};
    const uint32_t box[2] = {kBlockKBytes, box_rows};
    return encode_tmap_u8(map, q.a, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// D as bytes, boxes of 32 columns: 32 rows of two-byte or 16 of four-byte elements.
int encode_nv_output(CUtensorMap* map, const NvProblem& q)
{
    const uint32_t elem = static_cast<uint32_t>(float_bytes(q.d_type));
    const uint64_t row_bytes = static_cast<uint64_t>(q.n) * elem;
    const uint64_t dims[2] = {row_bytes, q.m};
    const uint64_t strides[1] = {row_bytes};
    const uint32_t box[2] = {32u * elem, 64u / elem};
    return encode_tmap_u8(map, q.d, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Rows of A per tile of a dense problem: the height whose waves over the pairs cost least.  (The scale blocks hold 128 rows:
// 192-row tiles start at a block's beginning or middle.)
uint32_t nv_tile_rows(uint32_t m, uint32_t n_tiles, uint32_t pairs)
{
    const long v = dev_knob("CB200_NV_TILEX", 0);
    if (v != 0) {
        return static_cast<uint32_t>(v);
    }
    constexpr uint32_t kRows[3] = {256, 192, 128};
    constexpr uint64_t kCost[3] = {100, 80, 65};  // of a stage
    uint32_t best = 0;
    uint64_t best_cost = ~0ull;
    for (uint32_t i = 0; i < 3; ++i) {
        const uint64_t tiles = static_cast<uint64_t>((m + kRows[i] - 1u) / kRows[i]) * n_tiles;
        const uint64_t cost = (tiles + pairs - 1u) / pairs * kCost[i];
        if (cost < best_cost) {
            best = kRows[i];
            best_cost = cost;
        }
    }
    return best;
}

int launch_nv_pair(const NvProblem& q, const NvPlan& plan, NvParams p, const DeviceState& dev, cudaStream_t stream)
{
    CUtensorMap tmap_w, tmap_sfw, tmap_sfx;
    NvRowMaps tmap_x;
    int rc = encode_nv_weights(&tmap_w, q, plan);
    for (uint32_t i = 0; i < 4 && rc == CB200_SUCCESS; ++i) {
        rc = encode_nv_rows(&tmap_x.box[i], q, 16u << i);
    }
    rc = rc != CB200_SUCCESS
             ? rc
             : encode_nv_scales(&tmap_sfw, p.sfb, plan.words, static_cast<uint64_t>(plan.sfb_blocks) * plan.matrices);
    rc = rc != CB200_SUCCESS
             ? rc
             : encode_nv_scales(&tmap_sfx, p.sfa, plan.words, plan.sfa_blocks);
    // rows of D that do not start on 16-byte boundaries are stored by the threads
    p.tma_store = (q.n * float_bytes(q.d_type)) % 16u == 0 ? 1u : 0u;
    CUtensorMap tmap_d = tmap_w;
    if (rc == CB200_SUCCESS && p.tma_store != 0) {
        rc = encode_nv_output(&tmap_d, q);
    }
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    static PerDeviceOnce once;
    int devid = 0;
    rc = current_device(&devid);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    rc = once.run(devid, [&]() -> int {
        CB200_CUDA_TRY(cudaFuncSetAttribute(nvfp4_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            NvPairSmem::kTotalBytes));
        return CB200_SUCCESS;
    });
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    uint32_t pairs = static_cast<uint32_t>(dev.sm_count) / 2u;
    if (q.block_num != 0 && q.block_num / 2u < pairs) {
        pairs = q.block_num < 2u ? 1u : q.block_num / 2u;
    }
    const uint32_t n_tiles = (q.n + kNvTileW - 1u) / kNvTileW;
    p.tile_x = q.group_count != 0 ? kNvTileX : nv_tile_rows(q.m, n_tiles, pairs);
    const uint64_t tiles =
        static_cast<uint64_t>(q.group_count != 0 ? plan.max_tiles : (q.m + p.tile_x - 1u) / p.tile_x) * n_tiles;
    pairs = tiles < pairs ? static_cast<uint32_t>(tiles) : pairs;
    CB200_CUDA_TRY(launch_dependent(nvfp4_pair_kernel, 2 * pairs, kNvPairThreads, NvPairSmem::kTotalBytes, stream,
                                    tmap_w, tmap_x, tmap_sfw, tmap_sfx, tmap_d, p));
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return CB200_SUCCESS;
}

int launch_nv_few(const NvProblem& q, const NvPlan& plan, const NvParams& p, const DeviceState& dev, cudaStream_t stream)
{
    NvFewParams fp;
    fp.g = p;
    fp.mt = nv_few_rows(q);
    CUtensorMap tmap_w, tmap_x;
    int rc = encode_nv_weights(&tmap_w, q, plan);
    rc = rc != CB200_SUCCESS ? rc : encode_nv_rows(&tmap_x, q, 16);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    static PerDeviceOnce once;
    int devid = 0;
    rc = current_device(&devid);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    rc = once.run(devid, [&]() -> int {
        CB200_CUDA_TRY(cudaFuncSetAttribute(nvfp4_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            kNvFewSmemBudget));
        return CB200_SUCCESS;
    });
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    uint32_t ctas = static_cast<uint32_t>(dev.sm_count);
    if (q.block_num != 0 && q.block_num < ctas) {
        ctas = q.block_num;
    }
    const uint64_t items = static_cast<uint64_t>(plan.max_tiles) * plan.sfb_blocks;
    fp.splits = nv_few_splits(fp.mt, items, p.num_k_blocks, ctas);
    fp.stages = kNvFewMaxStages;
    while (nv_few_smem_bytes(fp.mt, fp.stages, fp.splits) > kNvFewSmemBudget) {
        --fp.stages;
    }
    const uint32_t grid = static_cast<uint32_t>(items * fp.splits < ctas ? items * fp.splits : ctas);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(kNvFewThreads, 1, 1);
    cfg.dynamicSmemBytes = nv_few_smem_bytes(fp.mt, fp.stages, fp.splits);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = fp.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, nvfp4_few_kernel, tmap_w, tmap_x, fp));
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return CB200_SUCCESS;
}

int run_nv(const NvProblem& q, void* stream_v)
{
    NvPlan plan;
    int rc = plan_nv(q, &plan);
    if (rc != CB200_SUCCESS || q.m == 0 || q.n == 0) {
        return rc;
    }
    if (plan.total() != 0 && (q.workspace == nullptr || q.workspace_bytes < plan.total() ||
                              !aligned_to(q.workspace, 256))) {
        return CB200_INVALID;
    }
    DeviceState* dev = nullptr;
    rc = device_state(&dev);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    uint8_t* ws = static_cast<uint8_t*>(q.workspace);
    int4* table = reinterpret_cast<int4*>(ws);
    uint32_t* num_tiles = reinterpret_cast<uint32_t*>(ws + static_cast<uint64_t>(plan.max_tiles) * 16u);
    uint8_t* sfa = ws + plan.table_bytes;
    uint8_t* sfb = sfa + plan.sfa_bytes;
    if (plan.pack_b) {
        NvPackParams b = {};
        b.in = static_cast<const uint8_t*>(q.scale_b);
        b.out = sfb;
        b.rows = q.n;
        b.blocks = q.k / 16u;
        b.words = plan.words;
        b.in_batch = static_cast<uint64_t>(q.n) * b.blocks;
        b.out_batch = static_cast<uint64_t>(plan.sfb_blocks) * plan.words * 512u;
        const uint32_t gx = plan.matrices > 8u ? static_cast<uint32_t>(dev->sm_count) / 4u : dev->sm_count * 4u;
        nvfp4_pack_scales_kernel<<<dim3(gx, plan.matrices, 1), kNvPackThreads, 0, stream>>>(b);
        CB200_CUDA_TRY(cudaGetLastError());
        g_launches.fetch_add(1, std::memory_order_relaxed);
    }
    if (plan.pack_a) {
        NvPackParams a = {};
        a.in = static_cast<const uint8_t*>(q.scale_a);
        a.out = sfa;
        a.rows = q.m;
        a.blocks = q.k / 16u;
        a.words = plan.words;
        if (q.group_count != 0) {
            a.group_list = q.group_list;
            a.list_i32 = q.group_list_type == CB200_GROUP_LIST_INT32 ? 1u : 0u;
            a.list_prefix = q.group_list_kind == CB200_GROUP_LIST_PREFIX_SUMS ? 1u : 0u;
            a.groups = q.group_count;
            a.tile_rows = plan.tile_rows;
            a.table = table;
            a.num_row_tiles = num_tiles;
        }
        const uint64_t warps = static_cast<uint64_t>(plan.sfa_blocks) * ((plan.words + 3u) / 4u);
        const uint64_t want = (warps + kNvPackThreads / 32 - 1) / (kNvPackThreads / 32);
        const uint64_t cap = static_cast<uint64_t>(dev->sm_count) * 4u;
        nvfp4_pack_scales_kernel<<<static_cast<uint32_t>(want < cap ? want : cap), kNvPackThreads, 0, stream>>>(a);
        CB200_CUDA_TRY(cudaGetLastError());
        g_launches.fetch_add(1, std::memory_order_relaxed);
    }
    NvParams p;
    p.m = q.m;
    p.n = q.n;
    p.k = q.k;
    p.num_k_blocks = (q.k + kNvStageK - 1u) / kNvStageK;
    p.words = plan.words;
    // A band of the tile order holds ~32 MB of A, so that its rows stay in L2 while the band's weight tiles go by.  Groups
    // have weights of their own: four row tiles, two groups or fewer at a time, keep those in L2 instead (64 groups of 512
    // rows, n 4096, k 7168: 455 us against 490; the same rows with one weight matrix: 406 us against 396).
    p.band_rows = static_cast<uint32_t>((32ull << 20) / (256ull * (q.k / 2u)));
    p.band_rows = p.band_rows < 2u ? 2u : (p.band_rows > 32u ? 32u : p.band_rows);
    p.band_rows = q.group_count != 0 ? 4u : p.band_rows;
    p.sfb_blocks = plan.sfb_blocks;
    p.d_type = q.d_type;
    p.sfa = plan.pack_a ? sfa : static_cast<const uint8_t*>(q.scale_a);
    p.sfb = plan.pack_b ? sfb : static_cast<const uint8_t*>(q.scale_b);
    p.alpha = q.alpha;
    p.d = q.d;
    p.status = dev->status;
    p.table = q.group_count != 0 ? table : nullptr;
    p.num_row_tiles = q.group_count != 0 ? num_tiles : nullptr;
    p.tma_store = 0;
    p.tile_x = kNvTileX;
    return plan.few ? launch_nv_few(q, plan, p, *dev, stream) : launch_nv_pair(q, plan, p, *dev, stream);
}

NvProblem nv_dense_problem(const cb200_nvfp4_matmul_args* a)
{
    NvProblem q = {};
    q.m = a->m;
    q.n = a->n;
    q.k = a->k;
    q.scale_a_layout = a->scale_a_layout;
    q.scale_b_layout = a->scale_b_layout;
    q.d_type = a->d_type;
    q.a = a->a;
    q.b = a->b;
    q.scale_a = a->scale_a;
    q.scale_b = a->scale_b;
    q.alpha = a->alpha;
    q.d = a->d;
    q.workspace = a->workspace;
    q.workspace_bytes = a->workspace_bytes;
    q.block_num = a->block_num;
    q.flags = a->flags;
    return q;
}

NvProblem nv_grouped_problem(const cb200_nvfp4_grouped_matmul_args* a)
{
    NvProblem q = {};
    q.m = a->m;
    q.n = a->n;
    q.k = a->k;
    q.group_count = a->group_count;
    q.group_list_type = a->group_list_type;
    q.group_list_kind = a->group_list_kind;
    q.scale_a_layout = CB200_NVFP4_SCALES_ROWS;
    q.scale_b_layout = a->scale_b_layout;
    q.d_type = a->d_type;
    q.a = a->a;
    q.b = a->b;
    q.group_list = a->group_list;
    q.scale_a = a->scale_a;
    q.scale_b = a->scale_b;
    q.alpha = a->alpha;
    q.d = a->d;
    q.workspace = a->workspace;
    q.workspace_bytes = a->workspace_bytes;
    q.block_num = a->block_num;
    q.flags = a->flags;
    return q;
}

}  // namespace

extern "C" {

int cb200_nvfp4_matmul_can_implement(const cb200_nvfp4_matmul_args* args)
{
    NvPlan plan;
    return args == nullptr ? CB200_INVALID : plan_nv(nv_dense_problem(args), &plan);
}

uint64_t cb200_nvfp4_matmul_workspace_size(const cb200_nvfp4_matmul_args* args)
{
    NvPlan plan;
    return args != nullptr && plan_nv(nv_dense_problem(args), &plan) == CB200_SUCCESS ? plan.total() : 0;
}

int cb200_nvfp4_matmul(const cb200_nvfp4_matmul_args* args, void* stream)
{
    return args == nullptr ? CB200_INVALID : run_nv(nv_dense_problem(args), stream);
}

int cb200_nvfp4_grouped_matmul_slice_m_can_implement(const cb200_nvfp4_grouped_matmul_args* args)
{
    NvPlan plan;
    return args == nullptr || args->group_count == 0 ? CB200_INVALID : plan_nv(nv_grouped_problem(args), &plan);
}

uint64_t cb200_nvfp4_grouped_matmul_slice_m_workspace_size(const cb200_nvfp4_grouped_matmul_args* args)
{
    NvPlan plan;
    return args != nullptr && args->group_count != 0 && plan_nv(nv_grouped_problem(args), &plan) == CB200_SUCCESS
               ? plan.total()
               : 0;
}

int cb200_nvfp4_grouped_matmul_slice_m(const cb200_nvfp4_grouped_matmul_args* args, void* stream)
{
    return args == nullptr || args->group_count == 0 ? CB200_INVALID : run_nv(nv_grouped_problem(args), stream);
}

}  // extern "C"
