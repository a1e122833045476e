// C-ABI entry points of the operators around the grouped matmuls: routing, dispatch, combine, NVFP4 quantisation.
// (Part of capi.cu's translation unit; uses its helpers.)
#pragma once

namespace {

bool is_float_type(uint32_t type)
{
    return type == CB200_DTYPE_F32 || type == CB200_DTYPE_BF16 || type == CB200_DTYPE_F16;
}

uint64_t float_bytes(uint32_t type)
{
    return type == CB200_DTYPE_F32 ? 4u : 2u;
}

bool aligned_to(const void* p, uintptr_t bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Launch with programmatic dependent launch on the kernel before it on the stream: for kernels that call
// grid_dependency_wait() before they touch anything that kernel writes.
template <class... Params, class... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), uint32_t grid, uint32_t threads, size_t smem,
                             cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// pairs per CTA of the counting sort: at most kSortChunks chunks, each a multiple of a CTA's threads
constexpr uint32_t kSortChunks = 128;
uint32_t dispatch_chunk(uint64_t pairs)
{
    const uint64_t per = (pairs + kSortChunks - 1) / kSortChunks;
    const uint64_t least = 2u * kDispatchThreads;
    return static_cast<uint32_t>(((per < least ? least : per) + kDispatchThreads - 1) / kDispatchThreads *
                                 kDispatchThreads);
}

uint64_t dispatch_counts_bytes(const cb200_moe_dispatch_args* a)
{
    const uint64_t pairs = static_cast<uint64_t>(a->tokens) * a->top_k;
    if (pairs <= kDispatchFusedPairs) {
        return 0;
    }
    const uint32_t chunk = dispatch_chunk(pairs);
    const uint64_t chunks = (pairs + chunk - 1) / chunk;
    return chunks <= 1 ? 0 : align256(chunks * a->experts * 4u);
}

int check_dispatch(const cb200_moe_dispatch_args* a)
{
    if (a == nullptr || a->experts == 0 || a->experts > kDispatchMaxExperts || a->top_k == 0 ||
        a->top_k > kDispatchMaxTopK || a->format > CB200_DISPATCH_NVFP4 || a->group_list == nullptr) {
        return CB200_INVALID;
    }
    if ((a->group_list_type != CB200_GROUP_LIST_INT64 && a->group_list_type != CB200_GROUP_LIST_INT32) ||
        (a->row_index_type != CB200_GROUP_LIST_INT64 && a->row_index_type != CB200_GROUP_LIST_INT32) ||
        (a->group_list_kind != CB200_GROUP_LIST_SIZES && a->group_list_kind != CB200_GROUP_LIST_PREFIX_SUMS)) {
        return CB200_INVALID;
    }
    if (!aligned_to(a->group_list, a->group_list_type == CB200_GROUP_LIST_INT64 ? 8 : 4) ||
        static_cast<uint64_t>(a->tokens) * a->top_k >= (1u << 24)) {
        return CB200_INVALID;
    }
    if (a->tokens == 0) {
        return CB200_SUCCESS;
    }
    if (a->ids == nullptr || a->position == nullptr || (a->row_weight != nullptr && a->weights == nullptr) ||
        !aligned_to(a->ids, 4) || !aligned_to(a->position, 4) || !aligned_to(a->weights, 4) ||
        !aligned_to(a->row_weight, 4) ||
        !aligned_to(a->row_index, a->row_index_type == CB200_GROUP_LIST_INT64 ? 8 : 4)) {
        return CB200_INVALID;
    }
    if (a->format == CB200_DISPATCH_INDEX || a->k == 0) {
        return CB200_SUCCESS;
    }
    if (a->x == nullptr || a->q == nullptr || !is_float_type(a->x_type) || !aligned16(a->x) || !aligned16(a->q) ||
        a->k > 0x7fffff00u) {
        return CB200_INVALID;
    }
    const uint64_t elem = float_bytes(a->x_type);
    const uint64_t pitch = a->x_pitch != 0 ? a->x_pitch : a->k;
    if (pitch < a->k || (pitch * elem) % 16u != 0) {
        return CB200_INVALID;
    }
    switch (a->format) {
        case CB200_DISPATCH_COPY:
            return (a->k * elem) % 16u == 0 ? CB200_SUCCESS : CB200_INVALID;
        case CB200_DISPATCH_INT8:
            return a->k % 16u == 0 && a->scale != nullptr && aligned_to(a->scale, 4) ? CB200_SUCCESS : CB200_INVALID;
        case CB200_DISPATCH_MX_E4M3:
            return a->k % 32u == 0 && a->scale != nullptr ? CB200_SUCCESS : CB200_INVALID;
        default:
            return a->k % 16u == 0 && a->scale != nullptr && a->tensor_scale != nullptr &&
                           aligned_to(a->tensor_scale, 4)
                       ? CB200_SUCCESS
                       : CB200_INVALID;
    }
}

template <int kFormat, int kType>
cudaError_t launch_rows(const DispatchParams& p, bool fused, cudaStream_t stream)
{
    if (fused) {
        moe_rows_kernel<kFormat, kType, true><<<p.tokens, kDispatchThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    return launch_dependent(moe_rows_kernel<kFormat, kType, false>, p.tokens, kDispatchThreads, 0, stream, p);
}

template <int kFormat>
cudaError_t launch_rows_typed(const DispatchParams& p, uint32_t type, bool fused, cudaStream_t stream)
{
    switch (type) {
        case CB200_DTYPE_F32: return launch_rows<kFormat, 0>(p, fused, stream);
        case CB200_DTYPE_BF16: return launch_rows<kFormat, 1>(p, fused, stream);
        default: return launch_rows<kFormat, 2>(p, fused, stream);
    }
}

cudaError_t launch_rows_format(const DispatchParams& p, uint32_t format, uint32_t type, bool fused, cudaStream_t stream)
{
    switch (format) {
        case CB200_DISPATCH_INDEX: return launch_rows<kRowsIndex, 0>(p, fused, stream);
        case CB200_DISPATCH_COPY:  // (bytes: only the element size matters)
            return type == CB200_DTYPE_F32 ? launch_rows<kRowsCopy, 0>(p, fused, stream)
                                           : launch_rows<kRowsCopy, 1>(p, fused, stream);
        case CB200_DISPATCH_INT8: return launch_rows_typed<kRowsInt8>(p, type, fused, stream);
        case CB200_DISPATCH_MX_E4M3: return launch_rows_typed<kRowsMxE4M3>(p, type, fused, stream);
        default: return launch_rows_typed<kRowsNvfp4>(p, type, fused, stream);
    }
}

template <int kDType, int kVec, int kCols, int kSlots>
cudaError_t launch_combine_out(const CombineParams& p, uint32_t out_type, cudaStream_t stream)
{
    constexpr uint32_t kWide = kCombineThreads * kVec * kCols;
    const dim3 grid((p.n + kWide - 1) / kWide, p.tokens < 65535u ? p.tokens : 65535u, 1);
    switch (out_type) {
        case CB200_DTYPE_F32: moe_combine_kernel<kDType, 0, kVec, kCols, kSlots><<<grid, kCombineThreads, 0, stream>>>(p); break;
        case CB200_DTYPE_BF16: moe_combine_kernel<kDType, 1, kVec, kCols, kSlots><<<grid, kCombineThreads, 0, stream>>>(p); break;
        default: moe_combine_kernel<kDType, 2, kVec, kCols, kSlots><<<grid, kCombineThreads, 0, stream>>>(p); break;
    }
    return cudaGetLastError();
}

template <int kVec, int kCols, int kSlots>
cudaError_t launch_combine(const CombineParams& p, uint32_t d_type, uint32_t out_type, cudaStream_t stream)
{
    switch (d_type) {
        case CB200_DTYPE_F32: return launch_combine_out<0, kVec, kCols, kSlots>(p, out_type, stream);
        case CB200_DTYPE_BF16: return launch_combine_out<1, kVec, kCols, kSlots>(p, out_type, stream);
        default: return launch_combine_out<2, kVec, kCols, kSlots>(p, out_type, stream);
    }
}

template <bool kSwiglu>
void launch_nv_quant(const NvQuantParams& p, uint32_t type, uint32_t grid, cudaStream_t stream)
{
    switch (type) {
        case CB200_DTYPE_F32: nvfp4_quantize_kernel<0, kSwiglu><<<grid, kNvQuantThreads, 0, stream>>>(p); break;
        case CB200_DTYPE_BF16: nvfp4_quantize_kernel<1, kSwiglu><<<grid, kNvQuantThreads, 0, stream>>>(p); break;
        default: nvfp4_quantize_kernel<2, kSwiglu><<<grid, kNvQuantThreads, 0, stream>>>(p); break;
    }
}

}  // namespace

extern "C" {

int cb200_moe_route_can_implement(const cb200_moe_route_args* a)
{
    if (a == nullptr || a->experts == 0 || a->experts > 1024u || a->groups == 0 || a->groups > 32u ||
        a->experts % a->groups != 0 || a->groups_kept == 0 || a->groups_kept > a->groups || a->top_k == 0 ||
        a->top_k > 32u || a->top_k > a->groups_kept * (a->experts / a->groups)) {
        return CB200_INVALID;
    }
    if (a->score > CB200_ROUTE_SIGMOID || a->group_score > CB200_ROUTE_GROUP_TOP2_SUM ||
        (a->flags & ~CB200_ROUTE_RENORMALIZE) != 0 || !is_float_type(a->logits_type) ||
        (a->logits_pitch != 0 && a->logits_pitch < a->experts)) {
        return CB200_INVALID;
    }
    if (a->tokens == 0) {
        return CB200_SUCCESS;
    }
    if (a->logits == nullptr || a->weights == nullptr || a->ids == nullptr ||
        !aligned_to(a->logits, float_bytes(a->logits_type)) || !aligned_to(a->bias, 4) ||
        !aligned_to(a->token_count, 4) || !aligned_to(a->weights, 4) || !aligned_to(a->ids, 4) ||
        a->tokens > 0x7fffff00u) {
        return CB200_INVALID;
    }
    return CB200_SUCCESS;
}

int cb200_moe_route(const cb200_moe_route_args* a, void* stream_v)
{
    int rc = cb200_moe_route_can_implement(a);
    if (rc != CB200_SUCCESS || a->tokens == 0) {
        return rc;
    }
    DeviceState* dev = nullptr;
    rc = device_state(&dev);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    RouteParams p;
    p.tokens = a->tokens;
    p.experts = a->experts;
    p.top_k = a->top_k;
    p.groups = a->groups_kept == a->groups ? 1u : a->groups;  // (all groups kept: nothing to choose)
    p.groups_kept = a->groups_kept;
    p.per_group = a->experts / p.groups;
    p.softmax = a->score == CB200_ROUTE_SOFTMAX ? 1u : 0u;
    p.group_top2 = a->group_score == CB200_ROUTE_GROUP_TOP2_SUM ? 1u : 0u;
    p.renormalize = (a->flags & CB200_ROUTE_RENORMALIZE) != 0 ? 1u : 0u;
    p.logits_type = a->logits_type;
    p.scaling = a->scaling;
    p.pitch = a->logits_pitch != 0 ? a->logits_pitch : a->experts;
    p.logits = a->logits;
    p.bias = a->bias;
    p.token_count = a->token_count;
    p.weights = a->weights;
    p.ids = a->ids;
    p.score_needed = a->bias != nullptr || (p.groups > 1 && p.group_top2) ? 1u : 0u;
    // lanes that hold a group when every lane has `per` experts; 0: groups are not whole lanes
    auto group_lanes = [&](uint32_t per) {
        const uint32_t lanes = p.per_group / per;
        return p.per_group % per == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0u;
    };
    uint32_t per = 1;  // logits per lane: 1, 2, 4 ... 32
    while (per * 32u < a->experts) {
        per *= 2;
    }
    const uint32_t per_many = a->experts <= 64u ? 8u : (a->experts <= 128u ? 16u : 32u);
    const uint32_t lanes_many = p.groups == 1u ? 8u : group_lanes(per_many);
    const bool many = a->tokens >= kRouteManyTokens && a->top_k <= 8u && a->experts > 16u && a->experts <= 256u &&
                      lanes_many != 0 && lanes_many * p.groups <= 8u * (p.groups == 1u ? 8u : 1u);
    per = many ? per_many : per;
    const uint64_t share = per * float_bytes(a->logits_type);  // bytes of a lane's logits
    const uint64_t step = share < 16u ? share : 16u;
    p.vector = (p.pitch * float_bytes(a->logits_type)) % step == 0 && aligned_to(a->logits, step) ? 1u : 0u;
    p.group_lanes = many ? lanes_many : (group_lanes(per) * p.groups <= 32u ? group_lanes(per) : 0u);
    p.walk_lanes = 32;
    while (p.walk_lanes * p.groups > 32u) {
        p.walk_lanes /= 2;
    }
    const uint32_t per_cta = many ? kRouteWarps * 4u : kRouteWarps;  // tokens
    const uint32_t grid = (a->tokens + per_cta - 1) / per_cta;
    const uint32_t smem = kRouteWarps * a->experts * 8u;
    const uint32_t threads = kRouteWarps * 32;
    if (many) {
        switch (per) {
            case 8: moe_route_many_kernel<8><<<grid, threads, smem, stream>>>(p); break;
            case 16: moe_route_many_kernel<16><<<grid, threads, smem, stream>>>(p); break;
            default: moe_route_many_kernel<32><<<grid, threads, smem, stream>>>(p); break;
        }
    } else {
        switch (per) {
            case 1: moe_route_kernel<1><<<grid, threads, smem, stream>>>(p); break;
            case 2: moe_route_kernel<2><<<grid, threads, smem, stream>>>(p); break;
            case 4: moe_route_kernel<4><<<grid, threads, smem, stream>>>(p); break;
            case 8: moe_route_kernel<8><<<grid, threads, smem, stream>>>(p); break;
            case 16: moe_route_kernel<16><<<grid, threads, smem, stream>>>(p); break;
            default: moe_route_kernel<32><<<grid, threads, smem, stream>>>(p); break;
        }
    }
    CB200_CUDA_TRY(cudaGetLastError());
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return CB200_SUCCESS;
}

int cb200_moe_dispatch_can_implement(const cb200_moe_dispatch_args* args)
{
    return check_dispatch(args);
}

uint64_t cb200_moe_dispatch_workspace_size(const cb200_moe_dispatch_args* args)
{
    return check_dispatch(args) == CB200_SUCCESS ? dispatch_counts_bytes(args) : 0;
}

int cb200_moe_dispatch(const cb200_moe_dispatch_args* a, void* stream_v)
{
    int rc = check_dispatch(a);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    const uint64_t ws = dispatch_counts_bytes(a);
    if (ws != 0 && (a->workspace == nullptr || a->workspace_bytes < ws || !aligned_to(a->workspace, 256))) {
        return CB200_INVALID;
    }
    DeviceState* dev = nullptr;
    rc = device_state(&dev);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    DispatchParams p;
    p.tokens = a->tokens;
    p.experts = a->experts;
    p.top_k = a->top_k;
    p.k = a->k;
    p.pairs = a->tokens * a->top_k;
    p.chunk = dispatch_chunk(p.pairs);
    p.chunks = p.pairs == 0 ? 1u : (p.pairs + p.chunk - 1) / p.chunk;
    p.expert_begin = a->expert_begin;
    p.list_i32 = a->group_list_type == CB200_GROUP_LIST_INT32 ? 1u : 0u;
    p.list_prefix = a->group_list_kind == CB200_GROUP_LIST_PREFIX_SUMS ? 1u : 0u;
    p.index_i32 = a->row_index_type == CB200_GROUP_LIST_INT32 ? 1u : 0u;
    p.x_pitch = a->x_pitch != 0 ? a->x_pitch : a->k;
    p.x = a->x;
    p.ids = a->ids;
    p.weights = a->weights;
    p.tensor_scale = a->tensor_scale;
    p.q = a->q;
    p.scale = a->scale;
    p.group_list = a->group_list;
    p.position = a->position;
    p.row_index = a->row_index;
    p.row_weight = a->row_weight;
    p.counts = static_cast<uint32_t*>(a->workspace);
    const uint32_t format = a->k == 0 ? CB200_DISPATCH_INDEX : a->format;
    if (a->tokens != 0 && p.pairs <= kDispatchFusedPairs) {
        CB200_CUDA_TRY(launch_rows_format(p, format, a->x_type, true, stream));
        g_launches.fetch_add(1, std::memory_order_relaxed);
        return CB200_SUCCESS;
    }
    const size_t smem = (kDispatchWarps + 2) * static_cast<size_t>(p.experts) * 4u;
    if (p.chunks > 1) {
        moe_count_kernel<<<p.chunks, kDispatchThreads, 0, stream>>>(p);
        CB200_CUDA_TRY(cudaGetLastError());
        CB200_CUDA_TRY(launch_dependent(moe_place_kernel, p.chunks, kDispatchThreads, smem, stream, p));
        g_launches.fetch_add(2, std::memory_order_relaxed);
    } else {
        moe_place_kernel<<<1, kDispatchThreads, smem, stream>>>(p);
        CB200_CUDA_TRY(cudaGetLastError());
        g_launches.fetch_add(1, std::memory_order_relaxed);
    }
    if (format != CB200_DISPATCH_INDEX && a->tokens != 0) {
        CB200_CUDA_TRY(launch_rows_format(p, format, a->x_type, false, stream));
        g_launches.fetch_add(1, std::memory_order_relaxed);
    }
    return CB200_SUCCESS;
}

int cb200_moe_combine_can_implement(const cb200_moe_combine_args* a)
{
    if (a == nullptr || a->reserved != 0 || a->top_k == 0 || a->top_k > static_cast<uint32_t>(kCombineMaxTopK) ||
        !is_float_type(a->d_type) || !is_float_type(a->out_type)) {
        return CB200_INVALID;
    }
    if (a->tokens == 0 || a->n == 0) {
        return CB200_SUCCESS;
    }
    if ((a->d == nullptr && a->rows != 0) || a->position == nullptr || a->weights == nullptr || a->out == nullptr ||
        !aligned_to(a->d, float_bytes(a->d_type)) || !aligned_to(a->position, 4) || !aligned_to(a->weights, 4) ||
        !aligned_to(a->out, float_bytes(a->out_type)) || !aligned_to(a->shared, float_bytes(a->out_type)) ||
        a->n > 0x7fffff00u || a->tokens > 0x7fffff00u || a->rows > 0x7fffffffu) {
        return CB200_INVALID;
    }
    return CB200_SUCCESS;
}

int cb200_moe_combine(const cb200_moe_combine_args* a, void* stream_v)
{
    int rc = cb200_moe_combine_can_implement(a);
    if (rc != CB200_SUCCESS || a->tokens == 0 || a->n == 0) {
        return rc;
    }
    DeviceState* dev = nullptr;
    rc = device_state(&dev);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    CombineParams p;
    p.tokens = a->tokens;
    p.top_k = a->top_k;
    p.n = a->n;
    p.rows = a->rows;
    p.shared_weight = a->shared_weight;
    p.d = a->d;
    p.position = a->position;
    p.weights = a->weights;
    p.shared = a->shared;
    p.out = a->out;
    // eight columns per thread where every row of every matrix starts on a 16-byte boundary, else pairs where it starts
    // on a pair's, else single ones, at four places each unless two CTAs cover a row
    const uintptr_t all = reinterpret_cast<uintptr_t>(a->d) | reinterpret_cast<uintptr_t>(a->out) |
                          reinterpret_cast<uintptr_t>(a->shared);
    if ((a->n & 7u) == 0 && (all & 15u) == 0) {
        CB200_CUDA_TRY((a->top_k <= 4u ? launch_combine<8, 1, 4>(p, a->d_type, a->out_type, stream)
                                       : launch_combine<8, 1, 8>(p, a->d_type, a->out_type, stream)));
    } else if ((a->n & 1u) == 0 && (all & 7u) == 0) {
        CB200_CUDA_TRY((a->n <= 2u * 2u * kCombineThreads ? launch_combine<2, 1, 8>(p, a->d_type, a->out_type, stream)
                                                          : launch_combine<2, 4, 8>(p, a->d_type, a->out_type, stream)));
    } else {
        CB200_CUDA_TRY((a->n <= 2u * kCombineThreads ? launch_combine<1, 1, 8>(p, a->d_type, a->out_type, stream)
                                                     : launch_combine<1, 4, 8>(p, a->d_type, a->out_type, stream)));
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return CB200_SUCCESS;
}

uint64_t cb200_nvfp4_tiled_scale_bytes(uint32_t rows, uint32_t k)
{
    return static_cast<uint64_t>((static_cast<uint64_t>(rows) + 127u) / 128u) * ((static_cast<uint64_t>(k) + 63u) / 64u) *
           512u;
}

int cb200_nvfp4_quantize_can_implement(const cb200_nvfp4_quantize_args* a)
{
    if (a == nullptr || !is_float_type(a->x_type) || a->scale_layout > CB200_NVFP4_SCALES_TILED ||
        (a->flags & ~CB200_NVFP4_SWIGLU) != 0 ||
        (a->row_count_type != CB200_GROUP_LIST_INT64 && a->row_count_type != CB200_GROUP_LIST_INT32)) {
        return CB200_INVALID;
    }
    if (a->rows == 0 || a->k == 0) {
        return CB200_SUCCESS;
    }
    if (a->x == nullptr || a->tensor_scale == nullptr || a->q == nullptr || a->scale == nullptr || a->k % 16u != 0 ||
        a->k > 0x3fffff00u || a->rows > 0x7fffff00u || !aligned16(a->x) || !aligned_to(a->q, 8) ||
        !aligned_to(a->tensor_scale, 4) ||
        !aligned_to(a->row_count, a->row_count_type == CB200_GROUP_LIST_INT64 ? 8 : 4)) {
        return CB200_INVALID;
    }
    const uint64_t width = (a->flags & CB200_NVFP4_SWIGLU) != 0 ? 2ull * a->k : a->k;
    const uint64_t pitch = a->x_pitch != 0 ? a->x_pitch : width;
    if (pitch < width || (pitch * float_bytes(a->x_type)) % 16u != 0) {
        return CB200_INVALID;
    }
    return CB200_SUCCESS;
}

int cb200_nvfp4_quantize(const cb200_nvfp4_quantize_args* a, void* stream_v)
{
    int rc = cb200_nvfp4_quantize_can_implement(a);
    if (rc != CB200_SUCCESS || a->rows == 0 || a->k == 0) {
        return rc;
    }
    DeviceState* dev = nullptr;
    rc = device_state(&dev);
    if (rc != CB200_SUCCESS) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool swiglu = (a->flags & CB200_NVFP4_SWIGLU) != 0;
    NvQuantParams p;
    p.rows = a->rows;
    p.blocks = a->k / 16u;
    p.words = (p.blocks + 3u) / 4u;
    p.tiled = a->scale_layout == CB200_NVFP4_SCALES_TILED ? 1u : 0u;
    p.count_i32 = a->row_count_type == CB200_GROUP_LIST_INT32 ? 1u : 0u;
    p.pitch = a->x_pitch != 0 ? a->x_pitch : (swiglu ? 2ull * a->k : a->k);
    p.x = a->x;
    p.tensor_scale = a->tensor_scale;
    p.row_count = a->row_count;
    p.q = static_cast<uint8_t*>(a->q);
    p.scale = static_cast<uint8_t*>(a->scale);
    const uint64_t want = (static_cast<uint64_t>(p.rows) * p.blocks + kNvQuantThreads - 1) / kNvQuantThreads;
    const uint64_t cap = static_cast<uint64_t>(dev->sm_count) * nv_quant_ctas(a->x_type == CB200_DTYPE_F32 ? 0 : 1, swiglu);
    const uint32_t grid = static_cast<uint32_t>(want < cap ? want : cap);
    p.word_stores = p.blocks % 4u == 0 && aligned_to(a->scale, 4) ? 1u : 0u;
    p.step_rows = grid * kNvQuantThreads / p.blocks;
    p.step_blocks = grid * kNvQuantThreads % p.blocks;
    p.step_elements = p.step_rows * p.pitch + static_cast<uint64_t>(p.step_blocks) * 16u;
    if (swiglu) {
        launch_nv_quant<true>(p, a->x_type, grid, stream);
    } else {
        launch_nv_quant<false>(p, a->x_type, grid, stream);
    }
    CB200_CUDA_TRY(cudaGetLastError());
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return CB200_SUCCESS;
}

}  // extern "C"
