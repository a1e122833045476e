// Dispatch of routed tokens: a stable counting sort of the (token, slot) pairs by expert, then every token's row is
// read and quantised once and written to each of its rows.
//
//   moe_count_kernel   pairs cut into one contiguous chunk per CTA; per chunk the number of pairs of every expert
//   moe_place_kernel   the same chunks: row of a pair = pairs of smaller experts + pairs of its expert in earlier chunks,
//                      earlier warps of its chunk and earlier pairs of its warp (match.any).  No atomics decide an
//                      order, so the rows are the same on every run.  With one chunk it counts by itself.
//   moe_rows_kernel    one CTA per token: x[t] -> codes and scales, written to the rows position[t][0 .. top_k)
// Up to kDispatchFusedPairs pairs everything is one launch of moe_rows_kernel: a CTA finds the rows of its own pairs
// by comparing them with all pairs (1024 pairs, 64 experts, k 4096, int8: 4.5 us; sorted, 1032 pairs: 6.7).
// HBM-bound on the rows written: 8192 tokens to 8 of 64 experts, k 7168 bf16: MX E4M3 105 us = 5.8 TB/s (0.88 of the copy
// rate; the sort 6.8 us of it), int8 102, NVFP4 69; 65536 pairs sorted without rows: 6.8 us, 1 M pairs of 256 experts: 36.
#pragma once

#include <stdint.h>

#include "mx_quantize.cuh"
#include "nvfp4_quantize.cuh"
#include "quant_int8.cuh"

namespace cb200 {

constexpr int kDispatchThreads = 256;
constexpr int kDispatchWarps = kDispatchThreads / 32;
constexpr uint32_t kDispatchMaxExperts = 1024;
constexpr uint32_t kDispatchMaxTopK = 32;
constexpr uint32_t kDispatchFusedPairs = 1024;

// formats, as in the C ABI
constexpr int kRowsIndex = 0, kRowsCopy = 1, kRowsInt8 = 2, kRowsMxE4M3 = 3, kRowsNvfp4 = 4;

struct DispatchParams {
    uint32_t tokens, experts, top_k, k;
    uint32_t pairs, chunk, chunks;   // chunk: pairs per CTA of the sort, a multiple of kDispatchThreads
    int32_t expert_begin;
    uint32_t list_i32, list_prefix, index_i32;
    uint64_t x_pitch;
    const void* x;
    const int32_t* ids;
    const float* weights;
    const float* tensor_scale;
    void* q;
    void* scale;
    void* group_list;
    int32_t* position;
    void* row_index;
    float* row_weight;
    uint32_t* counts;                // [chunks][experts]
};

// local expert of pair i, or `experts` when the pair is dropped
__device__ __forceinline__ uint32_t dispatch_expert(const DispatchParams& p, uint32_t i)
{
    const int64_t e = static_cast<int64_t>(__ldg(p.ids + i)) - p.expert_begin;
    return e >= 0 && e < static_cast<int64_t>(p.experts) ? static_cast<uint32_t>(e) : p.experts;
}

__device__ __forceinline__ void dispatch_write_list(const DispatchParams& p, uint32_t e, uint32_t count, uint32_t end)
{
    const uint32_t v = p.list_prefix ? end : count;
    if (p.list_i32) {
        static_cast<int32_t*>(p.group_list)[e] = static_cast<int32_t>(v);
    } else {
        static_cast<int64_t*>(p.group_list)[e] = static_cast<int64_t>(v);
    }
}

__device__ __forceinline__ void dispatch_write_row(const DispatchParams& p, uint32_t pair, uint32_t row)
{
    if (p.row_index != nullptr) {
        const uint32_t token = pair / p.top_k;
        if (p.index_i32) {
            static_cast<int32_t*>(p.row_index)[row] = static_cast<int32_t>(token);
        } else {
            static_cast<int64_t*>(p.row_index)[row] = static_cast<int64_t>(token);
        }
    }
    if (p.row_weight != nullptr) {
        p.row_weight[row] = __ldg(p.weights + pair);
    }
}

// Exclusive prefix sums of vals[0 .. n) in place, by one warp; all lanes take part.
__device__ __forceinline__ void warp_exclusive_scan(uint32_t* vals, uint32_t n, uint32_t lane)
{
    uint32_t carry = 0;
    for (uint32_t base = 0; base < n; base += 32) {
        const uint32_t v = base + lane < n ? vals[base + lane] : 0u;
        uint32_t sum = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t below = __shfl_up_sync(0xffffffffu, sum, off);
            sum += lane >= static_cast<uint32_t>(off) ? below : 0u;
        }
        if (base + lane < n) {
            vals[base + lane] = carry + sum - v;
        }
        carry += __shfl_sync(0xffffffffu, sum, 31);
    }
}

__global__ void __launch_bounds__(kDispatchThreads)
moe_count_kernel(const DispatchParams p)
{
    __shared__ uint32_t s_count[kDispatchMaxExperts];
    grid_launch_dependents();
    for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
        s_count[e] = 0;
    }
    __syncthreads();
    const uint32_t begin = blockIdx.x * p.chunk + threadIdx.x;
    for (uint32_t i = 0; i < p.chunk; i += 4 * kDispatchThreads) {
        uint32_t e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // (four loads in flight)
            const uint32_t pair = begin + i + u * kDispatchThreads;
            e[u] = i + u * kDispatchThreads < p.chunk && pair < p.pairs ? dispatch_expert(p, pair) : p.experts;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (e[u] < p.experts) {
                atomicAdd(s_count + e[u], 1u);
            }
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
        p.counts[static_cast<size_t>(blockIdx.x) * p.experts + e] = s_count[e];
    }
}

// Dynamic shared memory: (kDispatchWarps + 2) * experts words.
__global__ void __launch_bounds__(kDispatchThreads)
moe_place_kernel(const DispatchParams p)
{
    extern __shared__ uint32_t place_smem[];
    uint32_t* s_warp = place_smem;                                // [warps][experts]: counts, then the next row
    uint32_t* s_first = place_smem + kDispatchWarps * p.experts;  // [experts]: first row of an expert
    uint32_t* s_before = s_first + p.experts;                     // [experts]: pairs in earlier chunks
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_launch_dependents();
    for (uint32_t i = threadIdx.x; i < kDispatchWarps * p.experts; i += kDispatchThreads) {
        s_warp[i] = 0;
    }
    __syncthreads();
    // a warp owns a contiguous part of the chunk
    const uint32_t per_warp = p.chunk / kDispatchWarps;
    const uint32_t begin = blockIdx.x * p.chunk + warp * per_warp;
    uint32_t* mine = s_warp + warp * p.experts;
    for (uint32_t i = 0; i < per_warp; i += 128) {
        uint32_t e[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t at = i + u * 32 + lane;
            e[u] = at < per_warp && begin + at < p.pairs ? dispatch_expert(p, begin + at) : p.experts;
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            if (e[u] < p.experts) {
                atomicAdd(mine + e[u], 1u);
            }
        }
    }
    for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
        s_first[e] = 0;
        s_before[e] = 0;
    }
    __syncthreads();
    grid_dependency_wait();  // the chunks' counts
    if (p.chunks == 1) {
        for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
            uint32_t total = 0;
            for (int w = 0; w < kDispatchWarps; ++w) {
                total += s_warp[w * p.experts + e];
            }
            s_first[e] = total;
        }
    } else {
        // Sums of an expert's counts over all chunks and over those in front: a column of the table is shared by as many
        // threads as there are (one thread per expert walking 128 chunks took 5 us), eight loads of each in flight.
        uint32_t wide = 32;
        while (wide < p.experts && wide < kDispatchThreads) {
            wide *= 2;
        }
        const uint32_t parts = kDispatchThreads / wide, part = threadIdx.x / wide;
        for (uint32_t e = threadIdx.x % wide; e < p.experts; e += wide) {
            uint32_t before = 0, total = 0;
            for (uint32_t c0 = part; c0 < p.chunks; c0 += 8 * parts) {
                uint32_t v[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    const uint32_t c = c0 + u * parts;
                    v[u] = c < p.chunks ? p.counts[static_cast<size_t>(c) * p.experts + e] : 0u;
                }
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    total += v[u];
                    before += c0 + u * parts < blockIdx.x ? v[u] : 0u;
                }
            }
            atomicAdd(s_first + e, total);  // (integers: the order does not matter)
            atomicAdd(s_before + e, before);
        }
    }
    __syncthreads();
    if (warp == 0) {
        warp_exclusive_scan(s_first, p.experts, lane);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
        uint32_t row = s_first[e] + s_before[e];
        for (int w = 0; w < kDispatchWarps; ++w) {
            const uint32_t n = s_warp[w * p.experts + e];
            s_warp[w * p.experts + e] = row;
            row += n;
        }
        if (blockIdx.x + 1 == p.chunks) {  // the last chunk's rows end where the expert's rows end
            dispatch_write_list(p, e, row - s_first[e], row);
        }
    }
    __syncthreads();
    for (uint32_t i0 = 0; i0 < per_warp; i0 += 32) {  // (the same trips for every lane)
        const uint32_t pair = begin + i0 + lane;
        const bool inside = i0 + lane < per_warp && pair < p.pairs;
        const uint32_t e = inside ? dispatch_expert(p, pair) : p.experts;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const uint32_t below = __popc(same & ((1u << lane) - 1u));
        uint32_t row = 0;
        if (e < p.experts) {
            row = mine[e] + below;
        }
        __syncwarp();
        if (e < p.experts && below == 0) {
            mine[e] += __popc(same);
        }
        __syncwarp();
        if (inside) {
            p.position[pair] = e < p.experts ? static_cast<int32_t>(row) : -1;
            if (e < p.experts) {
                dispatch_write_row(p, pair, row);
            }
        }
    }
}

// 16 values of a row -> 16 E4M3 codes by the rule of cb200_mx_quantize; block_max: the largest magnitude of the 32
// values they belong to.  (The factor's shift of one part in 4096 turns the conversion's nearest-even into the rule's
// tie to the smaller magnitude; inputs with more than 8 significant bits are first cut to 11 plus a sticky twelfth:
// see mx_quantize_staged_kernel.)
template <int kType>
__device__ __forceinline__ uint4 mx_e4m3_codes16(float (&v)[16], float block_max, uint32_t& scale_byte)
{
    int exp = 0;
    if (!(block_max < 1e-12f)) {
        exp = static_cast<int>((__float_as_uint(block_max) >> 23) & 0xFFu) - 127 - 8;
    }
    scale_byte = static_cast<uint32_t>(exp + 127);
    const float inv = __uint_as_float((static_cast<uint32_t>(126 - exp) << 23) | 0x007FF000u);
    uint32_t words[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float t[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float u = v[w * 4 + 2 * b + i];
                if constexpr (kType != 1) {
                    const uint32_t bits = __float_as_uint(u);
                    u = __uint_as_float((bits & 0xFFFFE000u) | ((bits & 0x00001FFFu) != 0 ? 0x00001000u : 0u));
                }
                t[i] = u * inv;
            }
            word |= mx_codes2_nudged<false>(t[0], t[1]) << (16 * b);
        }
        words[w] = word;
    }
    return make_uint4(words[0], words[1], words[2], words[3]);
}

// One CTA per token.  kFused: the CTA first finds the rows of its pairs itself and CTA 0 writes the group list;
// otherwise position comes from moe_place_kernel.
template <int kFormat, int kType, bool kFused>
__global__ void __launch_bounds__(kDispatchThreads)
moe_rows_kernel(const DispatchParams p)
{
    __shared__ int32_t s_row[kDispatchMaxTopK];
    __shared__ uint32_t s_expert[kFused ? kDispatchFusedPairs : 1];
    __shared__ uint32_t s_count[kFused ? kDispatchMaxExperts : 1];
    __shared__ float s_max[kDispatchWarps];
    const uint32_t token = blockIdx.x;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t kElemBytes = kType == 0 ? 4u : 2u;

    if constexpr (kFused) {
        for (uint32_t i = threadIdx.x; i < p.pairs; i += kDispatchThreads) {
            s_expert[i] = dispatch_expert(p, i);
        }
        __syncthreads();
        for (uint32_t j = warp; j < p.top_k; j += kDispatchWarps) {
            const uint32_t pair = token * p.top_k + j;
            const uint32_t e = s_expert[pair];
            uint32_t before = 0;
            for (uint32_t i = lane; i < p.pairs; i += 32) {
                const uint32_t other = s_expert[i];
                before += (other < e || (other == e && i < pair)) ? 1u : 0u;
            }
            const uint32_t row = __reduce_add_sync(0xffffffffu, before);
            if (lane == 0) {
                const bool kept = e < p.experts;
                s_row[j] = kept ? static_cast<int32_t>(row) : -1;
                p.position[pair] = kept ? static_cast<int32_t>(row) : -1;
                if (kept) {
                    dispatch_write_row(p, pair, row);
                }
            }
        }
        if (token == 0) {
            for (uint32_t e = threadIdx.x; e < p.experts; e += kDispatchThreads) {
                s_count[e] = 0;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < p.pairs; i += kDispatchThreads) {
                if (s_expert[i] < p.experts) {
                    atomicAdd(s_count + s_expert[i], 1u);
                }
            }
            __syncthreads();
            uint32_t count[kDispatchMaxExperts / kDispatchThreads];
#pragma unroll
            for (uint32_t i = 0; i < kDispatchMaxExperts / kDispatchThreads; ++i) {
                const uint32_t e = threadIdx.x + i * kDispatchThreads;
                count[i] = e < p.experts ? s_count[e] : 0u;
            }
            __syncthreads();
            if (warp == 0) {
                warp_exclusive_scan(s_count, p.experts, lane);
            }
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kDispatchMaxExperts / kDispatchThreads; ++i) {
                const uint32_t e = threadIdx.x + i * kDispatchThreads;
                if (e < p.experts) {
                    dispatch_write_list(p, e, count[i], s_count[e] + count[i]);
                }
            }
        }
        __syncthreads();
    }
    // The rows of this token's pairs.  In front of the wait x may be read (it was complete before the count kernel
    // started), nothing may be written.
    auto rows_known = [&]() {
        if constexpr (!kFused) {
            grid_dependency_wait();
            if (threadIdx.x < p.top_k) {
                s_row[threadIdx.x] = p.position[static_cast<uint64_t>(token) * p.top_k + threadIdx.x];
            }
            __syncthreads();
        }
    };
    if constexpr (kFormat == kRowsIndex) {
        return;
    }
    const uint8_t* xr = static_cast<const uint8_t*>(p.x) + token * p.x_pitch * kElemBytes;
    if constexpr (kFormat == kRowsCopy) {
        rows_known();
        const uint32_t vecs = p.k * kElemBytes / 16;
        for (uint32_t c = threadIdx.x; c < vecs; c += kDispatchThreads) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(xr) + c);
            for (uint32_t j = 0; j < p.top_k; ++j) {
                if (s_row[j] >= 0) {
                    reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.q) +
                                             static_cast<uint64_t>(s_row[j]) * p.k * kElemBytes)[c] = v;
                }
            }
        }
        return;
    }
    const uint32_t blocks = p.k / 16;
    float inv = 0.0f;
    if constexpr (kFormat == kRowsInt8) {
        float amax = 0.0f;
        for (uint32_t c = threadIdx.x; c < blocks; c += kDispatchThreads) {
            float v[16];
            load_vec<kType, 16>(xr, static_cast<uint64_t>(c) * 16, v);
            amax = quant_int8_amax16(v, amax);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        }
        if (lane == 0) {
            s_max[warp] = amax;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kDispatchWarps; ++w) {
            amax = fmaxf(amax, s_max[w]);
        }
        inv = amax > 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
        rows_known();
        if (threadIdx.x < p.top_k && s_row[threadIdx.x] >= 0) {
            static_cast<float*>(p.scale)[s_row[threadIdx.x]] = __fdiv_rn(amax, 127.0f);
        }
    }
    const float tensor_scale = kFormat == kRowsNvfp4 ? __ldg(p.tensor_scale) : 0.0f;
    const uint32_t ks = (p.k / 32 + 1u) & ~1u;
    Raw16<kType> raw;
    if (threadIdx.x < blocks) {
        raw.load(xr, static_cast<uint64_t>(threadIdx.x) * 16);
    }
    if constexpr (kFormat != kRowsInt8) {
        rows_known();
    }
    // (the same trips for every lane: the maximum of an MX block is exchanged between the two lanes that share it)
    for (uint32_t c0 = 0; c0 < blocks; c0 += kDispatchThreads) {
        const uint32_t c = c0 + threadIdx.x;
        const bool active = c < blocks;
        float v[16];
        if (active) {
            raw.floats(v);
            if (c + kDispatchThreads < blocks) {
                raw.load(xr, static_cast<uint64_t>(c + kDispatchThreads) * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = 0.0f;
            }
        }
        uint32_t scale_byte = 0;
        uint4 codes = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kFormat == kRowsInt8) {
            codes = quant_int8_codes16(v, inv);
        } else if constexpr (kFormat == kRowsMxE4M3) {
            float block_max = quant_int8_amax16(v, 0.0f);
            block_max = fmaxf(block_max, __shfl_xor_sync(0xffffffffu, block_max, 1));
            codes = mx_e4m3_codes16<kType>(v, block_max, scale_byte);
        } else {
            const uint2 packed = nvfp4_block(v, amax_bits16(v), tensor_scale, scale_byte);
            codes.x = packed.x;
            codes.y = packed.y;
        }
        if (!active) {
            continue;
        }
        for (uint32_t j = 0; j < p.top_k; ++j) {
            if (s_row[j] < 0) {
                continue;
            }
            const uint64_t row = static_cast<uint64_t>(s_row[j]);
            uint8_t* q = static_cast<uint8_t*>(p.q);
            uint8_t* scale = static_cast<uint8_t*>(p.scale);
            if constexpr (kFormat == kRowsNvfp4) {
                *reinterpret_cast<uint2*>(q + row * (p.k / 2) + c * 8) = make_uint2(codes.x, codes.y);
                scale[row * blocks + c] = static_cast<uint8_t>(scale_byte);
            } else {
                *reinterpret_cast<uint4*>(q + row * p.k + c * 16) = codes;
                if constexpr (kFormat == kRowsMxE4M3) {
                    if ((c & 1u) == 0) {
                        scale[row * ks + c / 2] = static_cast<uint8_t>(scale_byte);
                        if (c + 2 == blocks && ks != p.k / 32) {
                            scale[row * ks + ks - 1] = 127;  // the padding column
                        }
                    }
                }
            }
        }
    }
}

}  // namespace cb200
