// NVFP4 quantisation: 16 consecutive elements -> 16 E2M1 codes (8 bytes) and one E4M3 scale, in units of a tensor scale.
//
//   scale = e4m3( amax / (6 * tensor_scale) ),   q[i] = e2m1( x[i] * (1 / (scale * tensor_scale)) )
//
// A thread owns a block: it reads its 16 values with 16-byte loads, nothing is exchanged between threads.  HBM-bound:
// 2 (or 4) bytes read and 9/16 of a byte written per element.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "moe_combine.cuh"

namespace cb200 {

constexpr int kNvQuantThreads = 256;

// One block: its codes (element i in nibble i) and its scale byte.
__device__ __forceinline__ uint2 nvfp4_block(const float (&v)[16], float tensor_scale, uint32_t& scale_byte)
{
    uint32_t bits = 0;  // largest magnitude as an integer: NaN and Inf are the largest of all
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        bits = b > bits ? b : bits;
    }
    if (bits >= 0x7F800000u) {
        scale_byte = 0x7Fu;
        return make_uint2(0u, 0u);
    }
    const float ratio = __fdiv_rn(__uint_as_float(bits), 6.0f * tensor_scale);
    scale_byte = __nv_cvt_float_to_fp8(ratio, __NV_SATFINITE, __NV_E4M3);
    const float scale = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(scale_byte), __NV_E4M3)));
    const float inv = __frcp_rn(scale * tensor_scale);
    if (scale_byte == 0 || !(inv < __uint_as_float(0x7F800000u))) {
        scale_byte = 0;
        return make_uint2(0u, 0u);
    }
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t pair = __nv_cvt_float2_to_fp4x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_E2M1,
                                                       cudaRoundNearest);
        w[i >> 2] |= (pair & 0xFFu) << (8 * (i & 3));
    }
    return make_uint2(w[0], w[1]);
}

// act / (1 + exp(-act)) * gate, step by step in fp32 as the fused MX epilogue does
__device__ __forceinline__ float swiglu_f32(float act, float gate)
{
    return __fmul_rn(__fdiv_rn(act, __fadd_rn(expf(-act), 1.0f)), gate);
}

__device__ __forceinline__ int64_t load_count(const void* p, uint32_t is_i32)
{
    return is_i32 ? static_cast<int64_t>(*static_cast<const int32_t*>(p)) : *static_cast<const int64_t*>(p);
}

struct NvQuantParams {
    uint32_t rows, blocks;  // blocks of 16 per row
    uint32_t words;         // tiled: words of 4 blocks per row, ceil(blocks / 4)
    uint32_t tiled;
    uint32_t count_i32;
    uint64_t pitch;         // elements between rows of x
    const void* x;
    const float* tensor_scale;
    const void* row_count;
    uint8_t* q;
    uint8_t* scale;
};

__host__ __device__ inline uint64_t nvfp4_tiled_offset(uint32_t row, uint32_t block, uint32_t words)
{
    return (static_cast<uint64_t>(row / 128) * words + block / 4) * 512 + (row % 32) * 16 + (row % 128 / 32) * 4 +
           block % 4;
}

template <int kType, bool kSwiglu>
__global__ void __launch_bounds__(kNvQuantThreads)
nvfp4_quantize_kernel(const NvQuantParams p)
{
    const float tensor_scale = __ldg(p.tensor_scale);
    uint32_t rows = p.rows;
    if (p.row_count != nullptr) {
        const int64_t count = load_count(p.row_count, p.count_i32);
        rows = count < 0 ? 0u : (count < static_cast<int64_t>(rows) ? static_cast<uint32_t>(count) : rows);
    }
    const uint64_t items = static_cast<uint64_t>(rows) * p.blocks;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kNvQuantThreads;
    for (uint64_t item = blockIdx.x * static_cast<uint64_t>(kNvQuantThreads) + threadIdx.x; item < items; item += step) {
        const uint32_t row = static_cast<uint32_t>(item / p.blocks);
        const uint32_t block = static_cast<uint32_t>(item - static_cast<uint64_t>(row) * p.blocks);
        float v[16];
        const uint64_t at = row * p.pitch + static_cast<uint64_t>(block) * 16;
        load_vec<kType, 16>(p.x, at, v);
        if constexpr (kSwiglu) {
            float g[16];
            load_vec<kType, 16>(p.x, at + static_cast<uint64_t>(p.blocks) * 16, g);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = swiglu_f32(v[i], g[i]);
            }
        }
        uint32_t scale_byte;
        const uint2 codes = nvfp4_block(v, tensor_scale, scale_byte);
        *reinterpret_cast<uint2*>(p.q + item * 8) = codes;
        if (p.tiled) {
            p.scale[nvfp4_tiled_offset(row, block, p.words)] = static_cast<uint8_t>(scale_byte);
            if (block + 1 == p.blocks) {
                for (uint32_t b = p.blocks; b < p.words * 4; ++b) {  // the padding of the row's last word
                    p.scale[nvfp4_tiled_offset(row, b, p.words)] = 0;
                }
            }
        } else {
            p.scale[item] = static_cast<uint8_t>(scale_byte);
        }
    }
}

}  // namespace cb200
