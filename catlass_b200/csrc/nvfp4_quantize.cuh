// NVFP4 quantisation: 16 consecutive elements -> 16 E2M1 codes (8 bytes) and one E4M3 scale, in units of a tensor scale.
//
//   scale = e4m3( amax / (6 * tensor_scale) ),   q[i] = e2m1( x[i] * (1 / (scale * tensor_scale)) )
//
// A thread owns a block: it reads its 16 values with 16-byte loads, nothing is exchanged between threads.  HBM-bound:
// 2 (or 4) bytes read and 9/16 of a byte written per element.  bf16 32768 x 7168: 92 us = 6.5 TB/s, the HBM copy rate, scales
// tiled 94; 4111 x 7168: 14 us; fp32 8192 x 8192: 6.6 TB/s; SwiGLU in front, bf16 8192 x 4096: 27 us = 5.7 TB/s.  180
// instructions per block keep the SMs two thirds busy; without the next block's loads in flight the first took 126 us.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "moe_combine.cuh"

namespace cb200 {

constexpr int kNvQuantThreads = 256;
// CTAs of the quantiser that fit an SM; the grid is one such wave (more CTAs than that run in a second, emptier one)
__host__ __device__ constexpr int nv_quant_ctas(int type, bool swiglu) { return type == 0 || swiglu ? 4 : 5; }

// Eight values times inv -> eight E2M1 codes, value i in nibble i (nearest, ties to even, at most 6).
__device__ __forceinline__ uint32_t e2m1_codes8(const float* v, float inv)
{
    float y[8];
    const float2 f = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // (two products per instruction, each rounded as a product of its own)
        const float2 t = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), f);
        y[2 * i] = t.x;
        y[2 * i + 1] = t.y;
    }
    uint32_t w;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}\n"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

// The bit pattern of the largest magnitude: NaN and Inf are the largest of all.
__device__ __forceinline__ uint32_t amax_bits16(const float (&v)[16])
{
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        bits = b > bits ? b : bits;
    }
    return bits;
}

// One block whose largest magnitude has the given bit pattern: its codes (element i in nibble i) and its scale byte.
__device__ __forceinline__ uint2 nvfp4_block(const float (&v)[16], uint32_t amax_bits, float tensor_scale,
                                             uint32_t& scale_byte)
{
    if (amax_bits >= 0x7F800000u) {
        scale_byte = 0x7Fu;
        return make_uint2(0u, 0u);
    }
    const float ratio = __fdiv_rn(__uint_as_float(amax_bits), 6.0f * tensor_scale);
    scale_byte = __nv_cvt_float_to_fp8(ratio, __NV_SATFINITE, __NV_E4M3);
    const float scale = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(scale_byte), __NV_E4M3)));
    const float inv = __frcp_rn(scale * tensor_scale);
    if (scale_byte == 0 || !(inv < __uint_as_float(0x7F800000u))) {
        scale_byte = 0;
        return make_uint2(0u, 0u);
    }
    return make_uint2(e2m1_codes8(v, inv), e2m1_codes8(v + 8, inv));
}

// act / (1 + exp(-act)) * gate in fp32, from the approximate exponential and reciprocal: 2^-21 relative, plus |act| * 2^-24
__device__ __forceinline__ float swiglu_f32(float act, float gate)
{
    float t, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(act * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + t));
    return act * s * gate;
}

__device__ __forceinline__ int64_t load_count(const void* p, uint32_t is_i32)
{
    return is_i32 ? static_cast<int64_t>(*static_cast<const int32_t*>(p)) : *static_cast<const int64_t*>(p);
}

struct NvQuantParams {
    uint32_t rows, blocks;  // blocks of 16 per row
    uint32_t words;         // tiled: words of 4 blocks per row, ceil(blocks / 4)
    uint32_t tiled;
    uint32_t word_stores;   // rows have whole words and the words are aligned
    uint32_t step_rows, step_blocks;  // gridDim * 256 blocks as rows and blocks ...
    uint64_t step_elements;           // ... and as elements of x
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

// 16 elements as they lie in memory, and as floats
template <int kType>
struct Raw16 {
    uint4 w[kType == 0 ? 4 : 2];
    __device__ __forceinline__ void load(const void* base, uint64_t at)
    {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at * (kType == 0 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (kType == 0 ? 4 : 2); ++i) {
            w[i] = __ldg(src + i);
        }
    }
    // The bit pattern, as a float's, of the largest magnitude; two-byte types two at a time as they are.
    __device__ __forceinline__ uint32_t amax_bits() const
    {
        if constexpr (kType == 0) {
            float v[16];
            floats(v);
            return amax_bits16(v);
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                m = __vmaxu2(m, w[h].x & 0x7FFF7FFFu);
                m = __vmaxu2(m, w[h].y & 0x7FFF7FFFu);
                m = __vmaxu2(m, w[h].z & 0x7FFF7FFFu);
                m = __vmaxu2(m, w[h].w & 0x7FFF7FFFu);
            }
            const uint32_t top = (m >> 16) > (m & 0xFFFFu) ? m >> 16 : m & 0xFFFFu;
            return kType == 1 ? top << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top))));
        }
    }
    __device__ __forceinline__ void floats(float (&v)[16]) const
    {
#pragma unroll
        for (int h = 0; h < (kType == 0 ? 4 : 2); ++h) {
            const uint32_t x[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kType == 0) {
                    v[4 * h + i] = __uint_as_float(x[i]);
                } else if constexpr (kType == 1) {
                    v[8 * h + 2 * i] = __uint_as_float(x[i] << 16);
                    v[8 * h + 2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
                    v[8 * h + 2 * i] = f.x;
                    v[8 * h + 2 * i + 1] = f.y;
                }
            }
        }
    }
};

// The next block's loads are in flight while a block is worked on.  A thread's blocks are gridDim * 256 apart; (row,
// block) advance by that step without a division.  Four neighbouring lanes hold the four bytes of a scale word where a
// row has whole words (p.word_stores): one of them stores it.
template <int kType, bool kSwiglu>
__global__ void __launch_bounds__(kNvQuantThreads, nv_quant_ctas(kType, kSwiglu))
nvfp4_quantize_kernel(const NvQuantParams p)
{
    grid_launch_dependents();
    const float tensor_scale = __ldg(p.tensor_scale);
    uint32_t rows = p.rows;
    if (p.row_count != nullptr) {
        const int64_t count = load_count(p.row_count, p.count_i32);
        rows = count < 0 ? 0u : (count < static_cast<int64_t>(rows) ? static_cast<uint32_t>(count) : rows);
    }
    const uint32_t first = blockIdx.x * kNvQuantThreads + threadIdx.x;
    uint32_t row = first / p.blocks, block = first % p.blocks;
    Raw16<kType> raw, raw_gate;
    const uint64_t gate = static_cast<uint64_t>(p.blocks) * 16;
    uint64_t at = row * p.pitch + static_cast<uint64_t>(block) * 16;
    uint64_t item = first;
    auto fetch = [&]() {
        raw.load(p.x, at);
        if constexpr (kSwiglu) {
            raw_gate.load(p.x, at + gate);
        }
    };
    if (row < rows) {
        fetch();
    }
    while (row < rows) {
        float v[16];
        raw.floats(v);
        uint32_t amax;
        if constexpr (kSwiglu) {
            float g[16];
            raw_gate.floats(g);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = swiglu_f32(v[i], g[i]);
            }
            amax = amax_bits16(v);
        } else {
            amax = raw.amax_bits();
        }
        uint32_t next_row = row + p.step_rows, next_block = block + p.step_blocks;
        at += p.step_elements;
        if (next_block >= p.blocks) {
            next_block -= p.blocks;
            ++next_row;
            at += p.pitch - gate;
        }
        if (next_row < rows) {
            fetch();
        }
        uint32_t scale_byte;
        const uint2 codes = nvfp4_block(v, amax, tensor_scale, scale_byte);
        *reinterpret_cast<uint2*>(p.q + item * 8) = codes;
        if (p.word_stores) {
            // (the four lanes of a word are in the loop together: they share the row)
            const uint32_t lane = threadIdx.x & 31;
            const uint32_t mask = 0xFu << (lane & 28u);
            uint32_t word = scale_byte << (8 * (lane & 3u));
            word |= __shfl_xor_sync(mask, word, 1);
            word |= __shfl_xor_sync(mask, word, 2);
            if ((lane & 3u) == 0) {
                *reinterpret_cast<uint32_t*>(p.scale + (p.tiled ? nvfp4_tiled_offset(row, block, p.words) : item)) = word;
            }
        } else if (p.tiled) {
            p.scale[nvfp4_tiled_offset(row, block, p.words)] = static_cast<uint8_t>(scale_byte);
            if (block + 1 == p.blocks) {
                for (uint32_t b = p.blocks; b < p.words * 4; ++b) {  // the padding of the row's last word
                    p.scale[nvfp4_tiled_offset(row, b, p.words)] = 0;
                }
            }
        } else {
            p.scale[item] = static_cast<uint8_t>(scale_byte);
        }
        item += gridDim.x * kNvQuantThreads;
        row = next_row;
        block = next_block;
    }
}

}  // namespace cb200
