// Combine: out[t] = round( shared_weight * shared[t] + sum_j weights[t][j] * d[position[t][j]] ), fp32, j ascending.
// HBM-bound: every row of D is read once, 16 bytes per thread and row, eight rows of a token in flight together.
// 8192 tokens x 8 rows x 7168 bf16: 169 us, 6.26 TB/s, 0.96 of the HBM copy rate (CTAs of 256 threads, whose last one of a
// row is half empty: 179; of 64: 168, but 10.0 us instead of 6.5 for 7698 x 8 x 91 fp32).  Rows that do not start on 16-byte
// boundaries are read element by element: 1024 x 8 x 4100 bf16: 40 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "moe_route.cuh"

namespace cb200 {

constexpr int kCombineThreads = 128;
constexpr int kCombineMaxTopK = 32;

struct CombineParams {
    uint32_t tokens, top_k, n, rows;
    float shared_weight;
    const void* d;
    const int32_t* position;
    const float* weights;
    const void* shared;
    void* out;
};

// kVec elements of type code kType, 16 bytes (or one element) at p -> floats
template <int kType, int kVec>
__device__ __forceinline__ void load_vec(const void* base, uint64_t at, float (&v)[kVec])
{
    if constexpr (kVec == 1) {
        v[0] = load_as_float(base, at, kType);
    } else if constexpr (kType == 0) {
#pragma unroll
        for (int h = 0; h < kVec / 4; ++h) {
            const float4 raw = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at) + h);
            v[4 * h] = raw.x;
            v[4 * h + 1] = raw.y;
            v[4 * h + 2] = raw.z;
            v[4 * h + 3] = raw.w;
        }
    } else {
#pragma unroll
        for (int h = 0; h < kVec / 8; ++h) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at) + h);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kType == 1) {
                    v[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
                    v[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    v[8 * h + 2 * i] = f.x;
                    v[8 * h + 2 * i + 1] = f.y;
                }
            }
        }
    }
}

template <int kType, int kVec>
__device__ __forceinline__ void store_vec(void* base, uint64_t at, const float (&v)[kVec])
{
    if constexpr (kType == 0) {
        float* o = static_cast<float*>(base) + at;
        if constexpr (kVec == 1) {
            o[0] = v[0];
        } else {
#pragma unroll
            for (int h = 0; h < kVec / 4; ++h) {
                reinterpret_cast<float4*>(o)[h] = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
            }
        }
    } else {
        uint16_t* o = static_cast<uint16_t*>(base) + at;
        auto bits = [](float f) -> uint32_t {
            return kType == 1 ? static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(f)))
                              : static_cast<uint32_t>(__half_as_ushort(__float2half_rn(f)));
        };
        if constexpr (kVec == 1) {
            o[0] = static_cast<uint16_t>(bits(v[0]));
        } else {
#pragma unroll
            for (int h = 0; h < kVec / 8; ++h) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = bits(v[8 * h + 2 * i]) | bits(v[8 * h + 2 * i + 1]) << 16;
                }
                reinterpret_cast<uint4*>(o)[h] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// blockIdx.x: column chunk of kCombineThreads * kVec, blockIdx.y (strided): token.
template <int kDType, int kOutType, int kVec>
__global__ void __launch_bounds__(kCombineThreads)
moe_combine_kernel(const CombineParams p)
{
    const uint32_t col = (blockIdx.x * kCombineThreads + threadIdx.x) * kVec;
    if (col >= p.n) {
        return;
    }
    for (uint32_t t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        float acc[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            acc[i] = 0.0f;
        }
        const uint64_t out_at = static_cast<uint64_t>(t) * p.n + col;
        if (p.shared != nullptr) {
            float v[kVec];
            load_vec<kOutType, kVec>(p.shared, out_at, v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                acc[i] = p.shared_weight * v[i];
            }
        }
        const uint64_t slot = static_cast<uint64_t>(t) * p.top_k;
        for (uint32_t j0 = 0; j0 < p.top_k; j0 += 8) {
            float v[8][kVec], w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = 0.0f;
                const int32_t row = j0 + j < p.top_k ? __ldg(p.position + slot + j0 + j) : -1;
                if (row >= 0 && static_cast<uint32_t>(row) < p.rows) {
                    w[j] = __ldg(p.weights + slot + j0 + j);
                    load_vec<kDType, kVec>(p.d, static_cast<uint64_t>(row) * p.n + col, v[j]);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        v[j][i] = 0.0f;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    acc[i] = fmaf(w[j], v[j][i], acc[i]);
                }
            }
        }
        store_vec<kOutType, kVec>(p.out, out_at, acc);
    }
}

}  // namespace cb200
