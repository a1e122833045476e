// Combine: out[t] = round( shared_weight * shared[t] + sum_j weights[t][j] * d[position[t][j]] ), fp32, j ascending.
// HBM-bound: every row of D is read once, 16 bytes per thread and row, eight rows of a token in flight together.
// 8192 tokens x 8 rows x 7168 bf16: 159 us, 6.7 TB/s, the HBM copy rate (with CTAs of 256 threads, whose last one of a row is
// half empty, and a condition at each load: 179).  Rows off 16-byte boundaries: 5.0 TB/s in pairs (n 7166), 3.1 TB/s by
// single two-byte elements (n 7167), bound by load instructions; fp32 5.1.
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
    } else if constexpr (kVec == 2 && kType == 0) {
        const float2 raw = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(base) + at));
        v[0] = raw.x;
        v[1] = raw.y;
    } else if constexpr (kVec == 2) {
        const uint32_t raw = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(base) + at));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
        v[0] = kType == 1 ? __uint_as_float(raw << 16) : f.x;
        v[1] = kType == 1 ? __uint_as_float(raw & 0xFFFF0000u) : f.y;
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
        } else if constexpr (kVec == 2) {
            *reinterpret_cast<float2*>(o) = make_float2(v[0], v[1]);
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
        } else if constexpr (kVec == 2) {
            *reinterpret_cast<uint32_t*>(o) = bits(v[0]) | bits(v[1]) << 16;
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

// blockIdx.x: column chunk of kCombineThreads * kVec * kCols, blockIdx.y (strided): token.  A thread works on kVec
// neighbouring columns at kCols places, kCombineThreads * kVec apart: where rows allow no 16-byte loads, four places make
// up for the bytes that a narrow load has in flight.  kSlots rows are read together, without a branch between the loads: a
// slot that is skipped reads row 0 and drops it, a place past the row's end reads the row's last columns.  (With a
// condition at every load they went one after the other: 8192 x 8 x 7167 bf16 took 1170 us.)
template <int kDType, int kOutType, int kVec, int kCols, int kSlots>
__global__ void __launch_bounds__(kCombineThreads)
moe_combine_kernel(const CombineParams p)
{
    constexpr uint32_t kStep = kCombineThreads * kVec;
    const uint32_t first = blockIdx.x * kStep * kCols + threadIdx.x * kVec;
    if (first >= p.n) {
        return;
    }
    uint32_t col[kCols];
#pragma unroll
    for (int u = 0; u < kCols; ++u) {
        col[u] = first + u * kStep < p.n ? first + u * kStep : p.n - kVec;
    }
    for (uint32_t t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        float acc[kCols][kVec];
        const uint64_t out_at = static_cast<uint64_t>(t) * p.n;
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                acc[u][i] = 0.0f;
            }
            if (p.shared != nullptr) {
                float v[kVec];
                load_vec<kOutType, kVec>(p.shared, out_at + col[u], v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    acc[u][i] = p.shared_weight * v[i];
                }
            }
        }
        const uint64_t slot = static_cast<uint64_t>(t) * p.top_k;
        for (uint32_t j0 = 0; j0 < p.top_k && p.rows != 0; j0 += kSlots) {
            float v[kSlots][kCols][kVec], w[kSlots];
            bool valid[kSlots];
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
                const uint32_t at = j0 + j < p.top_k ? j0 + j : p.top_k - 1;
                const int32_t row = __ldg(p.position + slot + at);
                valid[j] = j0 + j < p.top_k && row >= 0 && static_cast<uint32_t>(row) < p.rows;
                w[j] = __ldg(p.weights + slot + at);
                const uint64_t base = static_cast<uint64_t>(valid[j] ? row : 0) * p.n;
#pragma unroll
                for (int u = 0; u < kCols; ++u) {
                    load_vec<kDType, kVec>(p.d, base + col[u], v[j][u]);
                }
            }
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
#pragma unroll
                for (int u = 0; u < kCols; ++u) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        acc[u][i] = valid[j] ? fmaf(w[j], v[j][u][i], acc[u][i]) : acc[u][i];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
            if (first + u * kStep < p.n) {
                store_vec<kOutType, kVec>(p.out, out_at + col[u], acc[u]);
            }
        }
    }
}

}  // namespace cb200
