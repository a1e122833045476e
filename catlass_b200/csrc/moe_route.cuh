// Routing of tokens to experts: scores, an optional bias, groups of experts, top-k, weights.
//
//   s[e]   = softmax_e(x) or 1 / (1 + exp(-x[e]));   key[e] = s[e] + bias[e], without a bias x[e] itself (same order)
//   a group's key is its largest key or the sum of its two largest; the experts of the best groups stay
//   ids = the top_k experts by key, ties to the lower index;  weights = s[ids] [/ their sum] * scaling
//
// One warp per token, kPer logits per lane (expert i * 32 + lane): a token's logits are read once, 64 or 128
// contiguous bytes per load, and everything else happens in registers, shuffles and redux.sync.
//
// Order.  The ids have to be those of the exact keys, but 32-bit scores carry a few units in the last place of error.
// Keys are compared as order-preserving integers (one redux.sync finds the warp's maximum); the kernel knows how far
// a 32-bit key can be off, and when two neighbours of the selected order (or the two groups at the border) are closer
// than that, the warp does its token again with 64-bit keys (route_select_exact).  Without a bias and without groups
// the logits are compared as they are, exactly.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cb200 {

constexpr int kRouteWarps = 4;  // tokens per CTA: small, so that a few tokens spread over the SMs

struct RouteParams {
    uint32_t tokens, experts, top_k, groups, groups_kept, per_group;
    uint32_t softmax, group_top2, renormalize, logits_type;
    float scaling;
    uint64_t pitch;
    const void* logits;
    const float* bias;
    const int32_t* token_count;
    float* weights;
    int32_t* ids;
};

// element i of a CB200_DTYPE_F32 / _BF16 / _F16 array (the type codes are those of the C ABI)
__device__ __forceinline__ float load_as_float(const void* p, uint64_t i, uint32_t type)
{
    if (type == 0) {
        return __ldg(static_cast<const float*>(p) + i);
    }
    const unsigned short raw = __ldg(static_cast<const unsigned short*>(p) + i);
    return type == 1 ? __uint_as_float(static_cast<uint32_t>(raw) << 16) : __half2float(__ushort_as_half(raw));
}

// A logit as the definition reads it: NaN cannot be chosen, like -inf.
__device__ __forceinline__ float route_logit(const RouteParams& p, uint32_t token, uint32_t e)
{
    const float x = load_as_float(p.logits, token * p.pitch + e, p.logits_type);
    return x == x ? x : -CUDART_INF_F;
}

// Unsigned integers in the order of the floats; every float maps above 0, which stands for "cannot be chosen".
__device__ __forceinline__ uint32_t route_order(float f)
{
    const uint32_t b = __float_as_uint(f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float route_unorder(uint32_t u)
{
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// exp(x - max) with the limit for logits of +inf (which share the softmax among themselves)
__device__ __forceinline__ float route_exp_diff(float x, float max)
{
    return x == max ? 1.0f : expf(x - max);
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, off);
    }
    return v;
}

__device__ __forceinline__ double warp_sum64(double v)
{
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, off);
    }
    return v;
}

// The two largest of a group's values (lanes of a group: `lanes` neighbours, a power of two), and the group's key.
// `vals` holds one value per expert; -inf: cannot be chosen.  Every lane of the warp calls this; lanes without a group
// get -inf.  The walk starts at another element in every group, so that the groups' reads fall on different banks.
template <class F>
__device__ __forceinline__ F route_group_key(const F* vals, uint32_t groups, uint32_t per_group, uint32_t lanes,
                                             uint32_t lane, bool top2, F minus_inf)
{
    const uint32_t g = lane / lanes, sub = lane % lanes;
    F first = minus_inf, second = minus_inf;
    if (g < groups) {
        const uint32_t steps = (per_group + lanes - 1) / lanes;
        uint32_t step = g % steps;
        for (uint32_t i = 0; i < steps; ++i) {
            const uint32_t at = sub + step * lanes;
            if (at < per_group) {
                const F v = vals[g * per_group + at];
                if (v > first) {
                    second = first;
                    first = v;
                } else if (v > second) {
                    second = v;
                }
            }
            step = step + 1 == steps ? 0 : step + 1;
        }
    }
    for (uint32_t off = 1; off < lanes; off <<= 1) {
        const F f = __shfl_xor_sync(0xffffffffu, first, off);
        const F s = __shfl_xor_sync(0xffffffffu, second, off);
        if (f > first) {
            second = first > s ? first : s;
            first = f;
        } else {
            second = f > second ? f : second;
        }
    }
    return top2 && second > minus_inf ? first + second : first;
}

// Bit g: group g is among the `kept` best (ties to the lower index).  All lanes get the mask.
template <class F>
__device__ __forceinline__ uint32_t route_keep_groups(F key, uint32_t groups, uint32_t kept, uint32_t lanes,
                                                      uint32_t lane)
{
    const uint32_t g = lane / lanes;
    uint32_t rank = 0;
    for (uint32_t h = 0; h < groups; ++h) {
        const F other = __shfl_sync(0xffffffffu, key, h * lanes);
        rank += (other > key || (other == key && h < g)) ? 1u : 0u;
    }
    const uint32_t at = __ballot_sync(0xffffffffu, g < groups && rank < kept);
    uint32_t mask = 0;
    for (uint32_t h = 0; h < groups; ++h) {
        mask |= ((at >> (h * lanes)) & 1u) << h;
    }
    return mask;
}

// The token's selection with 64-bit keys.  keys: shared memory of this warp, one double per expert.  Lane j receives
// the id of slot j in `id`; returns the number of slots filled.
__device__ __noinline__ uint32_t route_select_exact(const RouteParams& p, uint32_t token, double* keys,
                                                    uint32_t group_lanes, uint32_t lane, int32_t* id)
{
    const double kMinusInf = -CUDART_INF;
    float max = -CUDART_INF_F;
    double total = 1.0;
    if (p.softmax) {
        for (uint32_t e = lane; e < p.experts; e += 32) {
            max = fmaxf(max, route_logit(p, token, e));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            max = fmaxf(max, __shfl_xor_sync(0xffffffffu, max, off));
        }
        double sum = 0.0;
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const float x = route_logit(p, token, e);
            sum += x == max ? 1.0 : exp(static_cast<double>(x) - static_cast<double>(max));
        }
        total = warp_sum64(sum);
    }
    auto score = [&](float x) -> double {
        if (p.softmax) {
            return (x == max ? 1.0 : exp(static_cast<double>(x) - static_cast<double>(max))) / total;
        }
        return 1.0 / (1.0 + exp(-static_cast<double>(x)));
    };
    uint32_t keep = 0xffffffffu;
    __syncwarp();
    if (p.groups > 1) {
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const float x = route_logit(p, token, e);
            double v = kMinusInf;
            if (x > -CUDART_INF_F) {
                v = p.bias != nullptr ? score(x) + static_cast<double>(p.bias[e])
                                      : (p.group_top2 ? score(x) : static_cast<double>(x));
            }
            keys[e] = v > kMinusInf ? v : kMinusInf;
        }
        __syncwarp();
        const double g = route_group_key<double>(keys, p.groups, p.per_group, group_lanes, lane, p.group_top2 != 0,
                                                 kMinusInf);
        keep = route_keep_groups<double>(g, p.groups, p.groups_kept, group_lanes, lane);
        __syncwarp();
    }
    for (uint32_t e = lane; e < p.experts; e += 32) {
        const float x = route_logit(p, token, e);
        double v = kMinusInf;
        if (x > -CUDART_INF_F && ((keep >> (p.groups > 1 ? e / p.per_group : 0u)) & 1u) != 0) {
            v = p.bias != nullptr ? score(x) + static_cast<double>(p.bias[e]) : static_cast<double>(x);
        }
        keys[e] = v > kMinusInf ? v : kMinusInf;
    }
    uint32_t filled = 0;
    for (uint32_t j = 0; j < p.top_k; ++j) {
        double best = kMinusInf;
        uint32_t at = 0xffffffffu;
        for (uint32_t e = lane; e < p.experts; e += 32) {  // (each lane reads and clears its own experts only)
            if (keys[e] > best) {
                best = keys[e];
                at = e;
            }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const double b = __shfl_xor_sync(0xffffffffu, best, off);
            const uint32_t a = __shfl_xor_sync(0xffffffffu, at, off);
            if (b > best || (b == best && a < at)) {
                best = b;
                at = a;
            }
        }
        if (at == 0xffffffffu) {
            break;
        }
        if (at % 32 == lane) {
            keys[at] = kMinusInf;
        }
        if (lane == j) {
            *id = static_cast<int32_t>(at);
        }
        ++filled;
    }
    __syncwarp();
    return filled;
}

// Dynamic shared memory: kRouteWarps * experts doubles.
template <int kPer>
__global__ void __launch_bounds__(kRouteWarps * 32)
moe_route_kernel(const RouteParams p)
{
    extern __shared__ double route_smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t token = blockIdx.x * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    double* keys64 = route_smem + warp * p.experts;
    float* vals = reinterpret_cast<float*>(keys64);
    int32_t my_id = -1;
    uint32_t filled = 0;
    float max = -CUDART_INF_F, inv_total = 1.0f;
    const bool in_batch = p.token_count == nullptr || static_cast<int64_t>(token) < static_cast<int64_t>(*p.token_count);
    if (in_batch) {
        uint32_t group_lanes = 32;  // lanes that work on one group
        while (group_lanes * p.groups > 32) {
            group_lanes >>= 1;
        }
        float x[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t e = i * 32 + lane;
            x[i] = e < p.experts ? route_logit(p, token, e) : -CUDART_INF_F;
        }
        const bool score_needed = p.bias != nullptr || (p.groups > 1 && p.group_top2);
        float s[kPer];
        if (p.softmax) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                max = fmaxf(max, x[i]);
            }
            max = route_unorder(__reduce_max_sync(0xffffffffu, route_order(max)));
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                s[i] = route_exp_diff(x[i], max);
                sum += s[i];
            }
            inv_total = __frcp_rn(warp_sum(sum));
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                s[i] *= inv_total;
            }
        } else if (score_needed) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                s[i] = __fdividef(1.0f, 1.0f + expf(-x[i]));
            }
        }
        // keys as ordered integers; 0: cannot be chosen
        uint32_t order[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t e = i * 32 + lane;
            float key = x[i];
            if (p.bias != nullptr) {
                key = x[i] > -CUDART_INF_F ? s[i] + __ldg(p.bias + (e < p.experts ? e : 0)) : -CUDART_INF_F;
            }
            key += 0.0f;  // (-0 and +0 are the same key)
            order[i] = key > -CUDART_INF_F ? route_order(key) : 0u;
        }
        // How far apart two keys have to be to be told apart.  A sigmoid (at most 1) is off by 2^-22 from expf, 2^-24 from
        // the sum and 2^-22 from the quotient: two of them by less than 2^-19.  A softmax score (at most inv_total) is
        // off by 2^-22 from expf, |x - max| * 2^-24 from the difference (times the score: less than 2^-25), at most
        // 37 * 2^-24 from summing 1024 terms and 2^-23 from the quotient: two of them by less than 2^-17 * inv_total.
        // Adding the bias rounds once more, and a group's key is a sum of two keys.
        const float apart = p.softmax ? inv_total * 0x1p-17f : 0x1p-19f;
        bool suspect = false;
        if (p.groups > 1) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t e = i * 32 + lane;
                if (e < p.experts) {
                    const bool by_score = p.bias == nullptr && p.group_top2;
                    vals[e] = order[i] == 0 ? -CUDART_INF_F : (by_score ? s[i] : route_unorder(order[i]));
                }
            }
            __syncwarp();
            const float g = route_group_key<float>(vals, p.groups, p.per_group, group_lanes, lane, p.group_top2 != 0,
                                                   -CUDART_INF_F);
            const uint32_t keep = route_keep_groups<float>(g, p.groups, p.groups_kept, group_lanes, lane);
            if (p.bias != nullptr || p.group_top2) {
                const uint32_t mine = lane / group_lanes;
                const bool is_group = mine < p.groups, kept = is_group && ((keep >> mine) & 1u) != 0;
                const float low = route_unorder(__reduce_min_sync(0xffffffffu, kept ? route_order(g) : 0xffffffffu));
                const float high = route_unorder(
                    __reduce_max_sync(0xffffffffu, is_group && !kept ? route_order(g) : route_order(-CUDART_INF_F)));
                suspect = high > -CUDART_INF_F && low - high <= 2.0f * apart + 0x1p-21f * fabsf(low);
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t e = i * 32 + lane;
                const uint32_t mine = e / p.per_group;
                if (mine < p.groups && ((keep >> mine) & 1u) == 0) {
                    order[i] = 0;
                }
            }
        }
        const bool check = p.bias != nullptr;
        uint32_t last_order = 0, last_id = 0;
        const uint32_t rounds = p.top_k + (check ? 1u : 0u);  // (one more: the best that is not chosen)
        for (uint32_t j = 0; j < rounds && !suspect; ++j) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                best = order[i] > best ? order[i] : best;
            }
            const uint32_t top = __reduce_max_sync(0xffffffffu, best);
            if (top == 0) {
                break;
            }
            uint32_t at = 0xffffffffu;
#pragma unroll
            for (int i = kPer - 1; i >= 0; --i) {
                at = order[i] == top ? static_cast<uint32_t>(i) * 32 + lane : at;
            }
            at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                order[i] = static_cast<uint32_t>(i) * 32 + lane == at ? 0u : order[i];
            }
            if (check && j > 0) {
                const float above = route_unorder(last_order), here = route_unorder(top);
                if (above - here <= apart + 0x1p-22f * fabsf(above)) {
                    // the same logit with the same bias is the same key; anything else this close is not settled here
                    suspect = route_logit(p, token, at) != route_logit(p, token, last_id) || p.bias[at] != p.bias[last_id];
                }
            }
            last_order = top;
            last_id = at;
            if (j < p.top_k) {
                my_id = lane == j ? static_cast<int32_t>(at) : my_id;
                filled = j + 1;
            }
        }
        if (suspect) {
            my_id = -1;
            filled = route_select_exact(p, token, keys64, group_lanes, lane, &my_id);
        }
    }
    float w = 0.0f;
    if (lane < filled) {
        const float x = route_logit(p, token, static_cast<uint32_t>(my_id));
        w = p.softmax ? route_exp_diff(x, max) * inv_total : __fdividef(1.0f, 1.0f + expf(-x));
    }
    if (p.renormalize) {
        const float sum = warp_sum(w);
        w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
    }
    w *= p.scaling;
    if (lane < p.top_k) {
        const uint64_t at = static_cast<uint64_t>(token) * p.top_k + lane;
        p.ids[at] = lane < filled ? my_id : -1;
        p.weights[at] = lane < filled ? w : 0.0f;
    }
}

}  // namespace cb200
