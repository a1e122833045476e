// Routing of tokens to experts: scores, an optional bias, groups of experts, top-k, weights.
//
//   s[e]   = softmax_e(x) or 1 / (1 + exp(-x[e]));   key[e] = s[e] + bias[e], without a bias x[e] itself (same order)
//   a group's key is its largest key or the sum of its two largest; the experts of the best groups stay
//   ids = the top_k experts by key, ties to the lower index;  weights = s[ids] [/ their sum] * scaling
//
// One warp per token, kPer consecutive logits per lane, read once with wide loads; everything else happens in
// registers, shuffles and redux.sync.  A lane sorts its keys, the warp picks the largest of the lanes' first keys.
//
// Bound by instruction issue and, for one token, by latency: ~950 instructions per token here, ~450 in the kernel that
// shares a warp among four tokens (below); reading 16384 x 256 bf16 logits takes 1.4 us of the 16.4.
//
// Order.  The ids have to be those of the exact keys, but 32-bit scores carry a few units in the last place of error.
// Keys are compared as order-preserving integers; the kernel knows how far a 32-bit key can be off, and when two
// neighbours of the selected order are closer than that, the candidates' keys are worked out in 64 bits, a lane each.
// When two groups at the border are, or softmax scores with a bias, the warp does the whole token again with 64-bit keys
// (route_select_exact).  Logits that decide by themselves (no bias) are compared as they are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cb200 {

// From so many tokens on four of them share a warp, where the experts allow it.  256 experts in 8 groups with a bias, one /
// four tokens per warp: 512 tokens 4.7 / 6.4 us, 4096 7.9 / 7.9, 16384 23 / 16, 131072 144 / 96; 60 experts: 512 3.6 / 4.2,
// 4099 4.6 / 4.5, 16384 10.6 / 8.1.
constexpr uint32_t kRouteManyTokens = 4096;
constexpr int kRouteWarps = 4;  // tokens per CTA: small, so that a few tokens spread over the SMs

struct RouteParams {
    uint32_t tokens, experts, top_k, groups, groups_kept, per_group;
    uint32_t softmax, group_top2, renormalize, logits_type;
    uint32_t score_needed;  // a key, of an expert or a group, is made of scores
    uint32_t vector;        // every token's row starts on a boundary of a lane's share of it
    uint32_t group_lanes;   // lanes that hold exactly one group (a power of two), or 0: groups are walked in shared memory
    uint32_t walk_lanes;    // ... by so many lanes each (a power of two)
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

// Unsigned integers in the order of the doubles, 0 below them all.
__device__ __forceinline__ unsigned long long route_order64(double f)
{
    const unsigned long long b = __double_as_longlong(f);
    return b ^ (static_cast<unsigned long long>(static_cast<long long>(b) >> 63) | 0x8000000000000000ull);
}

// The token's selection with 64-bit keys, kPer experts (i * 32 + lane) per lane.  keys: shared memory of this warp, one
// double per expert, for the groups' walk.  Lane j receives the id of slot j in `id`; returns the number of slots filled.
template <int kPer>
__device__ __noinline__ uint32_t route_select_exact(const RouteParams& p, uint32_t token, double* keys, uint32_t lane,
                                                    int32_t* id)
{
    constexpr uint32_t kAll = 0xffffffffu;
    const double kMinusInf = -CUDART_INF;
    float x[kPer];
    double s[kPer], key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint32_t e = i * 32 + lane;
        x[i] = e < p.experts ? route_logit(p, token, e) : -CUDART_INF_F;
    }
    if (p.softmax) {
        float max = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            max = fmaxf(max, x[i]);
        }
        max = route_unorder(__reduce_max_sync(kAll, route_order(max)));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] = x[i] == max ? 1.0 : exp(static_cast<double>(x[i]) - static_cast<double>(max));
            sum += s[i];
        }
        sum = warp_sum64(sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] /= sum;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] = 1.0 / (1.0 + exp(-static_cast<double>(x[i])));
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint32_t e = i * 32 + lane;
        key[i] = p.bias == nullptr ? static_cast<double>(x[i])
                                   : s[i] + static_cast<double>(e < p.experts ? p.bias[e] : 0.0f);
        key[i] = x[i] > -CUDART_INF_F && key[i] > kMinusInf ? key[i] + 0.0 : kMinusInf;
    }
    if (p.groups > 1) {
        const bool by_score = p.bias == nullptr && p.group_top2;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t e = i * 32 + lane;
            if (e < p.experts) {
                keys[e] = by_score ? (key[i] > kMinusInf ? s[i] : kMinusInf) : key[i];
            }
        }
        __syncwarp();
        const double g = route_group_key<double>(keys, p.groups, p.per_group, p.walk_lanes, lane, p.group_top2 != 0,
                                                 kMinusInf);
        const uint32_t keep = route_keep_groups<double>(g, p.groups, p.groups_kept, p.walk_lanes, lane);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t of = (i * 32 + lane) / p.per_group;
            key[i] = of < p.groups && ((keep >> of) & 1u) != 0 ? key[i] : kMinusInf;
        }
        __syncwarp();
    }
    uint32_t filled = 0;
    for (uint32_t j = 0; j < p.top_k; ++j) {
        double best = kMinusInf;
        uint32_t at = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (key[i] > best) {
                best = key[i];
                at = i * 32 + lane;
            }
        }
        const unsigned long long order = best > kMinusInf ? route_order64(best) : 0ull;
        const uint32_t high = __reduce_max_sync(kAll, static_cast<uint32_t>(order >> 32));
        if (high == 0) {  // (a finite key is above 2^52 in this order)
            break;
        }
        const bool still = static_cast<uint32_t>(order >> 32) == high;
        const uint32_t low = __reduce_max_sync(kAll, still ? static_cast<uint32_t>(order) : 0u);
        at = __reduce_min_sync(kAll, still && static_cast<uint32_t>(order) == low ? at : kAll);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            key[i] = i * 32 + lane == at ? kMinusInf : key[i];
        }
        if (lane == j) {
            *id = static_cast<int32_t>(at);
        }
        ++filled;
    }
    return filled;
}

// The order of n candidates (one per lane) by their keys in 64 bits, equal ones by index; lane j < filled gets slot j's.
__device__ __noinline__ int32_t route_resolve(const RouteParams& p, uint32_t token, uint32_t candidate, uint32_t n,
                                              uint32_t filled, uint32_t lane)
{
    double key = 0.0;
    if (lane < n) {
        const double x = static_cast<double>(route_logit(p, token, candidate));
        key = p.bias == nullptr ? x : 1.0 / (1.0 + exp(-x)) + static_cast<double>(p.bias[candidate]);
    }
    uint32_t rank = 0;
    for (uint32_t h = 0; h < n; ++h) {
        const double other = __shfl_sync(0xffffffffu, key, h);
        const uint32_t at = __shfl_sync(0xffffffffu, candidate, h);
        rank += (other > key || (other == key && at < candidate)) ? 1u : 0u;
    }
    int32_t id = -1;
    for (uint32_t h = 0; h < n; ++h) {
        const uint32_t to = __shfl_sync(0xffffffffu, rank, h), at = __shfl_sync(0xffffffffu, candidate, h);
        id = to == lane && lane < filled ? static_cast<int32_t>(at) : id;
    }
    return id;
}

// kPer consecutive logits of a token, expert e0 first, as they are (-inf past the last expert): one or a few wide loads where every
// token's row starts on a boundary of a lane's share (p.vector), single ones otherwise.
template <int kPer>
__device__ __forceinline__ void route_load(const RouteParams& p, uint32_t token, uint32_t e0, float (&x)[kPer])
{
    if (!p.vector || e0 + kPer > p.experts) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] = e0 + i < p.experts ? load_as_float(p.logits, token * p.pitch + e0 + i, p.logits_type) : -CUDART_INF_F;
        }
        return;
    }
    const uint64_t at = token * p.pitch + e0;
    constexpr int kWords32 = kPer;
    uint32_t w[kPer];
    auto load = [&](const void* src, int words) {
        if (words % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kPer / 4; ++i) {
                if (4 * i < words) {
                    const uint4 v = __ldg(static_cast<const uint4*>(src) + i);
                    w[4 * i] = v.x;
                    w[4 * i + 1] = v.y;
                    w[4 * i + 2] = v.z;
                    w[4 * i + 3] = v.w;
                }
            }
        } else if (words == 2) {
            const uint2 v = __ldg(static_cast<const uint2*>(src));
            w[0] = v.x;
            w[kPer > 1 ? 1 : 0] = v.y;
        } else {
            w[0] = __ldg(static_cast<const uint32_t*>(src));
        }
    };
    if (p.logits_type == 0) {
        load(static_cast<const float*>(p.logits) + at, kWords32);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] = __uint_as_float(w[i]);
        }
    } else if constexpr (kPer == 1) {
        x[0] = load_as_float(p.logits, at, p.logits_type);
    } else {
        load(static_cast<const uint16_t*>(p.logits) + at, kPer / 2);
#pragma unroll
        for (int i = 0; i < kPer / 2; ++i) {
            if (p.logits_type == 1) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
}

// Sorts v descending (odd-even merge sort, all indices known at compile time).
template <int kN>
__device__ __forceinline__ void sort_descending(uint32_t (&v)[kN])
{
#pragma unroll
    for (int part = 1; part < kN; part <<= 1) {
#pragma unroll
        for (int k = part; k >= 1; k >>= 1) {
#pragma unroll
            for (int j = k % part; j + k < kN; j += 2 * k) {
#pragma unroll
                for (int i = 0; i < k; ++i) {
                    if (i + j + k < kN && (i + j) / (2 * part) == (i + j + k) / (2 * part)) {
                        const uint32_t a = v[i + j], b = v[i + j + k];
                        v[i + j] = a > b ? a : b;
                        v[i + j + k] = a > b ? b : a;
                    }
                }
            }
        }
    }
}

// 1 / (1 + exp(-x)) from the two approximate instructions (2^-22 and 2^-23 relative): for keys, not for weights
__device__ __forceinline__ float route_sigmoid_fast(float x)
{
    float t, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(x * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + t));
    return s;
}

// Dynamic shared memory: kRouteWarps * experts doubles.
template <int kPer>
__global__ void __launch_bounds__(kRouteWarps * 32)
moe_route_kernel(const __grid_constant__ RouteParams p)
{
    extern __shared__ double route_smem[];
    constexpr uint32_t kAll = 0xffffffffu;
    constexpr uint32_t kLow = kPer - 1;  // low bits of a key that hold the expert's place in its lane
    const float kMinusInf = -CUDART_INF_F;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t e0 = lane * kPer;
    const bool exact_keys = p.bias == nullptr;
    const uint32_t token = blockIdx.x * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    {
        int32_t my_id = -1;
        uint32_t filled = 0;
        float max = kMinusInf, inv_total = 1.0f;
        if (p.token_count == nullptr || static_cast<int64_t>(token) < static_cast<int64_t>(*p.token_count)) {
            float x[kPer], s[kPer], bias[kPer];
            route_load<kPer>(p, token, e0, x);
            // A lane whose logits and biases are all numbers needs no checks below; that is every lane of most warps.
            bool numbers = e0 + kPer <= p.experts;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                bias[i] = !exact_keys && e0 + i < p.experts ? __ldg(p.bias + e0 + i) : 0.0f;
                numbers = numbers && x[i] > kMinusInf && bias[i] > kMinusInf;
            }
            const bool clean = __all_sync(kAll, numbers);
            if (!clean) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    x[i] = x[i] > kMinusInf && bias[i] > kMinusInf ? x[i] : kMinusInf;  // (NaN cannot be chosen either)
                }
            }
            if (p.softmax) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    max = fmaxf(max, x[i]);
                }
                max = route_unorder(__reduce_max_sync(kAll, route_order(max)));
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
            } else if (p.score_needed) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    s[i] = route_sigmoid_fast(x[i]);
                }
            }
            // keys; -inf: cannot be chosen
            float key[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                key[i] = exact_keys ? x[i] + 0.0f : s[i] + bias[i];  // (-0 and +0 are the same logit)
            }
            if (!clean) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    key[i] = x[i] > kMinusInf ? key[i] : kMinusInf;
                }
            }
            // How far apart two keys have to be to be told apart.  A sigmoid (at most 1) is off by 2^-24 from the
            // exponential (s * (1 - s) <= 1/4 of its 2^-22), less than 2^-25 from its argument (s * (1 - s) * |x| of
            // 2^-23), 2^-24 from the sum and 2^-23 from the reciprocal: two of them by less than 2^-20.  A softmax score
            // (at most inv_total) is off by 2^-22 from expf, |x - max| * 2^-24 from the difference (times the score: less
            // than 2^-25), at most 37 * 2^-24 from summing 1024 terms and 2^-23 from the quotient: two of them by less
            // than 2^-17 * inv_total.  Adding the bias rounds once more, a key loses its low bits to its place, and a
            // group's key is a sum of two keys.
            const float apart = p.softmax ? inv_total * 0x1p-17f : 0x1p-20f;
            constexpr float kRounding = 0x1p-22f + kPer * 0x1p-23f;
            bool redo = false;     // the whole token again in 64 bits
            bool shut = false;     // this lane's experts lie in a group that is not kept
            if (p.groups > 1) {
                const bool by_score = exact_keys && p.group_top2;
                float g = kMinusInf;
                uint32_t mine;
                uint32_t lanes;    // lanes that hold the key of one group
                if (p.group_lanes != 0) {
                    // a group is p.group_lanes neighbouring lanes: its two largest from registers
                    lanes = p.group_lanes;
                    float second = kMinusInf;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const float v = by_score ? (key[i] > kMinusInf ? s[i] : kMinusInf) : key[i];
                        second = fmaxf(second, fminf(g, v));
                        g = fmaxf(g, v);
                    }
                    for (uint32_t off = 1; off < lanes; off <<= 1) {
                        const float f = __shfl_xor_sync(kAll, g, off), t = __shfl_xor_sync(kAll, second, off);
                        second = fmaxf(fminf(g, f), fmaxf(second, t));
                        g = fmaxf(g, f);
                    }
                    g = p.group_top2 && second > kMinusInf ? g + second : g;
                } else {
                    lanes = p.walk_lanes;
                    float* vals = reinterpret_cast<float*>(route_smem + warp * p.experts);
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        if (e0 + i < p.experts) {
                            vals[e0 + i] = by_score ? (key[i] > kMinusInf ? s[i] : kMinusInf) : key[i];
                        }
                    }
                    __syncwarp();
                    g = route_group_key<float>(vals, p.groups, p.per_group, lanes, lane, p.group_top2 != 0, kMinusInf);
                }
                // the best groups, one after the other; equal ones from the lowest
                mine = lane / lanes;
                uint32_t at = mine < p.groups ? route_order(g) : 0u;  // (0: no group, or taken)
                uint32_t keep = 0, low = 0;
                for (uint32_t r = 0; r < p.groups_kept; ++r) {
                    low = __reduce_max_sync(kAll, at);
                    const uint32_t h = (__ffs(__ballot_sync(kAll, at == low)) - 1) / lanes;
                    keep |= 1u << h;
                    at = mine == h ? 0u : at;
                }
                if (p.score_needed) {
                    const uint32_t high = __reduce_max_sync(kAll, at);
                    const float l = route_unorder(low), h = route_unorder(high);
                    redo = high > route_order(kMinusInf) && l - h <= 2.0f * apart + 0x1p-21f * fabsf(l);
                }
                if (p.group_lanes != 0) {
                    shut = mine >= p.groups || ((keep >> mine) & 1u) == 0;
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t of = (e0 + i) / p.per_group;
                        key[i] = of < p.groups && ((keep >> of) & 1u) != 0 ? key[i] : kMinusInf;
                    }
                }
            }
            if (!redo) {
                // Keys as ordered integers (0: cannot be chosen) with the expert's place in the low bits, lower places
                // larger.  Every lane sorts its own; the warp then takes the largest of the lanes' first keys, one after
                // the other, candidate n going to lane n.  Equal first keys: the lower lane, whose experts come first.
                uint32_t order[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    order[i] = (route_order(key[i]) & ~kLow) | (kLow - i);
                }
                if (!clean || p.groups > 1) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        order[i] = shut || !(key[i] > kMinusInf) ? 0u : order[i];
                    }
                }
                sort_descending<kPer>(order);
                uint32_t n = 0, last = 0, taken = 0, taken_from = 0;
                auto take = [&](uint32_t top) {
                    const uint32_t from = __ffs(__ballot_sync(kAll, order[0] == top)) - 1;
                    const bool owner = lane == from;
#pragma unroll
                    for (int i = 0; i + 1 < kPer; ++i) {
                        order[i] = owner ? order[i + 1] : order[i];
                    }
                    order[kPer - 1] = owner ? 0u : order[kPer - 1];
                    if (lane == n) {
                        taken = top;
                        taken_from = from;
                    }
                    last = top;
                    ++n;
                };
                // two neighbours in the order that may be the other way round
                const uint32_t unit = p.logits_type == 0 ? kPer : 0u;
                auto near = [&](uint32_t above, uint32_t here) {
                    if (exact_keys) {  // logits: only those that agree in all bits that were kept
                        return (above & ~kLow) - (here & ~kLow) <= unit;
                    }
                    const float a = route_unorder(above & ~kLow), b = route_unorder(here & ~kLow);
                    return a - b <= apart + kRounding * fabsf(a);
                };
                uint32_t top = 0;
                for (; n < p.top_k;) {
                    top = __reduce_max_sync(kAll, order[0]);
                    if (top == 0) {
                        break;
                    }
                    take(top);
                }
                filled = n;
                const uint32_t above = __shfl_up_sync(kAll, taken, 1);
                bool close = __any_sync(kAll, lane > 0 && lane < n && near(above, taken));
                while (top != 0) {  // the best that are not taken, while they may be as good as the last one taken
                    top = __reduce_max_sync(kAll, order[0]);
                    if (top == 0 || !near(last, top)) {
                        break;
                    }
                    if (n == 32) {
                        redo = true;
                        break;
                    }
                    close = true;
                    take(top);
                }
                const uint32_t candidate = taken_from * kPer + (kLow - (taken & kLow));
                my_id = lane < filled ? static_cast<int32_t>(candidate) : -1;
                redo |= close && !exact_keys && p.softmax;  // (those need the total in 64 bits)
                if (close && !redo) {
                    my_id = route_resolve(p, token, candidate, n, filled, lane);
                }
            }
            if (redo) {
                my_id = -1;
                filled = route_select_exact<kPer>(p, token, route_smem + warp * p.experts, lane, &my_id);
            }
        }
        float w = 0.0f;
        if (lane < filled) {
            const float x = route_logit(p, token, static_cast<uint32_t>(my_id));
            w = p.softmax ? route_exp_diff(x, max) * inv_total : __fdividef(1.0f, 1.0f + expf(-x));
        }
        if (p.renormalize) {
            float sum = w;  // (of the first lanes only: the others hold zeros and write nothing)
            for (uint32_t off = 1; off < p.top_k; off <<= 1) {
                sum += __shfl_xor_sync(kAll, sum, off);
            }
            w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
        }
        w *= p.scaling;
        if (lane < p.top_k) {
            const uint64_t at = static_cast<uint64_t>(token) * p.top_k + lane;
            p.ids[at] = lane < filled ? my_id : -1;
            p.weights[at] = lane < filled ? w : 0.0f;
        }
    }
}

// ---------------------------------------------------------------- many tokens: four per warp
//
// Eight lanes share a token, kPer experts each: reductions take three shuffles for four tokens at once, and the instructions
// of a token's selection, what the kernel above spends most of its time on, are shared by four.  At most 8 experts per
// token, 256 in all; groups are whole lanes, a power of two of them each.  What is in doubt is settled in place, by the
// candidates' keys in 64 bits; the rest goes to route_select_exact, a token at a time.

// a and b sorted descending: a becomes the eight largest of both, sorted; returns the largest of the others
__device__ __forceinline__ uint32_t merge_top8(uint32_t (&a)[8], const uint32_t (&b)[8])
{
    uint32_t rest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t x = a[i], y = b[7 - i];
        a[i] = x > y ? x : y;
        const uint32_t low = x > y ? y : x;
        rest = low > rest ? low : rest;
    }
#pragma unroll
    for (int k = 4; k >= 1; k >>= 1) {  // (a is bitonic now)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if ((i & k) == 0) {
                const uint32_t x = a[i], y = a[i + k];
                a[i] = x > y ? x : y;
                a[i + k] = x > y ? y : x;
            }
        }
    }
    return rest;
}

// Dynamic shared memory: kRouteWarps * experts doubles.
template <int kPer>
__global__ void __launch_bounds__(kRouteWarps * 32)
moe_route_many_kernel(const __grid_constant__ RouteParams p)
{
    extern __shared__ double route_smem[];
    static_assert(kPer == 8 || kPer == 16 || kPer == 32, "experts per lane");
    constexpr uint32_t kAll = 0xffffffffu;
    constexpr uint32_t kLow = kPer - 1;
    const float kMinusInf = -CUDART_INF_F;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sub = lane & 7u, base = lane & 24u;       // lane of the token, first lane of the token
    const uint32_t first_token = (blockIdx.x * kRouteWarps + warp) * 4;
    if (first_token >= p.tokens) {
        return;
    }
    const uint32_t token = first_token + (lane >> 3);
    const uint32_t e0 = sub * kPer;
    const bool exact_keys = p.bias == nullptr;
    const bool active = token < p.tokens && (p.token_count == nullptr ||
                                             static_cast<int64_t>(token) < static_cast<int64_t>(*p.token_count));
    float x[kPer], s[kPer], key[kPer];
    if (active) {
        route_load<kPer>(p, token, e0, x);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] = kMinusInf;
        }
    }
    bool numbers = e0 + kPer <= p.experts;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        key[i] = !exact_keys && e0 + i < p.experts ? __ldg(p.bias + e0 + i) : 0.0f;
        numbers = numbers && x[i] > kMinusInf && key[i] > kMinusInf;
    }
    const bool clean = __all_sync(kAll, numbers);
    if (!clean) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] = x[i] > kMinusInf && key[i] > kMinusInf ? x[i] : kMinusInf;
        }
    }
    float max = kMinusInf, inv_total = 1.0f;
    if (p.softmax) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            max = fmaxf(max, x[i]);
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
            max = fmaxf(max, __shfl_xor_sync(kAll, max, off));
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] = route_exp_diff(x[i], max);
            sum += s[i];
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
            sum += __shfl_xor_sync(kAll, sum, off);
        }
        inv_total = __frcp_rn(sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] *= inv_total;
        }
    } else if (p.score_needed) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s[i] = route_sigmoid_fast(x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        key[i] = exact_keys ? x[i] + 0.0f : s[i] + key[i];
    }
    if (!clean) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            key[i] = x[i] > kMinusInf ? key[i] : kMinusInf;
        }
    }
    // (the same distances as in the kernel above, which derives them)
    const float apart = p.softmax ? inv_total * 0x1p-17f : 0x1p-20f;
    constexpr float kRounding = 0x1p-22f + kPer * 0x1p-23f;
    // a lane's eight largest, sorted, and the largest of its others
    uint32_t list[8], rest = 0;
    {
        uint32_t part[kPer / 8][8];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t o = (route_order(key[i]) & ~kLow) | (kLow - i);
            part[i / 8][i % 8] = !clean && !(key[i] > kMinusInf) ? 0u : o;
        }
#pragma unroll
        for (int h = 0; h < kPer / 8; ++h) {
            sort_descending<8>(part[h]);
        }
        if constexpr (kPer == 32) {
            const uint32_t r0 = merge_top8(part[0], part[1]), r1 = merge_top8(part[2], part[3]);
            rest = merge_top8(part[0], part[2]);
            rest = rest > r0 ? rest : r0;
            rest = rest > r1 ? rest : r1;
        } else if constexpr (kPer == 16) {
            rest = merge_top8(part[0], part[1]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            list[i] = part[0][i];
        }
    }
    // a key in 64 bits (softmax scores without the common divisor)
    auto exact_key = [&](uint32_t e, bool by_score) -> double {
        const float logit = route_logit(p, token, e);
        if (exact_keys && !by_score) {
            return static_cast<double>(logit);
        }
        if (p.softmax) {
            return logit == max ? 1.0 : exp(static_cast<double>(logit) - static_cast<double>(max));
        }
        return 1.0 / (1.0 + exp(-static_cast<double>(logit))) + (exact_keys ? 0.0 : static_cast<double>(p.bias[e]));
    };
    bool redo = false;  // the whole token again in 64 bits
    if (p.groups > 1) {
        const bool by_score = exact_keys && p.group_top2;
        float g = kMinusInf, second = kMinusInf;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float v = by_score ? (key[i] > kMinusInf ? s[i] : kMinusInf) : key[i];
            second = fmaxf(second, fminf(g, v));
            g = fmaxf(g, v);
        }
        for (uint32_t off = 1; off < p.group_lanes; off <<= 1) {
            const float f = __shfl_xor_sync(kAll, g, off), u = __shfl_xor_sync(kAll, second, off);
            second = fmaxf(fminf(g, f), fmaxf(second, u));
            g = fmaxf(g, f);
        }
        g = p.group_top2 && second > kMinusInf ? g + second : g;
        const uint32_t mine = sub / p.group_lanes;
        uint32_t rank = 0;
        for (uint32_t h = 0; h < p.groups; ++h) {
            const float other = __shfl_sync(kAll, g, base + h * p.group_lanes);
            rank += (other > g || (other == g && h < mine)) ? 1u : 0u;
        }
        const bool is_group = mine < p.groups;
        bool shut = !is_group || rank >= p.groups_kept;
        if (p.score_needed) {
            float low = shut ? CUDART_INF_F : g, high = is_group && shut ? g : kMinusInf;
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) {
                low = fminf(low, __shfl_xor_sync(kAll, low, off));
                high = fmaxf(high, __shfl_xor_sync(kAll, high, off));
            }
            redo = high > kMinusInf && low - high <= 2.0f * apart + 0x1p-21f * fabsf(low);
        }
        if (__any_sync(kAll, redo)) {
            // The groups' keys of such a token in 64 bits: where a group is one lane, from the two largest of its list,
            // unless its third may belong to them.  (What cannot be settled so stays to be redone.)
            bool settled = p.group_lanes == 1 && !(p.softmax && !exact_keys);
            double g64 = -CUDART_INF;
            if (redo && settled && list[0] != 0) {
                const uint32_t e1 = e0 + (kLow - (list[0] & kLow)), e2 = e0 + (kLow - (list[1] & kLow));
                const double k1 = exact_key(e1, by_score), k2 = list[1] != 0 ? exact_key(e2, by_score) : -CUDART_INF;
                g64 = p.group_top2 && list[1] != 0 ? k1 + k2 : (k1 > k2 ? k1 : k2);
                if (list[2] != 0) {  // (the logits' own order is exact but for the bits that hold their place)
                    const float a = route_unorder(list[1] & ~kLow), b = route_unorder(list[2] & ~kLow);
                    settled = a - b > (exact_keys ? 0.0f : apart) + kRounding * fabsf(a);
                }
            }
            settled = ((__ballot_sync(kAll, settled) >> base) & 0xffu) == 0xffu;
            uint32_t rank64 = 0;
            for (uint32_t h = 0; h < p.groups; ++h) {
                const double other = __shfl_sync(kAll, g64, (base + h * p.group_lanes) & 31u);
                rank64 += (other > g64 || (other == g64 && h < mine)) ? 1u : 0u;
            }
            if (redo && settled) {
                shut = !is_group || rank64 >= p.groups_kept;
                redo = false;
            }
        }
        if (shut) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                list[i] = 0u;
            }
            rest = 0u;
        }
    }
    // One expert after the other: the largest of the lanes' first keys, of equal ones the lowest lane's; slot j in lane j.
    uint32_t filled = 0, taken = 0, taken_id = 0;
    uint32_t top = 0, from = 0;
    auto look = [&]() {  // top: the largest first key without its place (0: none left); from: its lane
        top = list[0] & ~kLow;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
            const uint32_t other = __shfl_xor_sync(kAll, top, off);
            top = other > top ? other : top;
        }
        const uint32_t at = (__ballot_sync(kAll, (list[0] & ~kLow) == top) >> base) & 0xffu;
        from = __ffs(at) - 1;  // (at least the lane of the maximum)
    };
    for (uint32_t j = 0; j < p.top_k; ++j) {
        look();
        const uint32_t value = __shfl_sync(kAll, list[0], base + from);
        if (sub == j) {
            taken = value;
            taken_id = from * kPer + (kLow - (value & kLow));
        }
        filled += top != 0 ? 1u : 0u;
        const bool owner = sub == from;
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            list[i] = owner ? list[i + 1] : list[i];
        }
        list[7] = owner ? rest : list[7];
        rest = owner ? 0u : rest;
    }
    // Two neighbours in the order, the last of them the best that is not taken, may be the other way round unless they are
    // clearly apart or the same logit with the same bias.
    look();
    const uint32_t next = __shfl_sync(kAll, list[0], base + from);
    const uint32_t next_id = from * kPer + (kLow - (next & kLow));
    uint32_t below = __shfl_down_sync(kAll, taken, 1), below_id = __shfl_down_sync(kAll, taken_id, 1);
    below = sub + 1 == p.top_k ? next : below;
    below_id = sub + 1 == p.top_k ? next_id : below_id;
    auto near = [&](uint32_t above, uint32_t here) {
        if (exact_keys) {  // logits: only those that agree in all bits that were kept; two-byte ones are then the same
            return p.logits_type == 0 && (above & ~kLow) - (here & ~kLow) <= kPer;
        }
        const float a = route_unorder(above & ~kLow), b = route_unorder(here & ~kLow);
        return a - b <= apart + kRounding * fabsf(a);
    };
    bool close = false;
    const bool last = sub + 1 == p.top_k;
    if (sub < p.top_k && sub < filled && (last ? top != 0 : sub + 1 < filled)) {
        close = near(taken, below);
    }
    const bool edge = last && close;  // the next best may belong to the taken ones, and what comes behind it too
    if (close) {
        close = route_logit(p, token, taken_id) != route_logit(p, token, below_id) ||
                (!exact_keys && p.bias[taken_id] != p.bias[below_id]);
    }
    int32_t my_id = sub < filled ? static_cast<int32_t>(taken_id) : -1;
    if (__any_sync(kAll, close || edge)) {
        // The keys of the taken ones and of the next best in 64 bits, and their order by those.  That settles a token unless
        // more than the next best are in question, or the softmax total would be needed in 64 bits.
        const uint32_t mine = (__ballot_sync(kAll, close) >> base) & 0xffu;
        const bool border = ((__ballot_sync(kAll, edge) >> base) & 0xffu) != 0;
        const bool owner = sub == from;
        const uint32_t behind = owner ? list[1] : list[0];
        bool more = behind != 0 ? near(next, behind) : kPer > 8 && owner;  // (nothing known behind the next best)
        more = ((__ballot_sync(kAll, more) >> base) & 0xffu) != 0;
        if ((border && more) || (mine != 0 && p.softmax && !exact_keys)) {
            redo = true;
        }
        double key64 = -CUDART_INF, next64 = -CUDART_INF;
        if (mine != 0 && sub < filled) {
            key64 = exact_key(taken_id, false);
        }
        if (mine != 0 && border) {
            next64 = exact_key(next_id, false);
        }
        uint32_t rank = border && (next64 > key64 || (next64 == key64 && next_id < taken_id)) ? 1u : 0u;
        uint32_t next_rank = 0;
        for (uint32_t h = 0; h < p.top_k; ++h) {
            const double other = __shfl_sync(kAll, key64, base + h);
            const uint32_t other_id = __shfl_sync(kAll, taken_id, base + h);
            if (h < filled) {
                rank += (other > key64 || (other == key64 && other_id < taken_id)) ? 1u : 0u;
                next_rank += (other > next64 || (other == next64 && other_id < next_id)) ? 1u : 0u;
            }
        }
        int32_t id = border && next_rank == sub ? static_cast<int32_t>(next_id) : -1;
        for (uint32_t h = 0; h < p.top_k; ++h) {
            const uint32_t to = __shfl_sync(kAll, rank, base + h), other_id = __shfl_sync(kAll, taken_id, base + h);
            id = h < filled && to == sub ? static_cast<int32_t>(other_id) : id;
        }
        my_id = mine != 0 && sub < filled ? id : my_id;
    }
    const uint32_t again = __ballot_sync(kAll, redo);
    if (again != 0) {
        for (uint32_t t = 0; t < 4; ++t) {
            if (((again >> (8 * t)) & 0xffu) != 0) {
                int32_t id = -1;
                const uint32_t n = route_select_exact<8>(p, first_token + t, route_smem + warp * p.experts, lane, &id);
                id = __shfl_sync(kAll, id, sub);
                if (lane >> 3 == t) {
                    my_id = id;
                    filled = n;
                }
            }
        }
    }
    float w = 0.0f;
    if (sub < filled) {
        const float logit = route_logit(p, token, static_cast<uint32_t>(my_id));
        w = p.softmax ? route_exp_diff(logit, max) * inv_total : __fdividef(1.0f, 1.0f + expf(-logit));
    }
    if (p.renormalize) {
        float sum = w;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
            sum += __shfl_xor_sync(kAll, sum, off);
        }
        w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
    }
    w *= p.scaling;
    if (sub < p.top_k && token < p.tokens) {
        const uint64_t at = static_cast<uint64_t>(token) * p.top_k + sub;
        p.ids[at] = sub < filled ? my_id : -1;
        p.weights[at] = sub < filled ? w : 0.0f;
    }
}

}  // namespace cb200
