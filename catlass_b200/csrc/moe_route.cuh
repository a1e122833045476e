// Routing of tokens to experts: scores, an optional bias, groups of experts, top-k, weights.
//
//   s[e]   = softmax_e(x) or 1 / (1 + exp(-x[e]));   key[e] = s[e] + bias[e], without a bias x[e] itself (same order)
//   a group's key is its largest key or the sum of its two largest; the experts of the best groups stay
//   ids = the top_k experts by key, ties to the lower index;  weights = s[ids] [/ their sum] * scaling
//
// One warp per token, kPer consecutive logits per lane, read once with wide loads; everything else happens in
// registers, shuffles and redux.sync.  A lane sorts its keys, the warp picks the largest of the lanes' first keys.
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

// The token's selection with 64-bit keys.  keys: shared memory of this warp, one double per expert.  Lane j receives
// the id of slot j in `id`; returns the number of slots filled.
__device__ __noinline__ uint32_t route_select_exact(const RouteParams& p, uint32_t token, double* keys, uint32_t lane,
                                                    int32_t* id)
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
    // keys[] by what decides: the groups' values first, then (the same unless groups go by score and experts by logit)
    // the experts' keys
    auto fill = [&](bool for_groups) {
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const float x = route_logit(p, token, e);
            double v = kMinusInf;
            if (x > -CUDART_INF_F) {
                v = p.bias != nullptr ? score(x) + static_cast<double>(p.bias[e])
                                      : (for_groups && p.group_top2 ? score(x) : static_cast<double>(x));
            }
            keys[e] = v > kMinusInf ? v : kMinusInf;
        }
    };
    __syncwarp();
    fill(p.groups > 1);
    if (p.groups > 1) {
        __syncwarp();
        const double g = route_group_key<double>(keys, p.groups, p.per_group, p.walk_lanes, lane, p.group_top2 != 0,
                                                 kMinusInf);
        const uint32_t keep = route_keep_groups<double>(g, p.groups, p.groups_kept, p.walk_lanes, lane);
        __syncwarp();
        if (p.bias == nullptr && p.group_top2) {
            fill(false);
        }
        for (uint32_t e = lane; e < p.experts; e += 32) {
            if (((keep >> (e / p.per_group)) & 1u) == 0) {
                keys[e] = kMinusInf;
            }
        }
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
                filled = route_select_exact(p, token, route_smem + warp * p.experts, lane, &my_id);
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

}  // namespace cb200
