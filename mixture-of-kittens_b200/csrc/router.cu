// The router of the layer: which experts a token goes to, with which weights, and the gradient of the logits.
//
//   softmax  s_e = exp(l_e - max) / sum exp(l - max);  the topk largest logits are picked
//   sigmoid  s_e = 1 / (1 + exp(-l_e));                the topk largest of s_e + bias_e are picked (bias: balancing, optional)
//   weights  w_k = scale * s_k, or with `renormalize` scale * s_k / sum of the picked s
// Experts whose logit is -inf or NaN are closed: s = 0, picked only when nothing else is left (then the lowest index first, weight 0),
// so that a token always has topk different experts, as the schedule wants.  Ties go to the lowest index, picks come in falling order.
//
// One warp per token; a lane holds PER of its logits in registers, so forward and backward read them once (a pick's own logit is read
// again by the lane that writes its weight: a cache hit).  The next token's row is on its way while one is worked on.
//
// Picking: a key is a 32-bit number of the logits' order whose low bits give way to the expert's index (inverted: the lowest index is the
// largest key), so that one maximum over the warp is a pick, and no two keys are alike.  Every lane keeps its two largest; only a lane that
// has given both looks for its next two.  For bf16 logits nothing is lost by that.  For fp32 ones the order of two that agree in all other
// bits is open: where that happens between neighbours in the order of the picks (the first that is left out among them), the row is done
// again by key and index.  With a bias the keys are s + bias, and two of them a rounding apart must not change places with how exp is
// evaluated: the order is that of the sums worked out in 64 bits and rounded to 32.  They too are first picked by such keys; then the picks'
// own sums in 32 bits, and the most that the next key can stand for, say whether that was the order, and the row is done again in 64 where
// neighbours are nearer than the error of that.  (Asking the keys themselves, short of seven bits and more, sends 6 % of the rows there at
// 128 experts: 28 us where this took 26; at 512 experts 57 where it took 39.)
// (16384 x 256, 8 picks: 28 us looking through all keys for every pick, 19 with keys and indices apart.)
//
// Bound by instructions at long micro-batches: of a row of 256 logits 690 warp instructions in the forward pass with the load figures and 420 in
// the backward pass, of 128 with a bias 680 and 320; 63 to 76 % of the cycles issue, memory is at a tenth to a third of its rate.  Graph replays back
// to back: 16384 x 256 in fp32, softmax, 8 picks: 11.5 us forward, 17.8 with the load figures, 6.3 backward, 9.6 with score sums; 32768 x 128 with a
// bias: 23.4, 30.0, 10.6 and 13.0; 16384 x 512 with a bias: 36.5, 45.8, 9.3 and 13.2.  The logits alone take 2.6 to 5.1 us.
#include <float.h>

#include "common.cuh"

namespace mokb {
namespace {

struct RouteParams {
    const void* logits;
    int64_t ld, T;
    int E, K, renormalize;
    float scale;
    const float* bias;
    int64_t* top_experts;
    float* weights;
    // load figures: a row per block, [blocks, E]
    int32_t* part_count;
    float* part_sum;
    // backward
    const int64_t* picked;
    const float* d_weights;
    const float* d_score_sums;
    void* d_logits;
};

template <bool VEC> __device__ __forceinline__ int expert_of(int i, int lane) { return VEC ? (i >> 2) * 128 + lane * 4 + (i & 3) : i * 32 + lane; }

template <bool BF16> __device__ __forceinline__ float load_one(const void* p, int64_t i) {
    return BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// This lane's part of a row in shared memory.
template <int PER, bool VEC>
__device__ __forceinline__ void load_shared(const float* row, int lane, float (&v)[PER]) {
    if (VEC) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const float4 w = *reinterpret_cast<const float4*>(row + expert_of<VEC>(i, lane));
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = row[expert_of<VEC>(i, lane)];
    }
}

// This lane's logits of one row as they are; -inf beyond E.
template <int PER, bool BF16, bool VEC>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t row, int lane, float (&v)[PER]) {
    const int64_t base = row * p.ld;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = -INFINITY;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const int e = expert_of<VEC>(i, lane);
            if (e >= p.E) continue;
            if (BF16) {
                const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.logits) + base + e);
                const float2 a = unpack_bf16(w.x), b = unpack_bf16(w.y);
                v[i] = a.x; v[i + 1] = a.y; v[i + 2] = b.x; v[i + 3] = b.y;
            } else {
                const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + base + e);
                v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<VEC>(i, lane);
            if (e < p.E) v[i] = load_one<BF16>(p.logits, base + e);
        }
    }
}
// NaN closes an expert like -inf; +inf counts as the largest number
__device__ __forceinline__ float clean(float v) { return fminf(v == v ? v : -INFINITY, FLT_MAX); }
template <bool BF16>
__device__ __forceinline__ float load_clean(const RouteParams& p, int64_t row, int e) { return clean(load_one<BF16>(p.logits, row * p.ld + e)); }

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// number -> key of the same order (0 and -0 alike), and back
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

constexpr uint32_t kClosedKey = 0x007fffffu;          // order_key(-inf)
// Scores that leave the kernel come from expf: an approximate exp's error grows with its argument (58 half-steps of fp32 for a softmax logit 80
// below the largest).  Quotients that make a weight are IEEE ones.  The denominator of a sigmoid, 1 + exp(-|l|), is between 1 and 2: its
// reciprocal is the IEEE one for the picks, and for all of a row's experts (load figures and the gradient of the score sums, where dozens
// of roundings follow) the approximate one, off by two units in the last place at most.  With the IEEE one there too: 30.8 instead of
// 30.0 us (32768 x 128, bias, figures) and 48.7 instead of 45.8 (16384 x 512), backward with score sums 14.2 and 17.0 instead of 13.0 and 13.2.
template <bool MANY>
__device__ __forceinline__ float reciprocal(float d) { return MANY ? __fdividef(1.0f, d) : __frcp_rn(d); }
template <bool MANY>
__device__ __forceinline__ float sigmoid(float l) {      // (-inf: 0)
    const float small = expf(-fabsf(l));
    return (l >= 0.0f ? 1.0f : small) * reciprocal<MANY>(1.0f + small);
}
// s (1 - s): of s near 1 the difference from 1 would be what rounding has left of it.
template <bool MANY>
__device__ __forceinline__ float sigmoid_slope(float l) {      // (-inf: 0)
    const float small = expf(-fabsf(l)), q = reciprocal<MANY>(1.0f + small);
    return small * q * q;
}
// For the order of the picks alone, which is settled by better sums wherever this could decide it.
__device__ __forceinline__ float sigmoid_for_order(float l) { return __fdividef(1.0f, 1.0f + __expf(-l)); }

// exp(l - top) of a row's logits, in place, and their sum (SIGMOID: the scores themselves).  Closed ones give 0; a row that is closed as a
// whole has top = -inf.
template <int PER, bool SIGMOID>
__device__ __forceinline__ float exponentials(float (&v)[PER], float top) {
    if (SIGMOID) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = sigmoid<true>(v[i]);
        return 1.0f;
    }
    float total = 0.0f;
    const float at = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        v[i] = expf(v[i] - at);
        total += v[i];
    }
    return warp_sum(total);
}
template <bool SIGMOID>
__device__ __forceinline__ float score_of(float l, float top, float total) {
    return SIGMOID ? sigmoid<false>(l) : l == -INFINITY ? 0.0f : expf(l - top) / total;      // (a logit that is open has a total of 1 or more)
}

// The picks' shares of the sum of their scores (lane k: the k-th pick, l = -inf in the others and for closed ones) come from scores relative to
// the largest pick's: exp(l - max), with sigmoid scores exp(l - c) / (1 + exp(l)) and c = min(max, 0).  So a row whose scores are all tiny still
// has shares, and their sum is 1/2 or more.  A row whose largest pick lies below -745, where sigmoid is 0 in 64 bits too, has none.
template <bool SIGMOID>
__device__ __forceinline__ float relative_score(float l, float max_l) {
    if (!SIGMOID) return l == -INFINITY ? 0.0f : expf(l - max_l);
    const float small = expf(-fabsf(l));
    float r = l >= 0.0f ? 1.0f : small;
    if (max_l < 0.0f) r = max_l < -745.0f ? 0.0f : expf(l - max_l);      // (the same in every lane: max_l is the row's)
    return r * __frcp_rn(1.0f + small);
}
__device__ __forceinline__ float warp_max(float v) { return key_value(__reduce_max_sync(0xffffffffu, order_key(v))); }

constexpr int index_bits(int per) { return per == 4 ? 7 : per == 8 ? 8 : per == 16 ? 9 : 10; }

// The topk largest keys, indices in their low bits, in falling order: lane k has the k-th one in *mine.  NEXT: *next is the one that follows.
template <int PER, bool NEXT>
__device__ __forceinline__ void pick(const uint32_t (&key)[PER], int K, int lane, uint32_t* mine, uint32_t* next) {
    uint32_t b1 = 0u, b2 = 0u, last = 0u;         // b1, b2: this lane's two largest that are not taken
    int cached = 2;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        b2 = max(b2, min(b1, key[i]));
        b1 = max(b1, key[i]);
    }
    *mine = 0u;
    const int rounds = NEXT ? K + 1 : K;
    for (int k = 0; k < rounds; ++k) {
        last = __reduce_max_sync(0xffffffffu, b1);
        if (lane == k) *mine = last;
        if (b1 == last) {
            b1 = b2;
            if (--cached == 0) {
                b1 = b2 = 0u;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const uint32_t below = key[i] < last ? key[i] : 0u;
                    b2 = max(b2, min(b1, below));
                    b1 = max(b1, below);
                }
                cached = 2;
            }
        }
    }
    *next = last;
}
// The same by key and index, for rows whose order that leaves open.
template <int PER, bool VEC>
__device__ __forceinline__ int pick_by_key_and_index(uint32_t (&key)[PER], int K, int lane) {
    int mine = 0;
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
        uint32_t best = 0u;
        int at = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > best) { best = key[i]; at = i; }            // (a lane's experts ascend with i)
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const int e = __reduce_min_sync(0xffffffffu, best == top ? expert_of<VEC>(at, lane) : 0x7fffffff);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (expert_of<VEC>(i, lane) == e) key[i] = 0u;
        if (lane == k) mine = e;
    }
    return mine;
}

constexpr int route_threads(int per) { return per <= 8 ? 256 : 128; }
constexpr int route_blocks_per_sm(int per) { return per <= 4 ? 5 : per <= 8 ? 4 : per <= 16 ? 5 : 3; }

template <int PER, bool BF16, bool VEC, bool SIGMOID>
__global__ void __launch_bounds__(route_threads(PER), route_blocks_per_sm(PER)) route_kernel(const RouteParams p) {
    extern __shared__ int32_t sm[];          // balance: [E] counts, [E] sums
    grid_dep_launch();                       // (the blocks that add up the load figures come in as these leave)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const bool balance = p.part_count != nullptr;
    float* const sums = reinterpret_cast<float*>(sm + p.E);
    float acc[PER];
    if (balance) {
        for (int e = threadIdx.x; e < 2 * p.E; e += blockDim.x) sm[e] = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
        __syncthreads();
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
    int64_t row = static_cast<int64_t>(blockIdx.x) * warps + warp;
    float next[PER];
    if (row < p.T) load_row<PER, BF16, VEC>(p, row, lane, next);
    for (; row < p.T; row += step) {
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = clean(next[i]);
        if (row + step < p.T) load_row<PER, BF16, VEC>(p, row + step, lane, next);
        constexpr uint32_t kIndex = (1u << index_bits(PER)) - 1u;
        uint32_t key[PER];                   // 0: no expert
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<VEC>(i, lane);
            float order = v[i];
            if (SIGMOID && p.bias && order > -INFINITY && e < p.E) order = clean(sigmoid_for_order(order) + __ldg(p.bias + e));      // (a NaN's key could be none)
            key[i] = e >= p.E ? 0u : (order_key(order) & ~kIndex) | (kIndex - static_cast<uint32_t>(e));
        }
        constexpr bool kExact = BF16 && !SIGMOID;      // (a bf16 logit's key loses nothing to the index)
        uint32_t mine_key, next_key;
        pick<PER, !kExact>(key, p.K, lane, &mine_key, &next_key);
        int mine = static_cast<int>(kIndex - (mine_key & kIndex));      // lane k: the k-th pick
        float l = lane < p.K ? load_clean<BF16>(p, row, mine) : -INFINITY;
        if (SIGMOID && p.bias) {
            // The picks' sums as they are, and the largest that one which is left out can be.  s of a key: an exp (off by some 2 + 1.2 |l|
            // units in the last place; s (1 - s) <= 1/4 and |l| s (1 - s) < 0.23 of that), a sum and a quotient: below 3e-7.  s + bias and the
            // 32-bit form of the exact sum are rounded once each.  Neighbours that are more than 1e-6 (1 + |s + bias|) apart are in order.
            const float hi = l > -INFINITY ? clean(sigmoid<false>(l) + __ldg(p.bias + mine)) : -INFINITY;
            float lo = __shfl_down_sync(0xffffffffu, hi, 1);
            if (lane == p.K - 1) lo = (next_key | kIndex) > kClosedKey ? key_value(next_key | kIndex) : -INFINITY;
            const bool unsettled = lane < p.K && lo > -INFINITY && !(hi - lo > 1e-6f + 1e-6f * fmaxf(fabsf(hi), fabsf(lo)));
            if (__any_sync(0xffffffffu, unsettled)) {
#pragma unroll 1
                for (int i = 0; i < PER; ++i) {
                    const int e = expert_of<VEC>(i, lane);
                    uint32_t exact = 0u;
                    if (e < p.E) {
                        const double x = load_clean<BF16>(p, row, e);
                        exact = x == -INFINITY ? kClosedKey : order_key(clean(static_cast<float>(1.0 / (1.0 + exp(-x)) + static_cast<double>(p.bias[e]))));
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        if (j == i) key[j] = exact;
                }
                mine = pick_by_key_and_index<PER, VEC>(key, p.K, lane);
                l = lane < p.K ? load_clean<BF16>(p, row, mine) : -INFINITY;
            }
        } else if (!BF16) {
            uint32_t below = __shfl_down_sync(0xffffffffu, mine_key, 1);
            if (lane == p.K - 1) below = next_key;
            // keys that differ only in the index (closed experts are in order by that)
            if (__any_sync(0xffffffffu, lane < p.K && (below | kIndex) > kClosedKey && (mine_key | kIndex) == (below | kIndex))) {
#pragma unroll
                for (int i = 0; i < PER; ++i) key[i] = expert_of<VEC>(i, lane) < p.E ? order_key(v[i]) : 0u;
                mine = pick_by_key_and_index<PER, VEC>(key, p.K, lane);
                l = lane < p.K ? load_clean<BF16>(p, row, mine) : -INFINITY;
            }
        }
        float total = 1.0f, top = 0.0f;
        if (!SIGMOID) top = __shfl_sync(0xffffffffu, l, 0);          // the first pick has the largest logit
        if (balance || (!SIGMOID && !p.renormalize)) {
            total = exponentials<PER, SIGMOID>(v, top);
            if (balance) {
                const float inv_total = SIGMOID ? 1.0f : total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i) acc[i] += SIGMOID ? v[i] : v[i] * inv_total;
                if (lane < p.K && l > -INFINITY) atomicAdd(&sm[mine], 1);
            }
        }
        float s;
        if (p.renormalize) {          // (the first pick's logit is the largest unless a bias has picked)
            s = relative_score<SIGMOID>(l, SIGMOID && p.bias ? warp_max(l) : __shfl_sync(0xffffffffu, l, 0));
            const float norm = warp_sum(s);
            s = norm > 0.0f ? s / norm : 0.0f;          // (0: no pick is open)
        } else {
            s = score_of<SIGMOID>(l, top, total);
        }
        if (lane < p.K) {
            p.top_experts[row * p.K + lane] = mine;
            p.weights[row * p.K + lane] = s * p.scale;
        }
    }
    if (!balance) return;
    // the warps' sums one after the other: the same result every time
    for (int w = 0; w < warps; ++w) {
        __syncthreads();
        if (warp == w) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = expert_of<VEC>(i, lane);
                if (e < p.E) sums[e] += acc[i];
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        p.part_count[static_cast<int64_t>(blockIdx.x) * p.E + e] = sm[e];
        p.part_sum[static_cast<int64_t>(blockIdx.x) * p.E + e] = sums[e];
    }
}

// Adds up the blocks' load figures in a fixed order: 8 experts per block, 128 threads each.
__global__ void __launch_bounds__(1024) route_reduce_kernel(const int32_t* part_count, const float* part_sum, int blocks, int E, int32_t* count, float* sum) {
    __shared__ int32_t c_sm[32][9];
    __shared__ float s_sm[32][9];
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3, e = blockIdx.x * 8 + x;
    int32_t c = 0;
    float s = 0.0f;
    grid_dep_wait();
    if (e < E) {
#pragma unroll 8
        for (int b = y; b < blocks; b += 128) {
            c += __ldcg(part_count + static_cast<int64_t>(b) * E + e);
            s += __ldcg(part_sum + static_cast<int64_t>(b) * E + e);
        }
    }
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {          // the four rows of a warp
        c += __shfl_xor_sync(0xffffffffu, c, o);
        s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if ((threadIdx.x & 31) < 8) {
        c_sm[threadIdx.x >> 5][x] = c;
        s_sm[threadIdx.x >> 5][x] = s;
    }
    __syncthreads();
    if (threadIdx.x < 8 && e < E) {
        c = 0;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) { c += c_sm[i][x]; s += s_sm[i][x]; }
        count[e] = c;
        sum[e] = s;
    }
}

// The gradient of the logits has two parts.  The picks' own, worked out by the lane of a pick and handed through shared memory (a row of zeros
// per warp between tokens) to the lane that holds its logit:
//   renormalised   share_k (dw_k - sum_j share_j dw_j), with sigmoid scores times 1 - s_k    (dw: d_router_weights times scale)
//   softmax        s_k dw_k                   sigmoid   s_k (1 - s_k) dw_k
// and that of the scores: s_e (ds_e - dot) (softmax) or s_e (1 - s_e) ds_e (sigmoid) with ds = d_score_sums, which lies in shared memory once
// per block, and dot = sum s ds (+ sum s_k dw_k where the weights are scores).  Without either the row's scores are not needed.
template <int PER, bool BF16, bool VEC, bool SIGMOID>
__global__ void __launch_bounds__(route_threads(PER), route_blocks_per_sm(PER)) route_bwd_kernel(const RouteParams p) {
    extern __shared__ __align__(16) float rows_sm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float* const part_sm = rows_sm + warp * PER * 32;
    float* const sums_sm = rows_sm + warps * PER * 32;
    uint8_t* const tag_sm = reinterpret_cast<uint8_t*>(sums_sm + PER * 32) + warp * PER * 32;      // who wrote an expert's number last
#pragma unroll
    for (int i = 0; i < PER; ++i) part_sm[expert_of<VEC>(i, lane)] = 0.0f;
    const bool with_sums = p.d_score_sums != nullptr, with_scores = with_sums || (!SIGMOID && !p.renormalize);
    for (int e = threadIdx.x; e < PER * 32; e += blockDim.x) sums_sm[e] = with_sums && e < p.E ? __ldg(p.d_score_sums + e) : 0.0f;
    __syncthreads();
    const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
    int64_t row = static_cast<int64_t>(blockIdx.x) * warps + warp;
    float next[PER];
    int64_t next_pick = -1;
    float next_dw = 0.0f;
    auto fetch = [&](int64_t r) {
        load_row<PER, BF16, VEC>(p, r, lane, next);
        if (lane < p.K) {
            next_pick = p.picked[r * p.K + lane];
            next_dw = p.d_weights[r * p.K + lane];
        }
    };
    if (row < p.T) fetch(row);
    for (; row < p.T; row += step) {
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = clean(next[i]);
        const int mine = next_pick >= 0 && next_pick < p.E ? static_cast<int>(next_pick) : -1;      // anything else has no logit
        const float l = mine >= 0 ? load_clean<BF16>(p, row, mine) : -INFINITY;
        const float dw = l > -INFINITY ? next_dw * p.scale : 0.0f;          // (a closed pick's weight is 0 for good)
        if (row + step < p.T) fetch(row + step);
        float top = 0.0f, total = 1.0f, dot = 0.0f;
        if (with_scores) {          // v: what d_score_sums is multiplied by, the scores or the sigmoid's slope
            if (SIGMOID) {
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] = sigmoid_slope<true>(v[i]);
            } else {
                top = v[0];
#pragma unroll
                for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
                top = warp_max(top);
                total = exponentials<PER, false>(v, top);
                const float inv_total = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] *= inv_total;
            }
        }
        float part;
        if (p.renormalize) {
            const float r = relative_score<SIGMOID>(l, warp_max(l));
            float norm = r, mean = r * dw;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                norm += __shfl_xor_sync(0xffffffffu, norm, o);
                mean += __shfl_xor_sync(0xffffffffu, mean, o);
            }
            const float inv = norm > 0.0f ? 1.0f / norm : 0.0f;          // (norm is 1/2 or more where a pick is open)
            part = r * inv * (dw - mean * inv);
            if (SIGMOID) part *= sigmoid<false>(-l);          // 1 - s
        } else {
            part = (SIGMOID ? sigmoid_slope<false>(l) : score_of<false>(l, top, total)) * dw;
            if (!SIGMOID) dot = part;                // (added up below, with the scores' own)
        }
        if (mine >= 0) tag_sm[mine] = static_cast<uint8_t>(lane);
        __syncwarp();
        if (mine >= 0) part_sm[mine] = part;
        if (__any_sync(0xffffffffu, mine >= 0 && tag_sm[mine] != lane)) {
            // a caller's list that names an expert twice: one after the other, in the list's order
            if (mine >= 0) part_sm[mine] = 0.0f;
            __syncwarp();
            for (int k = 0; k < p.K; ++k) {
                if (lane == k && mine >= 0) part_sm[mine] += part;
                __syncwarp();
            }
        }
        __syncwarp();
        if (with_scores) {
            float ds[PER];
            load_shared<PER, VEC>(sums_sm, lane, ds);
            if (SIGMOID) {
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] *= ds[i];
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) dot += v[i] * ds[i];
                dot = warp_sum(dot);
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] *= ds[i] - dot;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = 0.0f;
        }
        float own[PER];
        load_shared<PER, VEC>(part_sm, lane, own);
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] += own[i];
        __syncwarp();
        if (mine >= 0) part_sm[mine] = 0.0f;
        __syncwarp();
        const int64_t base = row * p.E;
        if (VEC) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                const int e = expert_of<VEC>(i, lane);
                if (e >= p.E) continue;
                if (BF16) *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.d_logits) + base + e) = make_uint2(pack_bf16(v[i], v[i + 1]), pack_bf16(v[i + 2], v[i + 3]));
                else *reinterpret_cast<float4*>(static_cast<float*>(p.d_logits) + base + e) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = expert_of<VEC>(i, lane);
                if (e >= p.E) continue;
                if (BF16) static_cast<__nv_bfloat16*>(p.d_logits)[base + e] = __float2bfloat16_rn(v[i]);
                else static_cast<float*>(p.d_logits)[base + e] = v[i];
            }
        }
    }
}

int route_blocks(int64_t T, int E) {
    const int per = (E + 31) / 32, warps = route_threads(per) / 32;
    const int64_t blocks = (T + warps - 1) / warps, most = static_cast<int64_t>(route_blocks_per_sm(per)) * sm_count();
    return static_cast<int>(blocks < most ? blocks : most);
}

template <int PER, bool BF16, bool VEC, bool SIGMOID>
int launch_route(const RouteParams& p, bool backward, cudaStream_t stream) {
    const int blocks = route_blocks(p.T, PER * 32);
    if (backward)      // a row of numbers and tags per warp, d_score_sums once
        route_bwd_kernel<PER, BF16, VEC, SIGMOID><<<blocks, route_threads(PER), (route_threads(PER) * 5 + 128) * PER, stream>>>(p);
    else route_kernel<PER, BF16, VEC, SIGMOID><<<blocks, route_threads(PER), p.part_count ? 8u * p.E : 0u, stream>>>(p);
    MOKB_CUDA(cudaGetLastError());
    note_launch();
    return MOKB_OK;
}
template <int PER>
int launch_route(const RouteParams& p, bool bf16, bool sigmoid, bool backward, cudaStream_t stream) {
    const uintptr_t align = bf16 ? 7 : 15;
    const bool vec = p.E % 4 == 0 && p.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p.logits) & align) == 0 &&
                     (reinterpret_cast<uintptr_t>(p.d_logits) & align) == 0;
    if (vec) {
        if (bf16) return sigmoid ? launch_route<PER, true, true, true>(p, backward, stream) : launch_route<PER, true, true, false>(p, backward, stream);
        return sigmoid ? launch_route<PER, false, true, true>(p, backward, stream) : launch_route<PER, false, true, false>(p, backward, stream);
    }
    if (bf16) return sigmoid ? launch_route<PER, true, false, true>(p, backward, stream) : launch_route<PER, true, false, false>(p, backward, stream);
    return sigmoid ? launch_route<PER, false, false, true>(p, backward, stream) : launch_route<PER, false, false, false>(p, backward, stream);
}
// logits of a lane, a power of two from 4 (128 experts) on
int lane_logits(int E) {
    int per = 4;
    while (per * 32 < E) per *= 2;
    return per;
}
int launch_route(const RouteParams& p, bool bf16, bool sigmoid, bool backward, cudaStream_t stream) {
    switch (lane_logits(p.E)) {
    case 4: return launch_route<4>(p, bf16, sigmoid, backward, stream);
    case 8: return launch_route<8>(p, bf16, sigmoid, backward, stream);
    case 16: return launch_route<16>(p, bf16, sigmoid, backward, stream);
    default: return launch_route<32>(p, bf16, sigmoid, backward, stream);
    }
}

int check_route(const void* logits, int64_t ld, int64_t T, int E, int K, int score, float scale) {
    MOKB_REQUIRE(T >= 0 && E >= 1 && E <= MOKB_ROUTE_MAX_EXPERTS, "route: num_experts must be in [1, %d]", MOKB_ROUTE_MAX_EXPERTS);
    MOKB_REQUIRE(K >= 1 && K <= MOKB_ROUTE_MAX_TOPK && K <= E, "route: topk must be in [1, min(num_experts, %d)]", MOKB_ROUTE_MAX_TOPK);
    MOKB_REQUIRE(ld >= E, "route: the row stride of the logits is less than a row");
    MOKB_REQUIRE(score == MOKB_SCORE_SOFTMAX || score == MOKB_SCORE_SIGMOID, "route: unknown score function %d", score);
    MOKB_REQUIRE(scale == scale, "route: scale is not a number");
    MOKB_REQUIRE(T == 0 || logits, "route: null pointer");
    return MOKB_OK;
}

}  // namespace
}  // namespace mokb

using namespace mokb;

extern "C" size_t mokb_route_scratch_bytes(int64_t num_tokens, int num_experts) {
    if (num_tokens < 0 || num_experts < 1 || num_experts > MOKB_ROUTE_MAX_EXPERTS) return 0;
    const size_t rows = route_blocks(num_tokens, lane_logits(num_experts) * 32);
    return rows * num_experts * 8 + 8;
}

extern "C" int mokb_route(const void* logits, int bf16, int64_t row_stride, int64_t num_tokens, int num_experts, int topk, int score,
                          const float* bias, int renormalize, float scale, int64_t* top_experts, float* router_weights,
                          int32_t* tokens_per_expert, float* score_sums, void* scratch, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    TraceScope trace(stream, "route");
    MOKB_TRY(check_route(logits, row_stride, num_tokens, num_experts, topk, score, scale));
    MOKB_REQUIRE(num_tokens == 0 || (top_experts && router_weights), "route: null pointer");
    MOKB_REQUIRE((tokens_per_expert == nullptr) == (score_sums == nullptr), "route: tokens_per_expert and score_sums go together");
    MOKB_REQUIRE(tokens_per_expert == nullptr || scratch, "route: the load figures need scratch");
    MOKB_REQUIRE(bias == nullptr || score == MOKB_SCORE_SIGMOID, "route: a bias goes with sigmoid scores");
    RouteParams p = {};
    p.logits = logits; p.ld = row_stride; p.T = num_tokens; p.E = num_experts; p.K = topk; p.renormalize = renormalize; p.scale = scale;
    p.bias = bias; p.top_experts = top_experts; p.weights = router_weights;
    const int blocks = route_blocks(num_tokens, lane_logits(num_experts) * 32);
    if (tokens_per_expert) {
        p.part_count = static_cast<int32_t*>(scratch);
        p.part_sum = reinterpret_cast<float*>(p.part_count + static_cast<size_t>(blocks) * num_experts);
    }
    if (num_tokens > 0) MOKB_TRY(launch_route(p, bf16 != 0, score == MOKB_SCORE_SIGMOID, false, stream));
    if (tokens_per_expert) {
        MOKB_TRY(launch_after(route_reduce_kernel, static_cast<unsigned>((num_experts + 7) / 8), 1024u, 0, stream, static_cast<const int32_t*>(p.part_count),
                              static_cast<const float*>(p.part_sum), blocks, num_experts, tokens_per_expert, score_sums));
    }
    return MOKB_OK;
}

extern "C" int mokb_route_bwd(const void* logits, int bf16, int64_t row_stride, int64_t num_tokens, int num_experts, int topk, int score,
                              int renormalize, float scale, const int64_t* top_experts, const float* d_router_weights,
                              const float* d_score_sums, void* d_logits, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    TraceScope trace(stream, "route_bwd");
    MOKB_TRY(check_route(logits, row_stride, num_tokens, num_experts, topk, score, scale));
    MOKB_REQUIRE(num_tokens == 0 || (top_experts && d_router_weights && d_logits), "route_bwd: null pointer");
    if (num_tokens == 0) return MOKB_OK;
    RouteParams p = {};
    p.logits = logits; p.ld = row_stride; p.T = num_tokens; p.E = num_experts; p.K = topk; p.renormalize = renormalize; p.scale = scale;
    p.picked = top_experts; p.d_weights = d_router_weights; p.d_score_sums = d_score_sums; p.d_logits = d_logits;
    return launch_route(p, bf16 != 0, score == MOKB_SCORE_SIGMOID, true, stream);
}
