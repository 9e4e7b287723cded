// The router of the layer: which experts a token goes to, with which weights, and the gradient of the logits.
//
//   softmax  s_e = exp(l_e - max) / sum exp(l - max);  the topk largest logits are picked
//   sigmoid  s_e = 1 / (1 + exp(-l_e));                the topk largest of s_e + bias_e are picked (bias: balancing, optional)
//   weights  w_k = scale * s_k, or with `renormalize` scale * s_k / sum of the picked s
// Experts whose logit is -inf or NaN are closed: s = 0, picked only when nothing else is left (then the lowest index first, weight 0),
// so that a token always has topk different experts, as the schedule wants.  Ties go to the lowest index, picks come in falling order.
//
// One warp per token; a lane holds PER of its logits in registers, so forward and backward read them once (a pick's own logit is read
// again by the lane that writes its weight: a cache hit).  A pick is a maximum over the lanes of an order-preserving 32-bit key and a
// minimum over the indices that have it.  Bound by instruction issue at long micro-batches: a pick costs about 3 PER + 20 instructions
// a warp.
#include <float.h>

#include "common.cuh"

namespace mokb {
namespace {

constexpr int kClosedKey = 1;          // below every number's key; 0: taken, or no expert

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

// This lane's logits of one row; experts beyond E and closed ones come as -inf, +inf as the largest number.
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
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = fminf(v[i] == v[i] ? v[i] : -INFINITY, FLT_MAX);
}
template <bool BF16>
__device__ __forceinline__ float clean_logit(const RouteParams& p, int64_t row, int e) {
    const float v = load_one<BF16>(p.logits, row * p.ld + e);
    return fminf(v == v ? v : -INFINITY, FLT_MAX);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// number -> key of the same order (0 and -0 alike); -inf is closed
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + expf(-l)); }

// The scores of one row, in place of its logits.  `top`: the row's largest logit (softmax).
template <int PER, bool SIGMOID>
__device__ __forceinline__ void scores(float (&v)[PER], float top, float* inv_total) {
    if (SIGMOID) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = sigmoid(v[i]);          // (-inf: 0)
        *inv_total = 1.0f;
        return;
    }
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        v[i] = v[i] == -INFINITY ? 0.0f : expf(v[i] - top);          // (a row that is closed as a whole: top is -inf too)
        total += v[i];
    }
    total = warp_sum(total);
    *inv_total = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] *= *inv_total;
}
template <bool SIGMOID>
__device__ __forceinline__ float score_of(float l, float top, float inv_total) {
    return SIGMOID ? sigmoid(l) : l == -INFINITY ? 0.0f : expf(l - top) * inv_total;
}

constexpr int route_threads(int per) { return per <= 8 ? 512 : 256; }

template <int PER, bool BF16, bool VEC, bool SIGMOID>
__global__ void __launch_bounds__(route_threads(PER)) route_kernel(const RouteParams p) {
    extern __shared__ int32_t sm[];          // balance: [E] counts, [E] sums
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
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * warps + warp; row < p.T; row += static_cast<int64_t>(gridDim.x) * warps) {
        float v[PER];
        load_row<PER, BF16, VEC>(p, row, lane, v);
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<VEC>(i, lane);
            if (SIGMOID && p.bias) {
                // Two scores a rounding apart must not change places with how exp is evaluated: in 64 bits, compared as 32-bit numbers.
                if (e < p.E) key[i] = v[i] == -INFINITY ? kClosedKey : order_key(static_cast<float>(1.0 / (1.0 + exp(-static_cast<double>(v[i]))) + static_cast<double>(p.bias[e])));
                else key[i] = 0u;
            } else {
                key[i] = e >= p.E ? 0u : v[i] == -INFINITY ? kClosedKey : order_key(v[i]);
            }
        }
        int mine = 0;                        // lane k: the k-th pick
        for (int k = 0; k < p.K; ++k) {
            uint32_t best = 0u;
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i] > best) { best = key[i]; at = i; }        // (a lane's experts ascend with i)
            const uint32_t top = __reduce_max_sync(0xffffffffu, best);
            const int e = __reduce_min_sync(0xffffffffu, best == top ? expert_of<VEC>(at, lane) : 0x7fffffff);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (expert_of<VEC>(i, lane) == e) key[i] = 0u;
            if (lane == k) mine = e;
        }
        const float l = lane < p.K ? clean_logit<BF16>(p, row, mine) : -INFINITY;
        float inv_total = 1.0f, top = 0.0f;
        if (!SIGMOID) top = __shfl_sync(0xffffffffu, l, 0);          // the first pick has the largest logit
        if (balance || (!SIGMOID && !p.renormalize)) {
            scores<PER, SIGMOID>(v, top, &inv_total);
            if (balance) {
#pragma unroll
                for (int i = 0; i < PER; ++i) acc[i] += v[i];
                if (lane < p.K && l > -INFINITY) atomicAdd(&sm[mine], 1);
            }
        }
        float s = lane < p.K ? score_of<SIGMOID>(l, top, inv_total) : 0.0f;
        if (p.renormalize) {
            const float norm = warp_sum(s);
            s = norm > 0.0f ? s / norm : 0.0f;
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

// Adds up the blocks' load figures: 32 experts per block, 32 threads each, in a fixed order.
__global__ void __launch_bounds__(1024) route_reduce_kernel(const int32_t* __restrict__ part_count, const float* __restrict__ part_sum,
                                                            int blocks, int E, int32_t* __restrict__ count, float* __restrict__ sum) {
    __shared__ int32_t c_sm[32][33];
    __shared__ float s_sm[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, e = blockIdx.x * 32 + x;
    int32_t c = 0;
    float s = 0.0f;
    if (e < E)
        for (int b = y; b < blocks; b += 32) {
            c += part_count[static_cast<int64_t>(b) * E + e];
            s += part_sum[static_cast<int64_t>(b) * E + e];
        }
    c_sm[y][x] = c;
    s_sm[y][x] = s;
    __syncthreads();
    if (y == 0 && e < E) {
        c = 0;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) { c += c_sm[i][x]; s += s_sm[i][x]; }
        count[e] = c;
        sum[e] = s;
    }
}

// d s_k from d w_k: scale * d w_k, or with `renormalize` scale * (d w_k - sum_j share_j d w_j) / norm; plus d_score_sums on every
// expert.  Then d l = s (d s - sum s d s) (softmax) or d s * s (1 - s) (sigmoid).
template <int PER, bool BF16, bool VEC, bool SIGMOID>
__global__ void __launch_bounds__(route_threads(PER)) route_bwd_kernel(const RouteParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * warps + warp; row < p.T; row += static_cast<int64_t>(gridDim.x) * warps) {
        float v[PER];
        load_row<PER, BF16, VEC>(p, row, lane, v);
        int mine = -1;
        float dw = 0.0f, l = -INFINITY;
        if (lane < p.K) {
            const int64_t e = p.picked[row * p.K + lane];
            if (e >= 0 && e < p.E) {                       // anything else has no logit
                mine = static_cast<int>(e);
                dw = p.d_weights[row * p.K + lane] * p.scale;
                l = clean_logit<BF16>(p, row, mine);
            }
        }
        float top = 0.0f, inv_total;
        if (!SIGMOID) {
            top = v[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
            top = warp_max(top);
        }
        scores<PER, SIGMOID>(v, top, &inv_total);
        const float s = score_of<SIGMOID>(l, top, inv_total);
        float d = dw;
        if (p.renormalize) {
            const float norm = warp_sum(s), inv = norm > 0.0f ? 1.0f / norm : 0.0f;
            d = (dw - warp_sum(s * inv * dw)) * inv;
        }
        if (mine < 0) d = 0.0f;
        float ds[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<VEC>(i, lane);
            ds[i] = p.d_score_sums && e < p.E ? __ldg(p.d_score_sums + e) : 0.0f;
        }
        for (int k = 0; k < p.K; ++k) {
            const int e = __shfl_sync(0xffffffffu, mine, k);
            const float dk = __shfl_sync(0xffffffffu, d, k);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (expert_of<VEC>(i, lane) == e) ds[i] += dk;
        }
        if (SIGMOID) {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = ds[i] * v[i] * (1.0f - v[i]);
        } else {
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) dot += v[i] * ds[i];
            dot = warp_sum(dot);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] *= ds[i] - dot;
        }
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
    const int warps = route_threads((E + 31) / 32) / 32;
    const int64_t blocks = (T + warps - 1) / warps, most = 2LL * sm_count();
    return static_cast<int>(blocks < most ? blocks : most);
}

template <int PER, bool BF16, bool VEC, bool SIGMOID>
int launch_route(const RouteParams& p, bool backward, cudaStream_t stream) {
    const int blocks = route_blocks(p.T, PER * 32);
    if (backward) route_bwd_kernel<PER, BF16, VEC, SIGMOID><<<blocks, route_threads(PER), 0, stream>>>(p);
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
        route_reduce_kernel<<<(num_experts + 31) / 32, 1024, 0, stream>>>(p.part_count, p.part_sum, blocks, num_experts, tokens_per_expert, score_sums);
        MOKB_CUDA(cudaGetLastError());
        note_launch();
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
