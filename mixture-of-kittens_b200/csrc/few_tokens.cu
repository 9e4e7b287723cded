// The whole layer for a few tokens (1 to MOKB_FEW_MAX_TOKENS): what a decoding step needs, where mokb_schedule pads every expert to 256
// rows and the grouped GEMMs multiply 256-row tiles that hold one or two real rows.
//
//   y[t] = shared(x[t]) + sum_k w[t, k] * expert_{e(t, k)}(x[t]),   expert(v) = W_down (silu(W_gate v) * (W_up v))
//
// Bound by the weights: every expert that has a token is read once, 6 H I bytes in bf16 (3.1 H I in MXFP8), for 6 H I multiply-adds a
// token: below some 250 tokens an expert the tensor cores wait for memory.  So the operands change roles against gemm.cu: the WEIGHTS
// are the 128-row side of tcgen05.mma (A, streamed by TMA) and the tokens of an expert its narrow side (N = 16 .. 128), and what is
// tuned is how evenly the stream of weights is spread over the SMs.
//
// Four launches, tied by programmatic dependent launch (a kernel's set-up, and the down projection's first weights, go ahead of the
// end of the kernel before it):
//   plan   one block: the tokens of every local expert, in `units` of at most 128 columns; clears the counters.  MXFP8: further blocks
//          quantise x (E4M3 + E8M0 along the hidden axis, what the layer's pull does).
//   gate/up  tile = 128 gate rows and the 128 up rows beside them (two accumulators, so a thread holds both): hidden = silu(g) * u
//   down     tile = 256 rows of W_down; fp32 results, one row per route
//   sum      y[t] = shared + sum over k = 0, 1, .. of w[t, k] * result, rounded once
// Work is cut by stages of the contraction, not by tiles: the stages of all tiles are numbered through and every CTA takes an equal,
// contiguous range (7 experts of 1408 x 5120 are 77 gate/up tiles on 148 SMs).  A tile that falls to several CTAs is summed by the one
// that finishes last, in the order of the contraction, from fp32 partial sums in global memory: nobody waits, so calls on several
// streams cannot block each other, and the result does not depend on who was last.  (Summing the routes of a token the same way, by
// whoever counts its last one, put a fence and four dependent round trips to a busy memory into every tile: down 260 us instead of 135
// for 24 tokens through 64 experts of 5120 x 1408.  So that is a launch of its own.)
//
// Graph replays back to back, weights from memory (6546 GB/s: a plain copy's rate here): one token through 8 of 32 experts of 7168 x 2048
// and the shared one 138 us (5.7 TB/s), 24 tokens through 64 of 5120 x 1408 389 us (6.5 TB/s), 48 tokens on one of two ranks' 64 experts of
// 4096 x 1536 in MXFP8 196 us (5.9 TB/s), 200 tokens through all of the first 528 us (5.5 TB/s), two tokens of the smallest layer (8 of
// 1024 x 512) 24 us.  One token: 5 us until the first weights arrive (plan, header, unit, memory), 3 us between the products (the last
// tiles' sums), the SMs end 8 us apart, 5 us for the sum and its launch.  Two tokens of the small layer are a chain of such latencies.
// What bounds a stage where memory does not: eight MMAs take about 45 clocks each whatever N is, of the 1300 that its 32 KB take to arrive.
// Three stages in the ring instead of six cost 4 %; units of 64 columns instead of 128 nothing up to 200 tokens, 45 % at 511 (their experts'
// weights are then read twice).
//
// hidden is rounded to bf16 (MXFP8: E4M3) between the products: both operands of a tcgen05 product have the weights' type, and the layer's own
// forward keeps it so.  Against 64 bits y is then off by 0.0023 of itself (root mean square) where a product of unrounded hidden would leave y's
// own rounding, 0.0017; hidden as two bf16 parts would be nearer, for twice the narrow operand.
//
//   warp 0     TMA producer: weights (two 128-row boxes of 128 bytes per stage) and, MXFP8, their scale tiles
//   warp 1     MMA issuer
//   warps 2-9  epilogue
//   warps 10-  the tokens' rows: gathered with 16-byte cp.async into the swizzled layout; the copies themselves arrive on the stage's
//              barrier, so as many stages are under way as the ring holds, and the MMA issuer makes them visible to the tensor cores
#include "common.cuh"
#include "mxfp8_codec.cuh"

namespace mokb {
namespace {

constexpr int kEpilogueWarps = 8;               // two per quarter of tensor memory
constexpr int kLoaderWarps = 4;
constexpr int kThreads = 32 * (2 + kEpilogueWarps + kLoaderWarps);
constexpr int A_BYTES = 2 * 128 * 128;          // two boxes of 128 rows x 128 bytes
constexpr int SF_BYTES = 3 * 512;               // MXFP8: the scale tiles of both boxes and of the tokens
constexpr int kMaxStages = 8;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kCtrlBytes = 512 + kLoaderWarps * 512;      // barriers, flags; a row list per loader warp
// No CTA takes fewer stages than this: below it, what a tile's partial sums cost is more than a stage's load.  (Two tokens, 8 experts of
// 1024 x 512: 24.3 us; with 2 stages 28, with 6 25.1, with 8 23.6, with 16 28.2.)
constexpr int kMinStages = 4;
// plan: threads, fewer for few routes; routes that a thread keeps in registers; routes whose experts are kept in shared memory
constexpr int kPlanThreads = 1024, kPlanThreadsSmall = 256, kKept = 4, kPlanIds = 8192;

// columns of a unit: two accumulators, double buffered, fill the 512 columns of tensor memory; MXFP8 keeps 32 of them for the scales
__host__ __device__ constexpr int unit_columns(bool mx) { return mx ? 112 : 128; }

// An expert's routes are cut into units of equal size; the tiles of its units alternate (rows first, then units), so that a second
// unit finds the weights in L2.
struct Unit {
    int expert;       // -1: the shared expert
    int n;            // columns (tokens)
    int slot0;        // first slot; shared: first token
    int place;        // number among the expert's units << 16 | how many those are
};

// The call's work area.
struct Work {
    int32_t* header;          // [0] units, [1] of them shared
    Unit* units;
    int32_t* slot_token;      // [T * K] token of a slot; slots are numbered expert by expert
    int32_t* pos;             // [T * K] slot of a route, -1: not of this rank, or without weight
    int32_t* counters;        // [2][SMs] tickets of the tiles that several CTAs share
    uint8_t* xq;              // MXFP8: [T, H] E4M3
    uint32_t* xs;             // MXFP8: [T, H / 128] four scale bytes each
    uint8_t* hid_q;           // MXFP8: [T * K, I]
    uint8_t* hid_s;           // MXFP8: [T * K, I / 128] four scale bytes each
    __nv_bfloat16* hid;       // [T * K + T, I]; row T * K + t: the shared expert's (MXFP8: only those are used)
    float* yr;                // [T * K + T, H] results before they are summed
    float* part;              // [SMs][2][2][columns][128] partial sums of split tiles
};

inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }
inline int column_cap(int T, bool mx) {      // (16 for an empty step too, whose work area is asked for like any other's)
    const int n = T > 0 ? (T + 15) / 16 * 16 : 16;
    return n < unit_columns(mx) ? n : unit_columns(mx);
}
inline int max_units(int T, int K, bool mx) { return T * K + T / column_cap(T, mx) + 2; }      // a routed unit has a route; shared ones

inline size_t carve_few(Work* w, void* base, int T, int H, int I, int K, bool mx, int sms) {
    char* const p0 = static_cast<char*>(base);
    char* p = p0;
    auto take = [&](size_t bytes) { char* q = p; p += align256(bytes); return q; };
    const size_t R = static_cast<size_t>(T) * K;
    Work v;
    v.header = reinterpret_cast<int32_t*>(take(64));
    v.units = reinterpret_cast<Unit*>(take(sizeof(Unit) * max_units(T, K, mx)));
    v.slot_token = reinterpret_cast<int32_t*>(take(R * 4));
    v.pos = reinterpret_cast<int32_t*>(take(R * 4));
    v.counters = reinterpret_cast<int32_t*>(take(static_cast<size_t>(sms) * 8));
    v.xq = reinterpret_cast<uint8_t*>(take(mx ? static_cast<size_t>(T) * H : 0));
    v.xs = reinterpret_cast<uint32_t*>(take(mx ? static_cast<size_t>(T) * (H / 128) * 4 : 0));
    v.hid_q = reinterpret_cast<uint8_t*>(take(mx ? R * I : 0));
    v.hid_s = reinterpret_cast<uint8_t*>(take(mx ? R * (I / 128) * 4 : 0));
    v.hid = reinterpret_cast<__nv_bfloat16*>(take((R + T) * I * 2));
    v.yr = reinterpret_cast<float*>(take((R + T) * static_cast<size_t>(H) * 4));
    v.part = reinterpret_cast<float*>(take(static_cast<size_t>(sms) * 4 * column_cap(T, mx) * 128 * 4));
    if (w) *w = v;
    return static_cast<size_t>(p - p0);
}

struct FewParams {
    int T, H, I, E, K, first_expert;
    int mx, shared, has_limit;
    float limit;
    int stages, col_cap, sms;          // ring stages, columns the ring has room for, CTAs of the two big launches
    const __nv_bfloat16* x;
    const int64_t* top_experts;
    const float* weights;
    __nv_bfloat16* y;
    int32_t* status;
    Work w;
};

struct FewMaps {                       // by-value kernel argument: the two boxes of a stage, and (MXFP8) their scale tiles
    CUtensorMap routed0, routed1, shared0, shared1, scale0, scale1;
};

__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory"); }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// arrives on the barrier (one of its expected arrivals) once this thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// 32 lanes x 16 consecutive fp32 columns of tensor memory
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, float (&f)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]);
}

// ---------------------------------------------------------------------------------------------------------------- plan
// Exclusive block-wide prefix sum of two counts per thread.
__device__ __forceinline__ int2 block_scan(int2 v, int2* total) {
    __shared__ int2 warp_sum[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, inc.x, o), b = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (lane >= o) { inc.x += a; inc.y += b; }
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int2 s = lane < warps ? warp_sum[lane] : make_int2(0, 0);       // every warp scans the sums for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
        if (lane >= o) { s.x += a; s.y += b; }
    }
    *total = make_int2(__shfl_sync(0xffffffffu, s.x, 31), __shfl_sync(0xffffffffu, s.y, 31));
    const int bx = __shfl_sync(0xffffffffu, s.x, max(warp - 1, 0)), by = __shfl_sync(0xffffffffu, s.y, max(warp - 1, 0));
    __syncthreads();
    return make_int2((warp ? bx : 0) + inc.x - v.x, (warp ? by : 0) + inc.y - v.y);
}

// Block 0 lays out the routes; with MXFP8 weights blocks 1.. quantise x, a warp per 1024 values of a row at a time.
// The order of an expert's tokens is that of the atomics where it has one unit: it decides which column a token gets, not what is computed
// for it.  Of several units, which one a token is in does (they are cut between CTAs at different places), so those are dealt out in order.
__global__ void __launch_bounds__(kPlanThreads) few_plan_kernel(const FewParams p) {
    grid_dep_launch();
    const int t0 = threadIdx.x;
    if (blockIdx.x > 0) {
        const int lane = t0 & 31, per_row = (p.H + 1023) / 1024;
        const int warps = blockDim.x >> 5, pieces = p.T * per_row, stride = (gridDim.x - 1) * warps;
        for (int i = (blockIdx.x - 1) * warps + (t0 >> 5); i < pieces; i += stride) {
            const int t = i / per_row, c0 = (i - t * per_row) * 1024 + lane * 32;      // a lane: one block of 32 values
            if (c0 >= p.H) continue;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.x + static_cast<size_t>(t) * p.H + c0);
            uint32_t w[16], m = 0u;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + q);
                w[4 * q] = v.x; w[4 * q + 1] = v.y; w[4 * q + 2] = v.z; w[4 * q + 3] = v.w;
            }
#pragma unroll
            for (int q = 0; q < 16; ++q) m = absmax2(m, w[q]);
            float inv;
            const uint32_t byte = scale_byte(fmaxf(bf16_lo(m), bf16_hi(m)), &inv);
            uint32_t o[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                o[q] = e4m3x4(bf16_lo(w[2 * q]) * inv, bf16_hi(w[2 * q]) * inv, bf16_lo(w[2 * q + 1]) * inv, bf16_hi(w[2 * q + 1]) * inv);
            st_global_32B(p.w.xq + static_cast<size_t>(t) * p.H + c0, o);
            reinterpret_cast<uint8_t*>(p.w.xs)[static_cast<size_t>(t) * (p.H / 32) + c0 / 32] = static_cast<uint8_t>(byte);
        }
        return;
    }
    extern __shared__ int32_t count[];           // [E] routes, then the experts' first slots; behind them the first kPlanIds routes' experts
    uint16_t* const ids = reinterpret_cast<uint16_t*>(count + p.E);
    const int NT = p.col_cap, R = p.T * p.K, n_threads = blockDim.x;      // (an expert named twice by a token can have more routes than there are tokens)
    // a thread keeps its first kKept routes in registers between the two passes; further ones leave their number in `pos`
    int expert[kKept], number[kKept];
    auto expert_of = [&](int j) {                // -1: not of this rank, or without weight (a weight that is NaN counts)
        const int64_t e = p.top_experts[j] - p.first_expert;
        return e >= 0 && e < p.E && p.weights[j] != 0.0f ? static_cast<int>(e) : -1;
    };
#pragma unroll
    for (int i = 0; i < kKept; ++i) expert[i] = t0 + i * n_threads < R ? expert_of(t0 + i * n_threads) : -1;
#pragma unroll
    for (int i = 0; i < kKept; ++i)
        if (t0 + i * n_threads < R) ids[t0 + i * n_threads] = static_cast<uint16_t>(expert[i]);      // (-1: no expert has that number)
    for (int i = t0; i < p.E; i += n_threads) count[i] = 0;
    for (int i = t0; i < 2 * p.sms; i += n_threads) p.w.counters[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i) number[i] = expert[i] >= 0 ? atomicAdd(&count[expert[i]], 1) : 0;
    for (int j = t0 + kKept * n_threads; j < R; j += n_threads) {
        const int e = expert_of(j);
        if (j < kPlanIds) ids[j] = static_cast<uint16_t>(e);
        p.w.pos[j] = e >= 0 ? atomicAdd(&count[e], 1) : -1;
    }
    __syncthreads();
    bool cut = false;
    for (int i = t0; i < p.E; i += n_threads) cut = cut || count[i] > NT;
    if (__syncthreads_or(cut)) {
        // a warp per such expert goes through the routes in order
        const int lane = t0 & 31;
        for (int e = t0 >> 5; e < p.E; e += n_threads >> 5) {
            if (count[e] <= NT) continue;
            int before = 0;
            for (int j0 = lane; j0 - lane < R; j0 += 128) {
                bool its[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 32 * i;
                    its[i] = j < R && (j < kPlanIds ? ids[j] == e : expert_of(j) == e);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned all = __ballot_sync(0xffffffffu, its[i]);
                    if (its[i]) p.w.pos[j0 + 32 * i] = before + __popc(all & ((1u << lane) - 1u));
                    before += __popc(all);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (expert[i] >= 0 && count[expert[i]] > NT) number[i] = p.w.pos[t0 + i * n_threads];
    }
    int2 carry = make_int2(0, 0);                // slots, units
    for (int e0 = 0; e0 < p.E; e0 += n_threads) {
        const int e = e0 + t0;
        const int n = e < p.E ? count[e] : 0;
        int2 total;
        const int cuts = (n + NT - 1) / NT;
        int2 at = block_scan(make_int2(n, cuts), &total);
        at.x += carry.x;
        at.y += carry.y;
        if (e < p.E) count[e] = at.x;
        for (int c = 0; c < cuts; ++c) {
            const int lo = static_cast<int>(static_cast<int64_t>(c) * n / cuts), hi = static_cast<int>(static_cast<int64_t>(c + 1) * n / cuts);
            p.w.units[at.y + c] = Unit{e, hi - lo, at.x + lo, c << 16 | cuts};
        }
        carry.x += total.x;
        carry.y += total.y;
    }
    const int shared_units = p.shared ? (p.T + NT - 1) / NT : 0;      // the last ones
    if (t0 < shared_units) {
        const int lo = t0 * p.T / shared_units, hi = (t0 + 1) * p.T / shared_units;
        p.w.units[carry.y + t0] = Unit{-1, hi - lo, lo, t0 << 16 | shared_units};
    }
    if (t0 == 0) {
        p.w.header[0] = carry.y + shared_units;
        p.w.header[1] = shared_units;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
        const int j = t0 + i * n_threads;
        if (j >= R) break;
        const int slot = expert[i] >= 0 ? count[expert[i]] + number[i] : -1;
        p.w.pos[j] = slot;
        if (slot >= 0) p.w.slot_token[slot] = j / p.K;
    }
    for (int j = t0 + kKept * n_threads; j < R; j += n_threads) {
        const int n = p.w.pos[j];
        if (n < 0) continue;
        const int slot = count[p.top_experts[j] - p.first_expert] + n;
        p.w.pos[j] = slot;
        p.w.slot_token[slot] = j / p.K;
    }
}

// ---------------------------------------------------------------------------------------------------------------- the two products
// The stages of all tiles in order, and this CTA's share of them.
struct Stream {
    int blocks;                   // tiles of a unit
    int ks_shared, ks_routed;     // stages of a tile
    int tiles_routed;             // they come first
    int64_t routed_stages, total;
    int ctas;                     // that take part
    __device__ Stream(const FewParams& p, int units, int shared_units, bool down) {
        const int contraction = down ? p.I : p.H;
        blocks = down ? p.H / 256 : p.I / 128;
        ks_shared = contraction / 64;
        ks_routed = p.mx ? contraction / 128 : contraction / 64;
        tiles_routed = (units - shared_units) * blocks;
        routed_stages = static_cast<int64_t>(tiles_routed) * ks_routed;
        total = routed_stages + static_cast<int64_t>(shared_units) * blocks * ks_shared;
        const int64_t most = total / kMinStages;
        ctas = most < 1 ? 1 : most < p.sms ? static_cast<int>(most) : p.sms;
    }
    __device__ int64_t begin(int64_t c) const { return c * total / ctas; }
    __device__ int owner(int64_t stage) const { return static_cast<int>(((stage + 1) * ctas - 1) / total); }
};
struct Segment {
    int tile, k0, k1, ks;         // stages [k0, k1) of the tile's ks
    int64_t first;                // the tile's first stage
};
__device__ __forceinline__ Segment segment_at(const Stream& st, int64_t s, int64_t end) {
    Segment g;
    if (s < st.routed_stages) {
        g.ks = st.ks_routed;
        g.tile = static_cast<int>(s / g.ks);
        g.first = static_cast<int64_t>(g.tile) * g.ks;
    } else {
        g.ks = st.ks_shared;
        const int64_t r = (s - st.routed_stages) / g.ks;
        g.tile = st.tiles_routed + static_cast<int>(r);
        g.first = st.routed_stages + r * g.ks;
    }
    g.k0 = static_cast<int>(s - g.first);
    const int64_t left = end - g.first;
    g.k1 = left < g.ks ? static_cast<int>(left) : g.ks;
    return g;
}
// The unit of a tile and the tile's number among the unit's row blocks.
__device__ __forceinline__ Unit unit_of(const FewParams& p, int tile, int blocks, int* blk) {
    const int4* const units = reinterpret_cast<const int4*>(p.w.units);
    int u = tile / blocks;
    int4 v = __ldcg(units + u);
    *blk = tile - u * blocks;
    const int cuts = v.w & 0xffff;
    if (cuts > 1) {
        u -= v.w >> 16;                                   // the expert's first unit
        const int in = tile - u * blocks;
        *blk = in / cuts;
        v = __ldcg(units + u + (in - *blk * cuts));
    }
    return Unit{v.x, v.y, v.z, v.w};
}

template <bool DOWN>
__global__ void __launch_bounds__(kThreads, 1) few_product_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const int S = p.stages;
    const uint32_t b_bytes = static_cast<uint32_t>(p.col_cap) * 128u;
    const uint32_t data_bytes = A_BYTES + b_bytes;
    const uint32_t sf_base = smem_base + S * data_bytes;
    const uint32_t ctrl_off = S * (data_bytes + (p.mx ? SF_BYTES : 0));
    const uint32_t bars = smem_base + ctrl_off;
    // control block: full[8] | empty[8] | tmem_full[2] | tmem_empty[2] | tmem pointer, abort, flag | row lists of the loader warps
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * kMaxStages + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * kMaxStages + 2 + a); };
    uint8_t* const ctrl = smem_gen + ctrl_off;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl + 8 * (2 * kMaxStages + 4));
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (2 * kMaxStages + 4) + 4);
    volatile int* const vote = reinterpret_cast<volatile int*>(ctrl + 8 * (2 * kMaxStages + 4) + 8);      // [2], used in turn

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1 + 32);                 // the weights' bytes, and an arrival per lane of the stage's loader warp
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), kEpilogueWarps);
        }
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&maps.routed0);
        tma_prefetch_desc(&maps.routed1);
        if (p.shared) { tma_prefetch_desc(&maps.shared0); tma_prefetch_desc(&maps.shared1); }
        if (p.mx) { tma_prefetch_desc(&maps.scale0); tma_prefetch_desc(&maps.scale1); }
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (!DOWN) grid_dep_wait();       // the plan
    grid_dep_launch();
    // DOWN: the gate/up kernel let this one start after it had seen the plan finished, so the plan may be read at once (through L2, past
    // lines that an earlier call may have left in L1); only what that kernel itself writes has to be waited for.
    const int n_units = __ldcg(p.w.header), n_shared = __ldcg(p.w.header + 1);
    const Stream st(p, n_units, n_shared, DOWN);
    const int cta = blockIdx.x;
    const int64_t s_begin = cta < st.ctas ? st.begin(cta) : 0, s_end = cta < st.ctas ? st.begin(cta + 1) : 0;
    // a stage of the routed experts: 64 columns of bf16 or 128 of E4M3; both are 128 bytes
    const int acc_cols = unit_columns(p.mx != 0);
    const uint32_t sf_cols0 = tmem_base + 4 * unit_columns(true);

    if (warp == 0) {
        // ------------------------------------------------------------ weights
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            const int rows = DOWN ? p.H : p.I, kt = (DOWN ? p.I : p.H) / 128;
            for (int64_t at = s_begin; ok && at < s_end;) {
                const Segment g = segment_at(st, at, s_end);
                at += g.k1 - g.k0;
                int blk;
                const int expert = unit_of(p, g.tile, st.blocks, &blk).expert;
                const bool sh = expert < 0, mx = p.mx && !sh;
                const CUtensorMap* const m0 = sh ? &maps.shared0 : &maps.routed0;
                const CUtensorMap* const m1 = sh ? &maps.shared1 : &maps.routed1;
                const int r0 = (sh ? 0 : expert * rows) + blk * (DOWN ? 256 : 128), r1 = DOWN ? r0 + 128 : r0;
                const int step = mx ? 128 : 64;
                for (int k = g.k0; k < g.k1; ++k) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, MOKB_ST_PIPELINE_TIMEOUT)) { ok = false; break; }
                    const uint32_t fb = full_bar(s), dst = smem_base + s * data_bytes;
                    mbar_expect_tx(fb, A_BYTES + (mx ? 1024 : 0));
                    tma_load_2d(dst, m0, fb, k * step, r0);
                    tma_load_2d(dst + A_BYTES / 2, m1, fb, k * step, r1);
                    if (mx) {
                        const uint32_t sf = sf_base + s * SF_BYTES;
                        tma_load_2d(sf, &maps.scale0, fb, 0, (r0 >> 7) * kt + k);
                        tma_load_2d(sf + 512, &maps.scale1, fb, 0, (r1 >> 7) * kt + k);
                    }
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            int s = 0, local = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int64_t at = s_begin; ok && at < s_end; ++local) {
                const Segment g = segment_at(st, at, s_end);
                at += g.k1 - g.k0;
                int blk;
                const Unit unit = unit_of(p, g.tile, st.blocks, &blk);
                const bool mx = p.mx && unit.expert >= 0;
                const uint32_t npad = static_cast<uint32_t>((unit.n + 15) & ~15);
                const int buf = local & 1;
                if (!mbar_wait(tempty_bar(buf), ((local >> 1) & 1u) ^ 1u, abort_flag, p.status, MOKB_ST_PIPELINE_TIMEOUT)) break;
                tc_fence_after();
                const uint32_t d0 = tmem_base + buf * 2 * acc_cols, d1 = d0 + acc_cols;
                // fp32 accumulators, M = 128, N = npad; bf16 x bf16, or E4M3 x E4M3 with E8M0 scales
                const uint32_t idesc = (npad >> 3) << 17 | (128u >> 4) << 24 | (mx ? 1u << 23 : 1u << 4 | 1u << 7 | 1u << 10);
                for (int k = g.k0; k < g.k1; ++k) {
                    if (!mbar_wait(full_bar(s), ph, abort_flag, p.status, MOKB_ST_PIPELINE_TIMEOUT)) { ok = false; break; }
                    fence_proxy_async_smem();          // the tokens' rows came through the generic proxy
                    tc_fence_after();
                    const uint32_t a = smem_base + s * data_bytes;
                    const uint64_t a0 = make_smem_desc(a, 16, 1024), a1 = make_smem_desc(a + A_BYTES / 2, 16, 1024);
                    const uint64_t b = make_smem_desc(a + A_BYTES, 16, 1024);
                    if (mx) {
                        const uint32_t sf = sf_base + s * SF_BYTES, cols = sf_cols0 + (s & 1) * 16;
                        tmem_cp_32x128b_warpx4(cols, make_smem_desc_plain16(sf));
                        tmem_cp_32x128b_warpx4(cols + 4, make_smem_desc_plain16(sf + 512));
                        tmem_cp_32x128b_warpx4(cols + 8, make_smem_desc_plain16(sf + 1024));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t id = idesc | static_cast<uint32_t>(i) << 4 | static_cast<uint32_t>(i) << 29;
                            umma_mxf8(d0, a0 + 2 * i, b + 2 * i, id, cols, cols + 8, (k > g.k0 || i) ? 1u : 0u);
                            umma_mxf8(d1, a1 + 2 * i, b + 2 * i, id, cols + 4, cols + 8, (k > g.k0 || i) ? 1u : 0u);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            umma_bf16(d0, a0 + 2 * i, b + 2 * i, idesc, (k > g.k0 || i) ? 1u : 0u);
                            umma_bf16(d1, a1 + 2 * i, b + 2 * i, idesc, (k > g.k0 || i) ? 1u : 0u);
                        }
                    }
                    umma_commit(empty_bar(s));
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (ok) umma_commit(tfull_bar(buf));
            }
        }
    } else if (warp >= 2 + kEpilogueWarps) {
        // ------------------------------------------------------------ the tokens' rows
        // Every fourth stage is this warp's as a whole.
        const int lw = warp - 2 - kEpilogueWarps, chunk = lane & 7, sub = lane >> 3;      // a lane: 16 bytes of one row of four
        int32_t* const rows = reinterpret_cast<int32_t*>(ctrl + 512 + lw * 512);      // [128]: the row that column n is read from
        int s = 0, turn = 0;
        uint32_t ph = 0;
        bool ok = true, waited = !DOWN;
        for (int64_t at = s_begin; ok && at < s_end;) {
            const Segment g = segment_at(st, at, s_end);
            at += g.k1 - g.k0;
            int blk;
            const Unit unit = unit_of(p, g.tile, st.blocks, &blk);
            const bool sh = unit.expert < 0, mx = p.mx && !sh;
            __syncwarp();
            for (int n = lane; n < unit.n; n += 32)
                rows[n] = DOWN ? unit.slot0 + n + (sh ? p.T * p.K : 0) : sh ? unit.slot0 + n : __ldcg(p.w.slot_token + unit.slot0 + n);
            __syncwarp();
            const int64_t row_bytes = (DOWN ? p.I : p.H) * (mx ? 1 : 2);
            const uint8_t* const src = (DOWN ? (mx ? p.w.hid_q : reinterpret_cast<const uint8_t*>(p.w.hid))
                                             : (mx ? p.w.xq : reinterpret_cast<const uint8_t*>(p.x))) + chunk * 16;
            const uint32_t* const scales = DOWN ? reinterpret_cast<const uint32_t*>(p.w.hid_s) : p.w.xs;
            const int kt = (DOWN ? p.I : p.H) / 128;
            if (!waited) {
                grid_dep_wait();              // hidden
                waited = true;
            }
            for (int k = g.k0; k < g.k1; ++k) {
                if (turn == lw) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, MOKB_ST_PIPELINE_TIMEOUT)) { ok = false; break; }
                    const uint32_t dst = smem_base + s * data_bytes + A_BYTES;
                    const uint8_t* const from = src + k * 128;
#pragma unroll 4
                    for (int n = sub; n < unit.n; n += 4)
                        cp_async_16(dst + n * 128u + static_cast<uint32_t>((chunk ^ (n & 7)) << 4), from + rows[n] * row_bytes);
                    if (mx) {
                        const uint32_t sf = sf_base + s * SF_BYTES + 1024;
                        for (int n = lane; n < unit.n; n += 32)
                            cp_async_4(sf + static_cast<uint32_t>((n & 31) * 16 + (n >> 5) * 4), scales + static_cast<int64_t>(rows[n]) * kt + k);
                    }
                    cp_async_arrive(full_bar(s));
                }
                if (++turn == kLoaderWarps) turn = 0;
                if (++s == S) { s = 0; ph ^= 1u; }
            }
        }
        cp_async_wait_all();
    } else {
        // ------------------------------------------------------------ epilogue
        // A warp: 32 rows (the quarter of tensor memory that it may read) and every other 16 columns.
        const int quarter = warp & 3, row = quarter * 32 + lane, first_col = ((warp - 2) >> 2) * 16, et = threadIdx.x - 64;
        const float limit = p.has_limit ? p.limit : __int_as_float(0x7f800000);
        const size_t part_stride = static_cast<size_t>(p.col_cap) * 128;      // one accumulator's partial sums
        // slot 1: the tile begins in CTA q (and ends in a later one); slot 0: it began in an earlier one
        auto part_of = [&](int q, int c_lo) { return p.w.part + (static_cast<size_t>(q) * 2 + (q == c_lo ? 1 : 0)) * 2 * part_stride + row; };
        if (DOWN) grid_dep_wait();      // (no CTA ends before the gate/up kernel has: what follows may overwrite the work area)
        int local = 0, votes = 0;
        for (int64_t at = s_begin; at < s_end; ++local) {
            const Segment g = segment_at(st, at, s_end);
            at += g.k1 - g.k0;
            int blk;
            const Unit unit = unit_of(p, g.tile, st.blocks, &blk);
            const bool sh = unit.expert < 0;
            const int buf = local & 1;
            // Is everybody else through with the tile?  Asked ahead of this CTA's own end: mostly it comes last (the next CTA began with
            // the tile's other part), and then its sums never leave tensor memory.
            const int c_lo = g.k0 == 0 && g.k1 == g.ks ? cta : st.owner(g.first), c_hi = c_lo == cta && g.k1 == g.ks ? cta : st.owner(g.first + g.ks - 1);
            int32_t* const ticket = p.w.counters + (DOWN ? p.sms : 0) + c_lo;
            // (a wait that ran out has set the status word, so what follows is void, but the barriers below need all eight warps)
            mbar_wait(tfull_bar(buf), (local >> 1) & 1u, abort_flag, p.status, MOKB_ST_PIPELINE_TIMEOUT);
            tc_fence_after();
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * 2 * acc_cols, t1 = t0 + acc_cols;
            bool mine_in_tmem = true;
            if (c_lo != c_hi) {
                // (a word of `vote` is written again only after a later barrier than the one before it was read)
                if (et == 0) vote[votes & 1] = ld_acquire_gpu(ticket) == c_hi - c_lo ? 1 : 0;
                epilogue_sync();
                if (!vote[votes++ & 1]) {
                    mine_in_tmem = false;
                    float* const mine = part_of(cta, c_lo);
                    for (int c = first_col; c < unit.n; c += 32) {
                        float a[16], b[16];
                        tmem_ld_32x16(t0 + c, a);
                        tmem_ld_32x16(t1 + c, b);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c + j < unit.n) {
                                mine[(c + j) * 128] = a[j];
                                mine[part_stride + (c + j) * 128] = b[j];
                            }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar(buf));
                    __threadfence();
                    epilogue_sync();
                    if (et == 0) vote[votes & 1] = atomicAdd(ticket, 1) == c_hi - c_lo ? 1 : 0;
                    epilogue_sync();
                    if (!vote[votes++ & 1]) continue;
                }
                __threadfence();
            }
            for (int c = first_col; c < unit.n; c += 32) {
                float a[16], b[16];
                if (c_lo == c_hi) {
                    tmem_ld_32x16(t0 + c, a);
                    tmem_ld_32x16(t1 + c, b);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) a[j] = b[j] = 0.0f;
                    for (int q = c_lo; q <= c_hi; ++q) {      // in the order of the contraction, whoever is last
                        float x[16], y[16];
                        if (q == cta && mine_in_tmem) {
                            tmem_ld_32x16(t0 + c, x);
                            tmem_ld_32x16(t1 + c, y);
                        } else {
                            const float* const theirs = part_of(q, c_lo);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                x[j] = c + j < unit.n ? __ldcg(theirs + (c + j) * 128) : 0.0f;
                                y[j] = c + j < unit.n ? __ldcg(theirs + part_stride + (c + j) * 128) : 0.0f;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            a[j] += x[j];
                            b[j] += y[j];
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (c + j >= unit.n) break;               // (the same in every lane)
                    const int64_t r = unit.slot0 + c + j;
                    if (DOWN) {
                        float* const dst = p.w.yr + (r + (sh ? p.T * p.K : 0)) * p.H + blk * 256 + row;
                        dst[0] = a[j];
                        dst[128] = b[j];
                    } else {
                        const float gate = fminf(a[j], limit), up = fminf(fmaxf(b[j], -limit), limit);
                        // the approximate reciprocal of a quarter of the denominator: of all of it, it would be zero for gates near -88
                        float h = __fdividef(0.25f * gate, fmaf(0.25f, __expf(-gate), 0.25f)) * up;
                        if (a[j] != a[j] || b[j] != b[j]) h = a[j] + b[j];      // (the clamps drop a NaN)
                        if (p.mx && !sh) {
                            // the warp's 32 rows are one block of the hidden axis
                            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu);
                            float inv;
                            const uint32_t byte = scale_byte(__uint_as_float(top), &inv);
                            uint16_t pair;
                            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(pair) : "f"(h * inv));
                            p.w.hid_q[r * p.I + blk * 128 + row] = static_cast<uint8_t>(pair);
                            if (lane == 0) p.w.hid_s[(r * (p.I / 128) + blk) * 4 + quarter] = static_cast<uint8_t>(byte);
                        } else {
                            p.w.hid[(r + (sh ? p.T * p.K : 0)) * p.I + blk * 128 + row] = __float2bfloat16_rn(h);
                        }
                    }
                }
            }
            if (mine_in_tmem) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(buf));
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: give copies still in flight time to land before the CTA's shared memory is released
        const unsigned long long c0 = clock64();
        while (clock64() - c0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------------------------------------------- sum
// A warp per 256 columns of a token: the shared expert's result, then the routes in order, eight at a time in flight.
// (The plan was complete before the down projection could start, so the routes' slots are read ahead of the wait.)
__global__ void __launch_bounds__(128) few_sum_kernel(const FewParams p) {
    const int lane = threadIdx.x & 31, blocks = p.H / 256;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
    const bool live = item < p.T * blocks;
    const int t = live ? item / blocks : 0, col = (item - t * blocks) * 256 + lane * 8;
    auto slot_of = [&](int k) { return k < p.K ? __ldcg(p.w.pos + t * p.K + k) : -1; };
    auto weight_of = [&](int k) { return k < p.K ? __ldg(p.weights + t * p.K + k) : 0.0f; };
    int mine = slot_of(lane);
    float weight = weight_of(lane);
    grid_dep_wait();
    if (!live) return;
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
    if (p.shared) {
        const float4* const v = reinterpret_cast<const float4*>(p.w.yr + static_cast<int64_t>(p.T * p.K + t) * p.H + col);
        const float4 a = __ldcg(v), b = __ldcg(v + 1);
        sum[0] = a.x; sum[1] = a.y; sum[2] = a.z; sum[3] = a.w; sum[4] = b.x; sum[5] = b.y; sum[6] = b.z; sum[7] = b.w;
    }
    for (int k0 = 0; k0 < p.K; k0 += 32) {
        if (k0 > 0) {
            mine = slot_of(k0 + lane);
            weight = weight_of(k0 + lane);
        }
        unsigned todo = __ballot_sync(0xffffffffu, mine >= 0);
        while (todo) {
            float4 a[8], b[8];
            float w[8];
            int n = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = 0.0f;
                if (todo) {
                    const int k = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const float4* const v = reinterpret_cast<const float4*>(p.w.yr + static_cast<int64_t>(__shfl_sync(0xffffffffu, mine, k)) * p.H + col);
                    w[i] = __shfl_sync(0xffffffffu, weight, k);
                    a[i] = __ldcg(v);
                    b[i] = __ldcg(v + 1);
                    ++n;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= n) break;
                sum[0] += w[i] * a[i].x; sum[1] += w[i] * a[i].y; sum[2] += w[i] * a[i].z; sum[3] += w[i] * a[i].w;
                sum[4] += w[i] * b[i].x; sum[5] += w[i] * b[i].y; sum[6] += w[i] * b[i].z; sum[7] += w[i] * b[i].w;
            }
        }
    }
    *reinterpret_cast<uint4*>(p.y + static_cast<size_t>(t) * p.H + col) =
        make_uint4(pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3]), pack_bf16(sum[4], sum[5]), pack_bf16(sum[6], sum[7]));
}

// once per device: the attribute belongs to the device's context
int allow_shared_memory() {
    static bool done[64] = {false};
    int dev = -1;
    MOKB_CUDA(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && __atomic_load_n(&done[dev], __ATOMIC_RELAXED)) return MOKB_OK;
    MOKB_CUDA(cudaFuncSetAttribute(few_product_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
    MOKB_CUDA(cudaFuncSetAttribute(few_product_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
    if (dev >= 0 && dev < 64) __atomic_store_n(&done[dev], true, __ATOMIC_RELAXED);
    return MOKB_OK;
}

int check_few_sizes(int T, int H, int I, int K) {
    MOKB_REQUIRE(T >= 0 && T <= MOKB_FEW_MAX_TOKENS, "few_tokens: num_tokens must be in [0, %d]", MOKB_FEW_MAX_TOKENS);
    MOKB_REQUIRE(H > 0 && H % 256 == 0 && H <= 65536, "few_tokens: hidden must be a positive multiple of 256, at most 65536");
    MOKB_REQUIRE(I > 0 && I % 128 == 0 && I <= 65536, "few_tokens: intermediate must be a positive multiple of 128, at most 65536");
    MOKB_REQUIRE(K >= 1 && K <= 255, "few_tokens: topk must be in [1, 255]");
    return MOKB_OK;
}

}  // namespace
}  // namespace mokb

using namespace mokb;

extern "C" size_t mokb_few_tokens_args_size(void) { return sizeof(mokb_few_tokens_args); }

extern "C" size_t mokb_few_tokens_workspace_bytes(int num_tokens, int hidden, int intermediate, int topk, int mxfp8) {
    if (check_few_sizes(num_tokens, hidden, intermediate, topk) != MOKB_OK) return 0;
    return carve_few(nullptr, nullptr, num_tokens, hidden, intermediate, topk, mxfp8 != 0, sm_count());
}

extern "C" int mokb_few_tokens_fwd(const mokb_few_tokens_args* a, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    TraceScope trace(stream, "few_tokens");
    MOKB_REQUIRE(a != nullptr, "few_tokens: null args");
    MOKB_TRY(check_few_sizes(a->num_tokens, a->hidden, a->intermediate, a->topk));
    MOKB_REQUIRE(a->num_local_experts >= 1 && a->num_local_experts <= 4096, "few_tokens: num_local_experts must be in [1, 4096]");
    MOKB_REQUIRE(a->first_expert >= 0, "few_tokens: first_expert must not be negative");
    if (a->num_tokens == 0) return MOKB_OK;
    const bool mx = a->mxfp8 != 0, shared = a->w_shared_gate != nullptr;
    MOKB_REQUIRE(a->x && a->top_experts && a->router_weights && a->y && a->workspace && a->status, "few_tokens: null pointer");
    MOKB_REQUIRE(a->w_routed_gate && a->w_routed_up && a->w_routed_down, "few_tokens: null weight");
    MOKB_REQUIRE(shared == (a->w_shared_up != nullptr) && shared == (a->w_shared_down != nullptr), "few_tokens: the shared expert's weights go together");
    MOKB_REQUIRE(!mx || (a->w_routed_gate_sc && a->w_routed_up_sc && a->w_routed_down_sc), "few_tokens: null scales");
    MOKB_REQUIRE(((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->y)) & 15) == 0, "few_tokens: x and y must be 16-byte aligned");
    MOKB_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 255) == 0, "few_tokens: workspace must be 256-byte aligned");

    FewParams p;
    p.T = a->num_tokens; p.H = a->hidden; p.I = a->intermediate; p.E = a->num_local_experts; p.K = a->topk; p.first_expert = a->first_expert;
    p.mx = mx; p.shared = shared; p.has_limit = a->has_swiglu_limit; p.limit = a->swiglu_limit;
    p.sms = sm_count();
    p.x = static_cast<const __nv_bfloat16*>(a->x);
    p.top_experts = a->top_experts;
    p.weights = a->router_weights;
    p.y = static_cast<__nv_bfloat16*>(a->y);
    p.status = a->status;
    carve_few(&p.w, a->workspace, p.T, p.H, p.I, p.K, mx, p.sms);
    p.col_cap = column_cap(p.T, mx);
    const int stage_bytes = A_BYTES + p.col_cap * 128 + (mx ? SF_BYTES : 0);
    p.stages = (kSmemLimit - 1024 - kCtrlBytes) / stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    const size_t smem = 1024 + static_cast<size_t>(p.stages) * stage_bytes + kCtrlBytes;

    const int H = p.H, I = p.I, eb = mx ? 1 : 2, box = 128 / eb;
    const uint64_t E = static_cast<uint64_t>(p.E);
    FewMaps gu, dn;
    MOKB_TRY(make_tmap_2d(&gu.routed0, a->w_routed_gate, eb, H, E * I, static_cast<uint64_t>(H) * eb, box, 128));
    MOKB_TRY(make_tmap_2d(&gu.routed1, a->w_routed_up, eb, H, E * I, static_cast<uint64_t>(H) * eb, box, 128));
    MOKB_TRY(make_tmap_2d(&dn.routed0, a->w_routed_down, eb, I, E * H, static_cast<uint64_t>(I) * eb, box, 128));
    dn.routed1 = dn.routed0;
    gu.shared0 = gu.shared1 = gu.scale0 = gu.scale1 = gu.routed0;
    dn.shared0 = dn.shared1 = dn.scale0 = dn.scale1 = dn.routed0;
    if (shared) {
        MOKB_TRY(make_tmap_2d(&gu.shared0, a->w_shared_gate, 2, H, I, 2ull * H, 64, 128));
        MOKB_TRY(make_tmap_2d(&gu.shared1, a->w_shared_up, 2, H, I, 2ull * H, 64, 128));
        MOKB_TRY(make_tmap_2d(&dn.shared0, a->w_shared_down, 2, I, H, 2ull * I, 64, 128));
        dn.shared1 = dn.shared0;
    }
    if (mx) {
        const uint64_t tiles = E * (I / 128) * (H / 128);
        MOKB_TRY(make_tmap_2d(&gu.scale0, a->w_routed_gate_sc, 4, 128, tiles, 512, 128, 1));
        MOKB_TRY(make_tmap_2d(&gu.scale1, a->w_routed_up_sc, 4, 128, tiles, 512, 128, 1));
        MOKB_TRY(make_tmap_2d(&dn.scale0, a->w_routed_down_sc, 4, 128, tiles, 512, 128, 1));
        dn.scale1 = dn.scale0;
    }
    MOKB_TRY(allow_shared_memory());
    // The order of the four launches is part of their synchronisation: gate/up may trigger down only after it has seen the plan's end, so down
    // and sum read the plan ahead of their own wait.  A launch between them, or a plan that is itself launched programmatically, would
    // take that away.
    // few routes: fewer threads to start and to wait for
    const int plan_threads = p.T * p.K <= kPlanThreadsSmall && p.E <= 2 * kPlanThreadsSmall ? kPlanThreadsSmall : kPlanThreads;
    const int pieces = p.T * ((H + 1023) / 1024), quant_blocks = mx ? (pieces + plan_threads / 32 - 1) / (plan_threads / 32) : 0;
    few_plan_kernel<<<1 + (quant_blocks < p.sms ? quant_blocks : p.sms), plan_threads,
                      static_cast<size_t>(p.E) * 4 + 2 * (p.T * p.K < kPlanIds ? p.T * p.K : kPlanIds), stream>>>(p);
    MOKB_CUDA(cudaGetLastError());
    note_launch();
    MOKB_TRY(launch_after(few_product_kernel<false>, static_cast<unsigned>(p.sms), kThreads, smem, stream, gu, p));
    MOKB_TRY(launch_after(few_product_kernel<true>, static_cast<unsigned>(p.sms), kThreads, smem, stream, dn, p));
    return launch_after(few_sum_kernel, static_cast<unsigned>((p.T * (H / 256) + 3) / 4), 128, 0, stream, p);
}
