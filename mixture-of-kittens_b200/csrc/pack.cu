// Activations kept in 8 bits between the forward and the backward pass: whole numbers in [-127, 127] with one fp32 scale per 128
// consecutive values of a row, 1.03 bytes a value instead of 2.
//
//   scale = max|x| / 127,  q = x / scale to the nearest, halves away from zero;   x ~ q * scale, off by at most half a step
// Of values drawn from one distribution that is three to four times nearer than E4M3 with a scale per 32 (whose step grows with the
// value), which is why this is not the layer's MXFP8 form.  A block whose largest value is below 2^-110 is kept as zeros; one that holds
// an infinity or NaN comes back as NaN, so that a fault stays visible.
//
//   pack_kernel        bf16 -> q, scales
//   unpack_kernel      q, scales -> bf16 (the x rows, which a weight-gradient GEMM reads)
//   swiglu_bwd_packed  the backward pass of SwiGLU straight from packed gate and up; gives `hidden` back as well, so the
//                      forward pass keeps two of its three [rows, I] tensors, in half the bytes
// All bound by HBM.  A lane works on 16 consecutive values: 32 bytes of bf16, 16 of q; eight lanes have one scale.
#include "common.cuh"
#include "mxfp8_codec.cuh"

namespace mokb {
namespace {

constexpr int kBlock = 128;
constexpr float kSmallest = 7.70371977754894e-34f;        // 2^-110
constexpr float kRound = 12582912.0f;

__device__ __forceinline__ int64_t live_rows(const int32_t* num_rows, int64_t cap) {
    if (!num_rows) return cap;
    const int64_t n = *num_rows;
    return n < 0 ? 0 : n < cap ? n : cap;
}

// 16-byte loads and stores of bytes that are used once
__device__ __forceinline__ uint4 ld_once(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }

// Eight lanes hold a block's 128 values (16 each, as bf16 pairs): q as bytes, and the scale, the same in all eight.
__device__ __forceinline__ uint4 pack_16(const uint32_t (&w)[8], float* scale) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);           // of the bits: NaN above infinity above numbers
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float top = __uint_as_float(m << 16);
    const bool bad = m >= 0x7f80u;
    *scale = bad ? __int_as_float(0x7fffffff) : top >= kSmallest ? __fdiv_rn(top, 127.0f) : 0.0f;
    // 127 / top, a little (2^-18) more: with 8-bit fractions x * 127 / top is a half exactly or at least 1.5e-5 of itself away from one,
    // so halves go away from zero and nothing else moves
    const float inv = bad || top < kSmallest ? 0.0f : __fdiv_rn(127.0f * (1.0f + 3.814697265625e-6f), top);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // 1.5 * 2^23 more: the sum's last place is 1, so that it is rounded to a whole number, whose low byte is the float's
        const uint32_t a = __float_as_uint(fmaf(bf16_lo(w[2 * i]), inv, kRound)), b = __float_as_uint(fmaf(bf16_hi(w[2 * i]), inv, kRound));
        const uint32_t c = __float_as_uint(fmaf(bf16_lo(w[2 * i + 1]), inv, kRound)), d = __float_as_uint(fmaf(bf16_hi(w[2 * i + 1]), inv, kRound));
        o[i] = bad ? 0u : __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// The four signed bytes of a word as numbers, through the mantissa of 2^23 + byte + 128 (exact; a conversion instruction per byte is a
// quarter-rate one, of which the exponential and the quotient have enough).
__device__ __forceinline__ void signed_bytes(uint32_t w, float (&f)[4]) {
    w ^= 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540u + j)) - 8388736.0f;
}

// 135168 x 2048: 130 us, 6.5 TB/s (with a float-to-integer conversion per value: 143); 135168 x 7168: 449 us, 6.5 TB/s.  Before that, 16 blocks per
// SM instead of 32 took 147 for 143, a block for every 64 scales 159, two groups of four scales in flight per warp 157.
// A warp takes four blocks at a time.  `per_row` blocks of a row, the last one shorter where 128 does not divide cols.
__global__ void __launch_bounds__(256) pack_kernel(const __nv_bfloat16* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scales,
                                                   const int32_t* __restrict__ num_rows, int64_t rows_cap, int cols, int per_row) {
    const int64_t items = live_rows(num_rows, rows_cap) * per_row * 8, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    const int lane = threadIdx.x & 31;
    const bool even = cols % kBlock == 0;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x - lane; i0 < items; i0 += stride) {      // the same trips in a warp
        const int64_t i = i0 + lane, block = i >> 3;
        int64_t at = i * 16;
        bool inside = i < items;
        if (!even) {
            const int64_t row = block / per_row;
            const int c = static_cast<int>(block - row * per_row) * kBlock + static_cast<int>(i & 7) * 16;
            inside = inside && c < cols;
            at = row * cols + c;
        }
        uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        if (inside) ld_global_32B(x + at, w);
        float scale;
        const uint4 o = pack_16(w, &scale);
        if (inside) *reinterpret_cast<uint4*>(q + at) = o;
        if ((i & 7) == 0 && i < items) scales[block] = scale;
    }
}

// 135168 x 2048: 125 us, 6.7 TB/s, every thread one unit (with a conversion per byte 130, and 145 where 16 blocks per SM go on);
// 135168 x 7168: 432 us, 6.8 TB/s.
__global__ void __launch_bounds__(256) unpack_kernel(const int8_t* __restrict__ q, const float* __restrict__ scales, __nv_bfloat16* __restrict__ x,
                                                     const int32_t* __restrict__ num_rows, int64_t rows_cap, int cols, int per_row) {
    const int64_t items = live_rows(num_rows, rows_cap) * (cols / 16), stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    const int units = cols / 16;
    const bool even = cols % kBlock == 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += stride) {
        int64_t block = i >> 3;
        if (!even) {
            const int64_t row = i / units;
            block = row * per_row + (i - row * units) / 8;
        }
        const uint4 v = ld_once(q + i * 16);
        const float s = __ldg(scales + block);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[4];
            signed_bytes(w[j], f);
            o[2 * j] = pack2(f[0] * s, f[1] * s);
            o[2 * j + 1] = pack2(f[2] * s, f[3] * s);
        }
        st_global_32B(x + i * 16, o);
    }
}

__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// A block takes up to eight consecutive rows, its threads their units in order, so that no lane idles behind a row's end and what is open
// in memory at a time is whole rows; the rows' sums of d_hidden * hidden go through shared memory, one number per unit, and are added up
// in a fixed order.  135168 x 2048 back to back for a second: 467 us, 6.0 TB/s; 25088 x 1408 with a limit: 71 us.  64 registers, none spilled: held to
// 48, of which a few spill, 477 and 71 us (one pass of pack, pack and this: 10 us more), with 76, 513 and 81.
// (Tried with an approximate quotient, which took 430 and 67 us: a warp per row 468 to 506, two rows to a block 509, sixteen 450; limited 73 to 94.)
// Back to back it is the board's power that bounds it (1 kW, 1.6 of 1.97 GHz), so instructions count.  The sigmoid's quotient is the IEEE one all
// the same, as in mokb_swiglu_bwd: the approximate one rounds some gradients to the neighbouring bf16 number (6 of two million).
constexpr int kRowsPerBlock = 8, kUnitsPerBlock = 8192;
template <bool LIMIT>
__global__ void __launch_bounds__(256, 4) swiglu_bwd_packed_kernel(
    const int8_t* __restrict__ gate_q, const float* __restrict__ gate_sc, const int8_t* __restrict__ up_q, const float* __restrict__ up_sc,
    const __nv_bfloat16* __restrict__ d_hidden, __nv_bfloat16* __restrict__ d_gate, __nv_bfloat16* __restrict__ d_up,
    __nv_bfloat16* __restrict__ hidden, const float* __restrict__ row_scale, float* __restrict__ row_grad,
    const int32_t* __restrict__ num_rows, int64_t rows_cap, int cols, int per_row, int rows_per_block, float limit) {
    extern __shared__ float unit_sum[];
    const int64_t rows = live_rows(num_rows, rows_cap);
    const int units = cols / 16;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_block; row0 < rows; row0 += static_cast<int64_t>(gridDim.x) * rows_per_block) {
        const int n = static_cast<int>(rows - row0 < rows_per_block ? rows - row0 : rows_per_block), items = n * units;
        for (int i = threadIdx.x; i < items; i += 256) {
            const int r = i / units, u = i - r * units;
            const int64_t at = row0 * cols + static_cast<int64_t>(i) * 16, block = (row0 + r) * per_row + (u >> 3);
            const uint4 gv = ld_once(gate_q + at), uv = ld_once(up_q + at);
            uint32_t dh[8];
            ld_global_32B(d_hidden + at, dh);
            const float gs = __ldg(gate_sc + block), us = __ldg(up_sc + block);
            const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w}, uw[4] = {uv.x, uv.y, uv.z, uv.w};
            uint32_t og[8], ou[8], oh[8];
            float sum = 0.0f;
            const float inv_w = row_grad && row_scale ? row_inverse(__ldg(row_scale + row0 + r)) : 1.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float g4[4], u4[4], dg[4], du[4], h[4];
                signed_bytes(gw[j], g4);
                signed_bytes(uw[j], u4);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float g0 = g4[b] * gs, u0 = u4[b] * us;
                    const float d = b & 1 ? bf16_hi(dh[2 * j + (b >> 1)]) : bf16_lo(dh[2 * j + (b >> 1)]);
                    const float g = LIMIT ? min_nan(g0, limit) : g0, up = LIMIT ? min_nan(max_nan(u0, -limit), limit) : u0;
                    const float sig = 1.0f / (1.0f + __expf(-g));
                    const float silu = g * sig;
                    h[b] = silu * up;
                    dg[b] = ((1.0f - silu) * sig + silu) * up * d;
                    du[b] = silu * d;
                    if (LIMIT && g0 > limit) dg[b] = 0.0f;
                    if (LIMIT && (u0 > limit || u0 < -limit)) du[b] = 0.0f;
                    sum += d * inv_w * h[b];
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    og[2 * j + b] = pack2(dg[2 * b], dg[2 * b + 1]);
                    ou[2 * j + b] = pack2(du[2 * b], du[2 * b + 1]);
                    oh[2 * j + b] = pack2(h[2 * b], h[2 * b + 1]);
                }
            }
            st_global_32B(d_gate + at, og);
            st_global_32B(d_up + at, ou);
            st_global_32B(hidden + at, oh);
            if (row_grad) unit_sum[i] = sum;
        }
        if (row_grad) {
            __syncthreads();
            for (int r = threadIdx.x >> 5; r < n; r += 8) {
                float sum = 0.0f;
                for (int u = threadIdx.x & 31; u < units; u += 32) sum += unit_sum[r * units + u];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if ((threadIdx.x & 31) == 0) {
                    const float w = row_scale ? __ldg(row_scale + row0 + r) : 1.0f;
                    row_grad[row0 + r] = w > 0.0f ? sum * row_rest(w) : 0.0f;      // (0 times a fault in the row would be NaN)
                }
            }
            __syncthreads();
        }
    }
}

int blocks_for(int64_t threads, int per_sm) {
    int64_t b = (threads + 255) / 256;
    const int64_t most = static_cast<int64_t>(sm_count()) * per_sm;
    if (b > most) b = most;
    return b < 1 ? 1 : static_cast<int>(b);
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace mokb

using namespace mokb;

#define CHECK_PACK(who)                                                                                                              \
    MOKB_REQUIRE(rows >= 0 && cols > 0 && cols % 16 == 0 && cols <= (1 << 24), who ": cols must be a positive multiple of 16")

extern "C" int mokb_pack_rows(const void* x, void* q, float* scales, const int32_t* num_rows, int64_t rows, int64_t cols, void* stream) {
    TraceScope trace(static_cast<cudaStream_t>(stream), "pack_rows");
    CHECK_PACK("pack_rows");
    if (rows == 0) return MOKB_OK;
    MOKB_REQUIRE(x && q && scales, "pack_rows: null pointer");
    MOKB_REQUIRE(aligned(x, 32) && aligned(q, 16), "pack_rows: x must be 32-byte and q 16-byte aligned");
    const int per_row = static_cast<int>((cols + kBlock - 1) / kBlock);
    pack_kernel<<<blocks_for(rows * per_row * 8, 32), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const __nv_bfloat16*>(x), static_cast<int8_t*>(q), scales, num_rows, rows, static_cast<int>(cols), per_row);
    MOKB_CUDA(cudaGetLastError());
    note_launch();
    return MOKB_OK;
}

extern "C" int mokb_unpack_rows(const void* q, const float* scales, void* x, const int32_t* num_rows, int64_t rows, int64_t cols, void* stream) {
    TraceScope trace(static_cast<cudaStream_t>(stream), "unpack_rows");
    CHECK_PACK("unpack_rows");
    if (rows == 0) return MOKB_OK;
    MOKB_REQUIRE(x && q && scales, "unpack_rows: null pointer");
    MOKB_REQUIRE(aligned(x, 32) && aligned(q, 16), "unpack_rows: x must be 32-byte and q 16-byte aligned");
    unpack_kernel<<<blocks_for(rows * (cols / 16), 4096), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const int8_t*>(q), scales, static_cast<__nv_bfloat16*>(x), num_rows, rows, static_cast<int>(cols),
        static_cast<int>((cols + kBlock - 1) / kBlock));
    MOKB_CUDA(cudaGetLastError());
    note_launch();
    return MOKB_OK;
}

extern "C" int mokb_swiglu_bwd_packed(const void* gate_q, const float* gate_scales, const void* up_q, const float* up_scales,
                                      const void* d_hidden, void* d_gate, void* d_up, void* hidden, const float* row_scale,
                                      float* row_grad_out, const int32_t* num_rows, int64_t rows, int64_t cols, int has_limit, float limit,
                                      void* stream) {
    TraceScope trace(static_cast<cudaStream_t>(stream), "swiglu_bwd_packed");
    CHECK_PACK("swiglu_bwd_packed");
    MOKB_REQUIRE(cols <= 16 * kUnitsPerBlock, "swiglu_bwd_packed: at most 131072 columns");
    if (rows == 0) return MOKB_OK;
    MOKB_REQUIRE(gate_q && gate_scales && up_q && up_scales && d_hidden && d_gate && d_up && hidden, "swiglu_bwd_packed: null pointer");
    MOKB_REQUIRE(aligned(gate_q, 16) && aligned(up_q, 16) && aligned(d_hidden, 32) && aligned(d_gate, 32) && aligned(d_up, 32) && aligned(hidden, 32),
                 "swiglu_bwd_packed: packed tensors must be 16-byte and bf16 tensors 32-byte aligned");
    auto* const kernel = has_limit ? swiglu_bwd_packed_kernel<true> : swiglu_bwd_packed_kernel<false>;
    const int units = static_cast<int>(cols / 16), rpb = kRowsPerBlock * units <= kUnitsPerBlock ? kRowsPerBlock : kUnitsPerBlock / units;
    const int64_t blocks = (rows + rpb - 1) / rpb;
    kernel<<<static_cast<unsigned>(blocks < (1 << 30) ? blocks : (1 << 30)), 256, row_grad_out ? sizeof(float) * rpb * units : 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const int8_t*>(gate_q), gate_scales, static_cast<const int8_t*>(up_q), up_scales, static_cast<const __nv_bfloat16*>(d_hidden),
        static_cast<__nv_bfloat16*>(d_gate), static_cast<__nv_bfloat16*>(d_up), static_cast<__nv_bfloat16*>(hidden), row_scale, row_grad_out,
        num_rows, rows, static_cast<int>(cols), static_cast<int>((cols + kBlock - 1) / kBlock), rpb, limit);
    MOKB_CUDA(cudaGetLastError());
    note_launch();
    return MOKB_OK;
}
