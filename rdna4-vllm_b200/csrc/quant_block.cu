// quant_block.cu — e4m3 quantisation with one scale per (row, 128 columns), with and without an
// RMS norm in front: the activation operand of the block-scaled FP8 products.
//
//   scale[r, g] = max(amax_{k in g} |y[r, k]|, 4.48e-6) / 448      (IEEE divide)
//   q[r, k]     = e4m3_rn_satfinite(y[r, k] / scale[r, g])          (IEEE quotient)
// with y = x (w4a8_act_quant_fp8_block), or the norm (w4a8_rms_norm_quant_fp8)
//   h = round_t(x + residual) (h = x without a residual), written as the new residual;
//   y = h * rsqrt(mean(h^2) + eps) * weight, fp32, and optionally normed = round_t(y).
// The clamp, the divide and the rounding are act_quant.cu's, applied per block of 128. The only
// roundings are h's (the residual stream is held in x's type) and the output's: sums, the norm
// and y stay in fp32.
//
// The amax ignores NaN: a NaN element becomes the e4m3 NaN and the rest of its block keeps its
// scale. An infinity makes its block's scale infinite, so that a product over it is not finite.
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"

namespace w4a8 {

namespace {

constexpr int kBlk = 128;  // columns of one scale

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One warp quantises one block of up to 128 values: v[j] is column lane + 32 j of the block.
__device__ __forceinline__ void quant_block_warp(const float (&v)[4], int cols, uint8_t* q,
                                                 float* scale) {
    const int lane = threadIdx.x & 31;
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(v[j]));
    amax = lanes_max<32>(amax);
    const float s = __fdiv_rn(fmaxf(amax, kAmaxFloor), kE4m3Max);
    if (lane == 0) *scale = s;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < cols)
            q[lane + 32 * j] = (uint8_t)f32x2_to_e4m3x2(__fdiv_rn(v[j], s), 0.f);
}

// Any K, any alignment: one warp per (row, block).
template <typename T>
__global__ void __launch_bounds__(256)
act_quant_block_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                       float* __restrict__ scales, int64_t blocks, int64_t K, int64_t G) {
    const int lane = threadIdx.x & 31;
    for (int64_t b = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks;
         b += (int64_t)gridDim.x * 8) {
        const int64_t r = b / G, k0 = (b - r * G) * kBlk;
        const int cols = (int)(K - k0 < kBlk ? K - k0 : kBlk);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = lane + 32 * j;
            v[j] = c < cols ? to_f32(x[r * K + k0 + c]) : 0.f;
        }
        quant_block_warp(v, cols, q + r * K + k0, scales + b);
    }
}

// Any H, any alignment: one CTA per row; the row is read once for the sum of squares and once
// more (from L2) for the output.
template <typename T, typename W>
__global__ void __launch_bounds__(256)
rms_norm_quant_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                      const W* __restrict__ weight, float eps, int64_t H, int64_t G,
                      uint8_t* __restrict__ q, float* __restrict__ scales,
                      T* __restrict__ residual_out, T* __restrict__ normed) {
    __shared__ float part[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t base = (int64_t)blockIdx.x * H;
    auto hidden = [&](int64_t k) {
        float h = to_f32(x[base + k]);
        if (residual) h = to_f32(from_f32<T>(h + to_f32(residual[base + k])));
        return h;
    };
    float ss = 0.f;
    for (int64_t k = threadIdx.x; k < H; k += 256) {
        const float h = hidden(k);
        ss += h * h;
    }
    ss = warp_sum(ss);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    float tot = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) tot += part[w];
    const float rstd = rsqrtf(tot / (float)H + eps);
    for (int64_t g = warp; g < G; g += 8) {
        const int64_t k0 = g * kBlk;
        const int cols = (int)(H - k0 < kBlk ? H - k0 : kBlk);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = lane + 32 * j;
            v[j] = 0.f;
            if (c < cols) {
                const float h = hidden(k0 + c);
                v[j] = h * rstd * to_f32(weight[k0 + c]);
                if (residual_out) residual_out[base + k0 + c] = from_f32<T>(h);
                if (normed) normed[base + k0 + c] = from_f32<T>(v[j]);
            }
        }
        quant_block_warp(v, cols, q + base + k0, scales + (int64_t)blockIdx.x * G + g);
    }
}

template <typename T>
int launch_quant(const void* x, int64_t M, int64_t K, uint8_t* q, float* scales, cudaStream_t st) {
    const int64_t G = (K + kBlk - 1) / kBlk, blocks = M * G;
    const int64_t want = (blocks + 7) / 8;
    const unsigned grid = (unsigned)(want < 148 * 64 ? want : 148 * 64);
    act_quant_block_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T*>(x), q, scales, blocks, K, G);
    return launch_status();
}

struct NormArgs {
    const void *x, *residual, *weight;
    float eps;
    int64_t M, H;
    uint8_t* q;
    float* scales;
    void *residual_out, *normed;
};

template <typename T, typename W>
int launch_norm(const NormArgs& a, cudaStream_t st) {
    rms_norm_quant_kernel<T, W><<<(unsigned)a.M, 256, 0, st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.residual),
        static_cast<const W*>(a.weight), a.eps, a.H, (a.H + kBlk - 1) / kBlk, a.q, a.scales,
        static_cast<T*>(a.residual_out), static_cast<T*>(a.normed));
    return launch_status();
}

template <typename T>
int launch_norm_w(const NormArgs& a, int32_t x_dtype, int32_t weight_dtype, cudaStream_t st) {
    return weight_dtype == x_dtype ? launch_norm<T, T>(a, st) : launch_norm<T, float>(a, st);
}

}  // namespace

}  // namespace w4a8

using namespace w4a8;

extern "C" int w4a8_act_quant_fp8_block(const void* x, int32_t x_dtype, int64_t M, int64_t K,
                                        uint8_t* q, float* scales, w4a8_stream_t stream) {
    const std::string o = "act_quant_fp8_block";
    if (x_dtype < 0 || x_dtype > 2)
        return set_error(o + ": x_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (M < 0 || K <= 0 || M > INT32_MAX || K > INT32_MAX)
        return set_error(o + ": bad sizes (0 <= M, 1 <= K, both below 2^31)");
    if (M == 0) return W4A8_OK;
    if (!x || !q || !scales) return set_error(o + ": null pointer");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (x_dtype) {
        case 0: return launch_quant<float>(x, M, K, q, scales, st);
        case 1: return launch_quant<__half>(x, M, K, q, scales, st);
        default: return launch_quant<__nv_bfloat16>(x, M, K, q, scales, st);
    }
}

extern "C" int w4a8_rms_norm_quant_fp8(const void* x, const void* residual, const void* weight,
                                       int32_t x_dtype, int32_t weight_dtype, float eps,
                                       int64_t M, int64_t H, uint8_t* q, float* scales,
                                       void* residual_out, void* normed, w4a8_stream_t stream) {
    const std::string o = "rms_norm_quant_fp8";
    if (x_dtype < 0 || x_dtype > 2)
        return set_error(o + ": x_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (weight_dtype != x_dtype && weight_dtype != 0)
        return set_error(o + ": weight must have x's type or fp32");
    if (M < 0 || H <= 0 || M > INT32_MAX || H > INT32_MAX)
        return set_error(o + ": bad sizes (0 <= M, 1 <= H, both below 2^31)");
    if (!(eps >= 0.f)) return set_error(o + ": eps must not be negative");
    if ((residual != nullptr) != (residual_out != nullptr))
        return set_error(o + ": residual and residual_out go together");
    if (M == 0) return W4A8_OK;
    if (!x || !weight || !q || !scales) return set_error(o + ": null pointer");
    const NormArgs a{x, residual, weight, eps, M, H, q, scales, residual_out, normed};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (x_dtype) {
        case 0: return launch_norm<float, float>(a, st);
        case 1: return launch_norm_w<__half>(a, x_dtype, weight_dtype, st);
        default: return launch_norm_w<__nv_bfloat16>(a, x_dtype, weight_dtype, st);
    }
}
