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

#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

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

// Eight consecutive values, packed as they lie in memory.
template <typename T>
struct Vec8 {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    // a buffer that this kernel also writes (the residual, updated in place): no read-only path
    __device__ __forceinline__ void load_rw(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = *(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(u[i]);
                v[i + 1] = __uint_as_float(u[i + 1]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i / 2]));
                v[i] = f.x;
                v[i + 1] = f.y;
            } else {  // a bf16 is the upper half of its fp32
                v[i] = __uint_as_float(u[i / 2] << 16);
                v[i + 1] = __uint_as_float(u[i / 2] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if constexpr (sizeof(T) == 4) {
                u[i] = __float_as_uint(v[i]);
                u[i + 1] = __float_as_uint(v[i + 1]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
                u[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
                u[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
};

// e4m3 bytes of v / s, IEEE quotients. With r the correctly rounded reciprocal of s and y = v r,
// the quotient's correctly rounded value is y + (v - y s) r, both steps fused multiply-adds
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).
// An infinite s has r = 0; its residual is taken with s = 0, which leaves y, as the divide would.
// Where the residual underflows, the quotient is far below e4m3's smallest value.
__device__ __forceinline__ float quotient(float v, float s, float r) {
    const float y = __fmul_rn(v, r);
    return __fmaf_rn(__fmaf_rn(-y, s, v), r, y);
}

// max(amax, floor) / 448, the IEEE quotient.
__device__ __forceinline__ float scale_of(float amax) {
    const float a = fmaxf(amax, kAmaxFloor);
    return isinf(a) ? a : quotient(a, kE4m3Max, 1.f / kE4m3Max);
}

// The steps of `quotient`, two values an instruction. Zeros keep their sign (the residual of a -0 is
// +0, and so would be its quotient).
__device__ __forceinline__ uint2 quant8(const float (&v)[8], float scale) {
    const float r = __frcp_rn(scale), s = isinf(scale) ? 0.f : -scale;
    const float2 r2 = make_float2(r, r), s2 = make_float2(s, s), none = make_float2(-0.f, -0.f);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 v2 = make_float2(v[i], v[i + 1]);
        float2 y = ffma2(v2, r2, none);
        y = ffma2(ffma2(y, s2, v2), r2, y);
        y = make_float2(copysignf(y.x, v2.x), copysignf(y.y, v2.y));
        u[i / 2] = f32x2_to_e4m3x2(y.x, y.y);
    }
    return make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
}

// The norm's: 16 lanes quantise one block, 8 values each (zeros past the row's end).
__device__ __forceinline__ uint2 quant_block_half(const float (&v)[8], float& s) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
    s = scale_of(lanes_max<16>(amax));
    return quant8(v, s);
}

// K % 8 == 0 and aligned rows: 8 lanes per block, two vectors of 8 each. Bound by HBM: 8192 x 4096
// bf16 in 18.5 us, 85 % of the measured copy bandwidth. What a block needs once, its maximum over
// the lanes and its scale, costs about as much as 16 values, so 16 lanes of 8 values took 20.5; two
// or four blocks a lane, all requested first, 19.0 and 20.5 (the last CTAs end later).
// kFull: K % 128 == 0, where blocks follow one another in memory and need no row arithmetic.
constexpr int kCtaBlocks = 32;
template <typename T, bool kFull>
__global__ void __launch_bounds__(8 * kCtaBlocks)
act_quant_block_vec_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                           float* __restrict__ scales, int64_t blocks, uint32_t K, uint32_t G) {
    const int sub = threadIdx.x & 7;
    const int64_t b = (int64_t)blockIdx.x * kCtaBlocks + (threadIdx.x >> 3);
    uint32_t k = sub * 8;  // column of the first vector; the second is 64 on
    int64_t at = b * kBlk + k;
    if (!kFull) {
        const int64_t r = blocks <= INT32_MAX ? (int64_t)((uint32_t)b / G) : b / G;
        k += (uint32_t)(b - r * G) * kBlk;
        at = r * K + k;
    }
    Vec8<T> x8[2];
    bool ok[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        ok[h] = b < blocks && (kFull || k + h * 64 < K);
        x8[h].zero();
        if (ok[h]) x8[h].load(x + at + h * 64);
    }
    float v[2][8], amax = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        x8[h].get(v[h]);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[h][j]));
    }
    const float s = scale_of(lanes_max<8>(amax));
    if (sub == 0 && b < blocks) scales[b] = s;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (ok[h]) *reinterpret_cast<uint2*>(q + at + h * 64) = quant8(v[h], s);
}

// The norm with the row in registers: kThreads threads per row, V vectors of 8 each (vector j of
// thread t is j * kThreads + t, so 16 neighbours hold one block). A CTA walks rows with the
// weights kept; rows of H % 8 == 0 elements, H <= 8 V kThreads, aligned. One pass over the rows,
// bound by HBM: 16381 x 2048 bf16 with a residual in 43.0 us, 85 % of the measured copy bandwidth.
// CTAs for half or five eighths of the threads that an SM holds take 0.3 and 0.7 us more.
template <typename T, typename W, int kThreads, int V>
__global__ void __launch_bounds__(kThreads)
rms_norm_quant_vec_kernel(const T* __restrict__ x, const T* residual, const W* __restrict__ weight,
                          float eps, int64_t M, uint32_t H, uint32_t G, uint8_t* __restrict__ q,
                          float* __restrict__ scales, T* residual_out, T* __restrict__ normed) {
    __shared__ float part[2][kThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t vecs = H / 8;
    Vec8<W> w8[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w8[j].zero();
        if (j * kThreads + tid < vecs) w8[j].load(weight + (j * kThreads + tid) * 8);
    }
    int turn = 0;
    for (int64_t r = blockIdx.x; r < M; r += gridDim.x, turn ^= 1) {
        const int64_t base = r * H;
        Vec8<T> x8[V], r8[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t n = j * kThreads + tid;
            x8[j].zero();
            r8[j].zero();
            if (n < vecs) {
                x8[j].load(x + base + n * 8);
                if (residual) r8[j].load_rw(residual + base + n * 8);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float h[8];
            x8[j].get(h);
            if (residual) {
                float d[8];
                r8[j].get(d);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] += d[i];
                x8[j].set(h);
                x8[j].get(h);
                const uint32_t n = j * kThreads + tid;
                if (n < vecs) x8[j].store(residual_out + base + n * 8);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += h[i] * h[i];
        }
        ss = warp_sum(ss);
        if (lane == 0) part[turn][warp] = ss;
        __syncthreads();  // the next row writes the other half of `part`
        float tot = 0.f;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) tot += part[turn][i];
        const float rstd = rsqrtf(tot / (float)H + eps);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t n = j * kThreads + tid;
            float v[8], wv[8], s;
            x8[j].get(v);  // zeros past the row's end
            w8[j].get(wv);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * rstd * wv[i];
            if (n >= vecs) {  // 0 * rstd is NaN in a row that overflowed
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
            }
            const uint2 u = quant_block_half(v, s);
            if (n < vecs) {
                if ((tid & 15) == 0) scales[r * G + n / 16] = s;
                *reinterpret_cast<uint2*>(q + base + n * 8) = u;
                if (normed) {
                    x8[j].set(v);
                    x8[j].store(normed + base + n * 8);
                }
            }
        }
    }
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

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

// Any K, any alignment: one warp per (row, block), a value a lane and load. 8192 x 4095 bf16 in 56 us,
// a third of the vectorised kernel's rate.
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
// more (from L2) for the output. 16381 x 2047 bf16 with a residual in 93 us, 43 at H = 2048 by the
// vectorised kernel.
template <typename T, typename W>
__global__ void __launch_bounds__(256)
rms_norm_quant_kernel(const T* __restrict__ x, const T* residual,
                      const W* __restrict__ weight, float eps, int64_t H, int64_t G,
                      uint8_t* __restrict__ q, float* __restrict__ scales,
                      T* residual_out, T* __restrict__ normed) {
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
    if (K % 8 == 0 && aligned(x, 16) && aligned(q, 8)) {
        const int64_t ctas = (blocks + kCtaBlocks - 1) / kCtaBlocks;
        if (ctas <= INT32_MAX) {
            if (K % kBlk == 0)
                act_quant_block_vec_kernel<T, true><<<(unsigned)ctas, 8 * kCtaBlocks, 0, st>>>(
                    static_cast<const T*>(x), q, scales, blocks, (uint32_t)K, (uint32_t)G);
            else
                act_quant_block_vec_kernel<T, false><<<(unsigned)ctas, 8 * kCtaBlocks, 0, st>>>(
                    static_cast<const T*>(x), q, scales, blocks, (uint32_t)K, (uint32_t)G);
            return launch_status();
        }
    }
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

template <typename T, typename W, int kThreads, int V>
int launch_norm_vec(const NormArgs& a, cudaStream_t st) {
    const int64_t most = (int64_t)148 * (2048 / kThreads);  // CTAs that fill the GPU
    rms_norm_quant_vec_kernel<T, W, kThreads, V><<<(unsigned)(a.M < most ? a.M : most), kThreads, 0, st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.residual),
        static_cast<const W*>(a.weight), a.eps, a.M, (uint32_t)a.H,
        (uint32_t)((a.H + kBlk - 1) / kBlk), a.q, a.scales, static_cast<T*>(a.residual_out),
        static_cast<T*>(a.normed));
    return launch_status();
}

template <typename T, typename W>
int launch_norm(const NormArgs& a, cudaStream_t st) {
    if (a.H % 8 == 0 && a.H <= 16384 && aligned(a.x, 16) && aligned(a.residual, 16) &&
        aligned(a.weight, 16) && aligned(a.q, 8) && aligned(a.residual_out, 16) &&
        aligned(a.normed, 16)) {
        if (a.H <= 1024) return launch_norm_vec<T, W, 128, 1>(a, st);
        if (a.H <= 2048) return launch_norm_vec<T, W, 128, 2>(a, st);
        if (a.H <= 4096) return launch_norm_vec<T, W, 256, 2>(a, st);
        if (a.H <= 8192) return launch_norm_vec<T, W, 256, 4>(a, st);
        return launch_norm_vec<T, W, 512, 4>(a, st);
    }
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
