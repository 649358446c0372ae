// reduce.cu — topk-weighted gather-reduce of the down-projection rows back to tokens.
//
// Semantics of mmq_fp8_moe_gather_reduce (w4a8_fp8_wmma/moe_kernel.hip:1230-1262):
//   slot_to_row[slot] = r for every r < ntp with sorted_token_ids[r] = slot < M*top_k, else -1;
//   out[t, n] = sum_{j ascending} w[t*top_k + j] * out2[slot_to_row[t*top_k + j], n]   (fp32)
// The sum is a plain fp32 multiply then add in slot order, the order the reference oracle uses
// (w4a8_fp8_wmma/test_moe_experts.py:182-190).
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace w4a8 {

namespace {

// Row element types: fp16, or the rows of a block-scaled down product, bf16 for a bf16 model and
// fp32 for an fp32 result.
__device__ __forceinline__ float row_f32(float v) { return v; }
__device__ __forceinline__ float row_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float row_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename InT>
__device__ __forceinline__ float2 pair_f32(uint32_t w) {
    const InT* h = reinterpret_cast<const InT*>(&w);
    return make_float2(row_f32(h[0]), row_f32(h[1]));
}
// The values of 16 bytes of a row.
template <typename InT>
__device__ __forceinline__ void unpack16(uint4 v, float (&f)[16 / sizeof(InT)]) {
    const uint32_t h[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if constexpr (sizeof(InT) == 4) {
            f[c] = __uint_as_float(h[c]);
        } else {
            const float2 p = pair_f32<InT>(h[c]);
            f[2 * c] = p.x;
            f[2 * c + 1] = p.y;
        }
    }
}

__global__ void build_inverse_map_kernel(const int32_t* __restrict__ sorted_ids,
                                         const int32_t* __restrict__ ntp, int32_t* slot_to_row,
                                         int64_t P, int64_t num_slots) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= P || r >= ntp[0]) return;
    const int32_t slot = sorted_ids[r];
    if (slot >= 0 && slot < num_slots) slot_to_row[slot] = (int32_t)r;
}

// The token of a CTA: tokens lie over y and z of the grid, since y alone ends at 65535.
__device__ __forceinline__ int64_t grid_token() {
    return (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
}

// One CTA per (token, 512-channel chunk); each thread reduces 2 adjacent channels. Generic
// path for rows that 16 bytes do not divide or that are unaligned. `pairs`: 16-bit rows that all start
// on a 4-byte boundary (N even, and out2 itself: a view may start at any element), so that two channels
// are one load.
template <typename InT, typename OutT>
__global__ void __launch_bounds__(256)
gather_reduce_kernel(const InT* __restrict__ out2, const int32_t* __restrict__ slot_to_row,
                     const float* __restrict__ topk_w, OutT* __restrict__ out, int64_t M,
                     int64_t N, int top_k, bool pairs) {
    const int64_t t = grid_token();
    const int64_t n = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 2;
    if (t >= M || n >= N) return;
    float a0 = 0.f, a1 = 0.f;
    const bool pair = (n + 1 < N);
    for (int j = 0; j < top_k; ++j) {
        const int32_t r = slot_to_row[t * top_k + j];
        if (r < 0) continue;
        const float w = topk_w[t * top_k + j];
        const InT* rowp = out2 + (int64_t)r * N + n;
        if constexpr (sizeof(InT) == 2) {
            if (pairs) {  // N is even: n + 1 < N
                const float2 v = pair_f32<InT>(*reinterpret_cast<const uint32_t*>(rowp));
                a0 = __fadd_rn(a0, __fmul_rn(w, v.x));
                a1 = __fadd_rn(a1, __fmul_rn(w, v.y));
                continue;
            }
        }
        a0 = __fadd_rn(a0, __fmul_rn(w, row_f32(rowp[0])));
        if (pair) a1 = __fadd_rn(a1, __fmul_rn(w, row_f32(rowp[1])));
    }
    out[t * N + n] = (OutT)a0;
    if (pair) out[t * N + n + 1] = (OutT)a1;
}

// Vector path (16-byte aligned rows): 16 bytes of channels per thread (8, or 4 of fp32);
// the top_k row indices and weights of the token are staged once per CTA, then every slot's
// 16-byte row chunk is requested before the in-order accumulation.
constexpr int kMaxTopK = 16;
template <typename InT, typename OutT>
__global__ void __launch_bounds__(256)
gather_reduce_vec_kernel(const InT* __restrict__ out2, const int32_t* __restrict__ slot_to_row,
                         const float* __restrict__ topk_w, OutT* __restrict__ out, int64_t M,
                         int64_t N, int top_k) {
    constexpr int kPer = 16 / sizeof(InT);
    __shared__ int32_t rows[kMaxTopK];
    __shared__ float wts[kMaxTopK];
    const int64_t t = grid_token();
    if (t >= M) return;
    if (threadIdx.x < top_k) {
        rows[threadIdx.x] = slot_to_row[t * top_k + threadIdx.x];
        wts[threadIdx.x] = topk_w[t * top_k + threadIdx.x];
    }
    __syncthreads();
    const int64_t n = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * kPer;
    if (n >= N) return;
    uint4 v[kMaxTopK];
#pragma unroll
    for (int j = 0; j < kMaxTopK; ++j)
        if (j < top_k && rows[j] >= 0)
            v[j] = __ldg(reinterpret_cast<const uint4*>(out2 + (int64_t)rows[j] * N + n));
    float acc[kPer];
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxTopK; ++j) {
        if (j < top_k && rows[j] >= 0) {
            const float w = wts[j];
            float f[kPer];
            unpack16<InT>(v[j], f);
#pragma unroll
            for (int c = 0; c < kPer; ++c) acc[c] = __fadd_rn(acc[c], __fmul_rn(w, f[c]));
        }
    }
    if constexpr (sizeof(OutT) == 4) {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + t * N + n);
#pragma unroll
        for (int c = 0; c < kPer; c += 4)
            o[c / 4] = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    } else {
        static_assert(sizeof(OutT) == 4 || kPer == 8, "16-bit results are made of 16-bit rows");
        uint4 o;
        uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const __half2 h2 = __floats2half2_rn(acc[2 * c], acc[2 * c + 1]);
            ow[c] = *reinterpret_cast<const uint32_t*>(&h2);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(out) + t * N + n) = o;
    }
}

}  // namespace

template <typename InT, typename OutT>
static int launch_reduce(const InT* out2, const int32_t* slot_to_row, const float* topk_w,
                         OutT* out, int64_t M, int64_t N, int top_k, cudaStream_t stream) {
    if (M <= 0) return W4A8_OK;
    constexpr int kPer = 16 / sizeof(InT);
    const bool vec = N % kPer == 0 && top_k <= kMaxTopK &&
                     (reinterpret_cast<uintptr_t>(out2) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int64_t z = (M + 65534) / 65535;
    const unsigned y = (unsigned)((M + z - 1) / z);
    if (vec) {
        const dim3 grid((unsigned)((N / kPer + 255) / 256), y, (unsigned)z);
        gather_reduce_vec_kernel<InT, OutT><<<grid, 256, 0, stream>>>(out2, slot_to_row, topk_w,
                                                                      out, M, N, top_k);
    } else {
        const bool pairs = sizeof(InT) == 2 && N % 2 == 0 && (reinterpret_cast<uintptr_t>(out2) & 3) == 0;
        const dim3 grid((unsigned)((N + 511) / 512), y, (unsigned)z);
        gather_reduce_kernel<InT, OutT><<<grid, 256, 0, stream>>>(out2, slot_to_row, topk_w, out,
                                                                  M, N, top_k, pairs);
    }
    return launch_status();
}

int launch_gather_reduce(const __half* out2, const int32_t* slot_to_row, const float* topk_w,
                         void* out, bool out_half, int64_t M, int64_t N, int top_k,
                         cudaStream_t stream) {
    if (out_half)
        return launch_reduce(out2, slot_to_row, topk_w, static_cast<__half*>(out), M, N, top_k, stream);
    return launch_reduce(out2, slot_to_row, topk_w, static_cast<float*>(out), M, N, top_k, stream);
}

}  // namespace w4a8

extern "C" size_t w4a8_moe_gather_reduce_workspace_size(int64_t M, int64_t top_k) {
    return w4a8::align_up((size_t)(M * top_k) * sizeof(int32_t), 256);
}

namespace w4a8 {
namespace {

template <typename InT>
int gather_reduce_entry(const void* out2, const int32_t* sorted_token_ids,
                        const float* topk_weights, const int32_t* num_tokens_post_padded,
                        float* out, int64_t M, int64_t N, int64_t P, int64_t top_k,
                        void* workspace, size_t workspace_bytes, w4a8_stream_t stream) {
    if (M < 0 || N <= 0 || P < 0 || top_k <= 0) return set_error("gather_reduce: bad sizes");
    if (M * top_k > INT32_MAX) return set_error("gather_reduce: size overflow");
    if (M == 0) return W4A8_OK;
    if (!out || !topk_weights || (P > 0 && (!out2 || !sorted_token_ids || !num_tokens_post_padded)))
        return set_error("gather_reduce: null pointer");
    if (!workspace || workspace_bytes < w4a8_moe_gather_reduce_workspace_size(M, top_k))
        return set_error("gather_reduce: workspace too small");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int32_t* map = static_cast<int32_t*>(workspace);
    cudaError_t e = cudaMemsetAsync(map, 0xFF, (size_t)(M * top_k) * sizeof(int32_t), st);
    if (e != cudaSuccess) return (int)e;
    if (P > 0) {
        build_inverse_map_kernel<<<(unsigned)((P + 255) / 256), 256, 0, st>>>(
            sorted_token_ids, num_tokens_post_padded, map, P, M * top_k);
        if (int rc = launch_status()) return rc;
    }
    return launch_reduce(static_cast<const InT*>(out2), map, topk_weights, out, M, N, (int)top_k,
                         st);
}

}  // namespace
}  // namespace w4a8

extern "C" int w4a8_moe_gather_reduce(const void* out2, const int32_t* sorted_token_ids,
                                      const float* topk_weights,
                                      const int32_t* num_tokens_post_padded, float* out,
                                      int64_t M, int64_t N, int64_t P, int64_t top_k,
                                      void* workspace, size_t workspace_bytes,
                                      w4a8_stream_t stream) {
    return w4a8::gather_reduce_entry<__half>(out2, sorted_token_ids, topk_weights,
                                             num_tokens_post_padded, out, M, N, P, top_k,
                                             workspace, workspace_bytes, stream);
}

extern "C" int w4a8_moe_gather_reduce_bf16(const void* out2, const int32_t* sorted_token_ids,
                                           const float* topk_weights,
                                           const int32_t* num_tokens_post_padded, float* out,
                                           int64_t M, int64_t N, int64_t P, int64_t top_k,
                                           void* workspace, size_t workspace_bytes,
                                           w4a8_stream_t stream) {
    return w4a8::gather_reduce_entry<__nv_bfloat16>(out2, sorted_token_ids, topk_weights,
                                                    num_tokens_post_padded, out, M, N, P, top_k,
                                                    workspace, workspace_bytes, stream);
}

extern "C" int w4a8_moe_gather_reduce_f32(const void* out2, const int32_t* sorted_token_ids,
                                          const float* topk_weights,
                                          const int32_t* num_tokens_post_padded, float* out,
                                          int64_t M, int64_t N, int64_t P, int64_t top_k,
                                          void* workspace, size_t workspace_bytes,
                                          w4a8_stream_t stream) {
    return w4a8::gather_reduce_entry<float>(out2, sorted_token_ids, topk_weights,
                                            num_tokens_post_padded, out, M, N, P, top_k, workspace,
                                            workspace_bytes, stream);
}

namespace w4a8 {
namespace {

// out[r][i] = fp16(silu(fp16 gate)) * fp16 up with gate = x[r][i], up = x[r][I + i]: vLLM's
// silu_and_mul on fp16 tensors, the step between gate_up and down in the unfused composition.
__global__ void __launch_bounds__(256) silu_and_mul_kernel(const __half* __restrict__ x,
                                                           __half* __restrict__ out, int64_t M,
                                                           int64_t I) {
    const int64_t n = M * I;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / I, c = i - r * I;
        out[i] = silu_mul_h(x[r * 2 * I + c], x[r * 2 * I + I + c]);
    }
}

}  // namespace
}  // namespace w4a8

extern "C" int w4a8_silu_and_mul(const void* x, void* out, int64_t M, int64_t inter,
                                 w4a8_stream_t stream) {
    using namespace w4a8;
    if (M < 0 || inter < 0) return set_error("silu_and_mul: negative size");
    if (M == 0 || inter == 0) return W4A8_OK;
    if (!x || !out) return set_error("silu_and_mul: null pointer");
    const int64_t n = M * inter;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 16);
    silu_and_mul_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        static_cast<const __half*>(x), static_cast<__half*>(out), M, inter);
    return launch_status();
}
