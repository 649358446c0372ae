// gemm_fp8_block.cu — block-scaled FP8 products: the C entry points and the plain kernel.
//
//   out[r, n] = sum_g xs[src(r), g] * ws[n / 128, g] * sum_{k in g} x[src(r), k] * w[n, k]
// over blocks g of 128 columns. e4m3 x e4m3 products are exact in fp32; the sum over a block and
// the sum over the blocks are held in fp32, and the result is rounded once, to the output's type.
// Grouped: row block b of block_m rows uses the matrix expert_ids[b], and row r of it the
// activation row sorted_ids[r] / top_k. Rows of an absent expert (id < 0) and padding rows (slot
// >= num_slots) are written as zeros; rows at or past num_tokens_post_padded are left as they
// were. The SiLU form has gate rows [0, inter) and up rows [inter, 2 inter), and quantises
// silu(gate) * up, in fp32, per block of 128 outputs (quant_block.cu's rule).
#include <cuda_bf16.h>

#include "common.cuh"
#include "fp8_block.h"
#include "internal.h"

namespace w4a8 {

namespace {

constexpr int kBlk = 128;
constexpr int kRows = 16;  // rows of a tile; block_m is a multiple
constexpr int kKc = 32;    // columns of w and x staged at a time

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
    if (dtype == 0) static_cast<float*>(out)[i] = v;
    else if (dtype == 1) static_cast<__half*>(out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// One CTA: 16 rows x 128 outputs, thread = (row tid / 16, outputs tid % 16 + 16 j). fp32 FMAs on
// the CUDA cores from staged fp32 copies; it takes every K and every alignment. Bound by the reads
// of the staged copies, 16 a weight value: 1024 x 1024 x 1000 takes 226 us, where the tensor-core
// kernels take 6.2 on the device (8.9 a call) for K = 1024.
template <bool SILU>
__global__ void __launch_bounds__(256) fp8_simple_kernel(const Fp8Args a) {
    constexpr int kNw = SILU ? 256 : 128;  // weight rows of the tile
    __shared__ float wt[kNw][kKc + 1];
    __shared__ float xt[kRows][kKc + 1];
    const int tid = threadIdx.x, row = tid >> 4, c0 = tid & 15;
    const int64_t P_valid = a.ntp ? min((int64_t)a.ntp[0], a.P) : a.P;
    const int64_t inter = a.N / 2;
    const int64_t n0 = (int64_t)blockIdx.x * 128;
    for (int64_t t = blockIdx.y; t * kRows < P_valid; t += gridDim.y) {
        const int64_t r = t * kRows + row;
        const int e = a.expert_ids ? a.expert_ids[t * kRows / a.block_m] : 0;
        int64_t src = -1;
        if (e >= 0 && e < a.E && r < P_valid) {
            const int64_t slot = a.sorted_ids ? a.sorted_ids[r] : r;
            if (!a.sorted_ids) src = slot;
            else if (slot >= 0 && slot < a.num_slots) src = slot / a.top_k;
        }
        float tot[kNw / 16];
#pragma unroll
        for (int j = 0; j < kNw / 16; ++j) tot[j] = 0.f;
        if (e >= 0 && e < a.E) {
            const uint8_t* w = a.w + (int64_t)e * a.N * a.K;
            const float* ws = a.ws + (int64_t)e * ((a.N + kBlk - 1) / kBlk) * a.G;
            for (int64_t g = 0; g < a.G; ++g) {
                float acc[kNw / 16];
#pragma unroll
                for (int j = 0; j < kNw / 16; ++j) acc[j] = 0.f;
                for (int64_t k0 = g * kBlk; k0 < (g + 1) * kBlk && k0 < a.K; k0 += kKc) {
                    __syncthreads();
                    for (int i = tid; i < kNw * kKc; i += 256) {
                        const int m = i / kKc, k = i % kKc;
                        const int64_t n = !SILU ? n0 + m : m < 128 ? n0 + m : inter + n0 + m - 128;
                        wt[m][k] = n < a.N && k0 + k < a.K ? e4m3_to_f32(w[n * a.K + k0 + k]) : 0.f;
                    }
                    for (int k = c0; k < kKc; k += 16)
                        xt[row][k] = src >= 0 && k0 + k < a.K ? e4m3_to_f32(a.x[src * a.K + k0 + k]) : 0.f;
                    __syncthreads();
                    for (int k = 0; k < kKc; ++k) {
                        const float xv = xt[row][k];
#pragma unroll
                        for (int j = 0; j < kNw / 16; ++j) acc[j] += xv * wt[c0 + 16 * j][k];
                    }
                }
                const float sx = src >= 0 ? a.xs[src * a.G + g] : 0.f;
                const float sw = ws[(n0 / kBlk) * a.G + g];
                const float sw_up = SILU ? ws[((inter + n0) / kBlk) * a.G + g] : 0.f;
#pragma unroll
                for (int j = 0; j < kNw / 16; ++j) tot[j] += acc[j] * (sx * (j < 8 ? sw : sw_up));
            }
        }
        if (SILU) {
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // silu by exp(-|gate|), which does not overflow (fp8_tc.cuh: silu_mul2)
                const float gate = tot[j], e = expf(-fabsf(gate));
                const float silu = (gate >= 0.f ? gate : gate * e) / (1.f + e);
                tot[j] = src >= 0 ? silu * tot[(j + 8) % (kNw / 16)] : 0.f;
                amax = fmaxf(amax, fabsf(tot[j]));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float s = __fdiv_rn(fmaxf(amax, kAmaxFloor), kE4m3Max);
            if (r < P_valid) {
                if (c0 == 0) a.qs[r * (inter / kBlk) + n0 / kBlk] = s;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    a.q[r * inter + n0 + c0 + 16 * j] =
                        (uint8_t)f32x2_to_e4m3x2(__fdiv_rn(tot[j], s), 0.f);
            }
        } else if (r < P_valid) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t n = n0 + c0 + 16 * j;
                if (n < a.N) store_out(a.out, a.out_dtype, r * a.N + n, src >= 0 ? tot[j] : 0.f);
            }
        }
    }
}

}  // namespace

int launch_fp8_simple(const Fp8Args& a, cudaStream_t st) {
    const int64_t n = a.silu ? a.N / 2 : a.N;
    const int64_t tiles = (a.P + kRows - 1) / kRows;
    const dim3 grid((unsigned)((n + 127) / 128), (unsigned)(tiles < 32768 ? tiles : 32768));
    if (a.silu) fp8_simple_kernel<true><<<grid, 256, 0, st>>>(a);
    else fp8_simple_kernel<false><<<grid, 256, 0, st>>>(a);
    return launch_status();
}

namespace {

// TMA needs rows of a multiple of 16 bytes from a 16-byte boundary; everything else takes the
// plain kernel.
int run_fp8(const Fp8Args& a, cudaStream_t st) {
    return fp8_tc_ok(a) ? launch_fp8_tc(a, st) : launch_fp8_simple(a, st);
}

// Sizes and routing checks of the two grouped entries; 0 or W4A8_ERR_INVALID.
int check_grouped(const std::string& o, const Fp8Args& a, int64_t top_k, int64_t block_m) {
    if (a.x_rows < 0 || a.E <= 0 || a.N <= 0 || a.K <= 0 || a.P < 0)
        return set_error(o + ": bad sizes");
    if (a.x_rows > INT32_MAX || a.P > INT32_MAX || a.K > INT32_MAX || a.E > INT32_MAX ||
        a.N > INT32_MAX / a.E)
        return set_error(o + ": T, P, K and E * N must be below 2^31");
    if (top_k <= 0 || top_k > INT32_MAX || a.x_rows > INT32_MAX / top_k)
        return set_error(o + ": top_k must be positive and T * top_k below 2^31");
    if (block_m != 16 && block_m != 32 && block_m != 64 &&
        (block_m <= 0 || block_m % 128 != 0 || block_m > INT32_MAX))
        return set_error(o + ": block_m must be 16, 32, 64 or a multiple of 128");
    if (a.P % block_m != 0) return set_error(o + ": P not divisible by block_m");
    if (a.P == 0) return W4A8_OK;
    if (!a.w || !a.ws || !a.expert_ids || !a.ntp || (a.x_rows > 0 && (!a.x || !a.xs)))
        return set_error(o + ": null pointer");
    if (!a.sorted_ids && a.x_rows != a.P)
        return set_error(o + ": without sorted_token_ids x must have P rows");
    return W4A8_OK;
}

}  // namespace

}  // namespace w4a8

using namespace w4a8;

extern "C" int w4a8_fp8_block_gemm(const uint8_t* x, const float* x_scales, const uint8_t* w,
                                   const float* w_scales, void* out, int32_t out_dtype, int64_t M,
                                   int64_t N, int64_t K, w4a8_stream_t stream) {
    const std::string o = "fp8_block_gemm";
    if (out_dtype < 0 || out_dtype > 2)
        return set_error(o + ": out_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
        return set_error(o + ": bad sizes (0 <= M, 1 <= N, 1 <= K, all below 2^31)");
    if (M == 0) return W4A8_OK;
    if (!x || !x_scales || !w || !w_scales || !out) return set_error(o + ": null pointer");
    Fp8Args a{};
    a.x = x;
    a.xs = x_scales;
    a.w = w;
    a.ws = w_scales;
    a.out = out;
    a.out_dtype = out_dtype;
    a.x_rows = a.P = M;
    a.N = N;
    a.K = K;
    a.E = 1;
    a.G = (K + kBlk - 1) / kBlk;
    a.top_k = 1;
    a.block_m = 128;
    return run_fp8(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int w4a8_fp8_block_moe_gemm(const uint8_t* x, const float* x_scales, const uint8_t* w,
                                       const float* w_scales, const int32_t* sorted_token_ids,
                                       const int32_t* expert_ids,
                                       const int32_t* num_tokens_post_padded, void* out,
                                       int32_t out_dtype, int64_t T, int64_t E, int64_t N,
                                       int64_t K, int64_t P, int64_t top_k, int64_t block_m,
                                       w4a8_stream_t stream) {
    const std::string o = "fp8_block_moe_gemm";
    if (out_dtype < 0 || out_dtype > 2)
        return set_error(o + ": out_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    Fp8Args a{};
    a.x = x;
    a.xs = x_scales;
    a.w = w;
    a.ws = w_scales;
    a.sorted_ids = sorted_token_ids;
    a.expert_ids = expert_ids;
    a.ntp = num_tokens_post_padded;
    a.out = out;
    a.out_dtype = out_dtype;
    a.x_rows = T;
    a.P = P;
    a.N = N;
    a.K = K;
    a.E = E;
    if (int rc = check_grouped(o, a, top_k, block_m)) return rc;
    if (P == 0) return W4A8_OK;
    if (!out) return set_error(o + ": null pointer");
    a.G = (K + kBlk - 1) / kBlk;
    a.num_slots = (int)(T * top_k);
    a.top_k = (int)top_k;
    a.block_m = (int)block_m;
    return run_fp8(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int w4a8_fp8_block_moe_gemm1_silu(
    const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales,
    const int32_t* sorted_token_ids, const int32_t* expert_ids,
    const int32_t* num_tokens_post_padded, uint8_t* q, float* q_scales, int64_t T, int64_t E,
    int64_t inter, int64_t K, int64_t P, int64_t top_k, int64_t block_m, w4a8_stream_t stream) {
    const std::string o = "fp8_block_moe_gemm1_silu";
    if (inter <= 0 || inter % kBlk != 0 || inter > INT32_MAX / 2)
        return set_error(o + ": inter must be a multiple of 128");
    Fp8Args a{};
    a.x = x;
    a.xs = x_scales;
    a.w = w;
    a.ws = w_scales;
    a.sorted_ids = sorted_token_ids;
    a.expert_ids = expert_ids;
    a.ntp = num_tokens_post_padded;
    a.q = q;
    a.qs = q_scales;
    a.silu = true;
    a.x_rows = T;
    a.P = P;
    a.N = 2 * inter;
    a.K = K;
    a.E = E;
    if (int rc = check_grouped(o, a, top_k, block_m)) return rc;
    if (P == 0) return W4A8_OK;
    if (!q || !q_scales) return set_error(o + ": null pointer");
    a.G = (K + kBlk - 1) / kBlk;
    a.num_slots = (int)(T * top_k);
    a.top_k = (int)top_k;
    a.block_m = (int)block_m;
    return run_fp8(a, reinterpret_cast<cudaStream_t>(stream));
}
