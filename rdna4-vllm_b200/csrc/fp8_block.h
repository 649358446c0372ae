// fp8_block.h — arguments of the block-scaled FP8 products, shared by the launchers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace w4a8 {

struct Fp8Args {
    const uint8_t* x;           // (x_rows, K) e4m3
    const float* xs;            // (x_rows, G)
    const uint8_t* w;           // (E, N, K) e4m3; N = 2 * inter, [gate | up], for the SiLU form
    const float* ws;            // (E, ceil(N / 128), G)
    const int32_t* sorted_ids;  // (P,) slot of each row, or null: row r reads x's row r
    const int32_t* expert_ids;  // (P / block_m,), or null: one matrix for all rows
    const int32_t* ntp;         // rows in use, or null: all P
    void* out;                  // (P, N), or null for the SiLU form
    uint8_t* q;                 // SiLU form: (P, N / 2) e4m3
    float* qs;                  // SiLU form: (P, N / 256)
    int64_t x_rows, P, N, K, E, G;
    int num_slots, top_k, block_m;
    int out_dtype;              // 0 fp32, 1 fp16, 2 bf16
    bool silu;
};

int launch_fp8_simple(const Fp8Args& a, cudaStream_t st);
bool fp8_tc_ok(const Fp8Args& a);  // sizes and alignment that the tensor-core kernel takes
int launch_fp8_tc(const Fp8Args& a, cudaStream_t st);
int launch_fp8_swap(const Fp8Args& a, cudaStream_t st);  // its form for blocks of up to 64 rows

}  // namespace w4a8
