// fp8_tc.cuh — what the two tensor-core kernels of the block-scaled FP8 products share: tile walk,
// copies, cluster reads, the SiLU and rounding steps, and the epilogue of a row whose partial sums
// are parked in shared memory.
#pragma once

#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "fp8_block.h"
#include "internal.h"
#include "sm100.cuh"
#include "tcgen05.cuh"

namespace w4a8 {
namespace fp8tc {

constexpr int kBlk = 128;
constexpr int kThreads = 384;
constexpr int kFoldWarp0 = 4;  // warps 4 to 11 fold
constexpr int kFoldWarps = 8;
constexpr int kMaxSplit = 8;

struct TcArgs {
    Fp8Args f;
    int split;    // CTAs per cluster
    int n_tiles;  // weight tiles per row block
    int out_vec;  // out's rows are 16-byte aligned
};

template <int N>
struct Ring {
    uint32_t idx = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++idx == N) {
            idx = 0;
            phase ^= 1;
        }
    }
};

// Tiles of one cluster: t = unit + i * units, t = row_block * n_tiles + n_tile.
struct Walk {
    int rb, nt, drb, dnt, n_tiles, blocks;
    __device__ __forceinline__ Walk(int unit, int units, int n_tiles_, int blocks_)
        : rb(unit / n_tiles_), nt(unit % n_tiles_), drb(units / n_tiles_), dnt(units % n_tiles_),
          n_tiles(n_tiles_), blocks(blocks_) {}
    __device__ __forceinline__ bool more() const { return rb < blocks; }
    __device__ __forceinline__ void next() {
        rb += drb;
        nt += dnt;
        if (nt >= n_tiles) {
            nt -= n_tiles;
            ++rb;
        }
    }
};

// A load that stays where it is written: fetched a tile ahead of its use, it would otherwise be
// moved down to it to save a register. Not on the read-only path (ld.global.nc): in a kernel that
// starts early (launch_persistent) the work ahead may write this memory while the kernel is there.
__device__ __forceinline__ float fetch(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ int fetch(const int32_t* p) {
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// True in one lane of a converged warp. The copies, MMAs and commits take uniform operands, and
// behind this condition the compiler need not serialise the lanes to make them so (a comparison
// of the lane number cost 200 cycles for each).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}

// A kernel launched with kEarly (launch_persistent) may start before the stream's work ahead of it
// is done; up to here it touches no memory, and from here on that work has ended.
__device__ __forceinline__ void follow_launch() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, int x,
                                            const int (&y)[4], uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
        "r"(smem_u32(bar))
        : "memory");
}

// Whether a phase is complete, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ void st_cluster(const float* p, uint32_t rank, float v) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float4 ld_cluster(const float* p, uint32_t rank) {
    uint32_t addr;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}

// silu(g) * u of two outputs, g0 and u0 replaced by the results. With e = exp(-|g|), which cannot
// overflow, silu(g) is g / (1 + e) for g >= 0 and g e / (1 + e) below, and u comes last. One reciprocal
// serves both denominators d = 1 + e in (1, 2], 1 / d0 = d1 / (d0 d1): the special-function unit, at 16
// a cycle and SM, is what this step waits for. A NaN's d is cut to 2, so that its neighbour keeps its
// value. Together within 16 units of 2^-24, plus 1.25 |g| of them for g < 0 from the exponential's
// argument; below -87 e is subnormal, each of e and silu within 2^-149, and from -104 on it is 0.
__device__ __forceinline__ void silu_mul2(float& g0, float& g1, float u0, float u1) {
    const float e0 = __expf(-fabsf(g0)), e1 = __expf(-fabsf(g1));
    const float d0 = 1.f + fminf(e0, 1.f), d1 = 1.f + fminf(e1, 1.f);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d0 * d1));
    const float2 g = make_float2(g0 >= 0.f ? g0 : g0 * e0, g1 >= 0.f ? g1 : g1 * e1);
    const float2 h = mul2(mul2(g, mul2(make_float2(d1, d0), make_float2(r, r))), make_float2(u0, u1));
    g0 = h.x;
    g1 = h.y;
}

// Four e4m3 bytes of v / scale, rcp = 1 / scale. The values carry more than the 2^-23 by which the
// product may miss the quotient; the exact quotient's slow path, 32 times inlined, cost 5x the
// whole epilogue in instruction fetches.
__device__ __forceinline__ uint32_t quant4(float v0, float v1, float v2, float v3, float rcp) {
    return (uint32_t)f32x2_to_e4m3x2(v0 * rcp, v1 * rcp) |
           (uint32_t)f32x2_to_e4m3x2(v2 * rcp, v3 * rcp) << 16;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Adds the S parts of a row, `stride` floats apart in this CTA's shared memory (kRemote: at the same
// place in each CTA of the cluster), in rank order, and writes its outputs. A part is W floats (the
// SiLU form: 128 gate, then 128 up); n0: the first output. One warp; lane l has columns 4 l of each
// 128. `dead`: a row of zeros.
template <int W, typename Out, bool kRemote>
__device__ __forceinline__ void finish_row(const Fp8Args& a, bool vec, const float* part, int S, int stride,
                                           int64_t r, int64_t n0, bool dead) {
    const int lane = threadIdx.x & 31;
    float4 sum[W / 128];
#pragma unroll
    for (int c = 0; c < W / 128; ++c) {
        const float* p = part + c * 128 + 4 * lane;
        float4 v[kMaxSplit];
#pragma unroll
        for (int k = 0; k < kMaxSplit; ++k)
            if (k < S) v[k] = kRemote ? ld_cluster(p, k) : *reinterpret_cast<const float4*>(p + k * stride);
        sum[c] = v[0];
#pragma unroll
        for (int k = 1; k < kMaxSplit; ++k)
            if (k < S) {
                sum[c].x += v[k].x;
                sum[c].y += v[k].y;
                sum[c].z += v[k].z;
                sum[c].w += v[k].w;
            }
        if (dead) sum[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if constexpr (std::is_void<Out>::value) {
        const float4 g4 = sum[0], u4 = sum[W / 128 - 1];
        float h[4] = {g4.x, g4.y, g4.z, g4.w};
        silu_mul2(h[0], h[1], u4.x, u4.y);
        silu_mul2(h[2], h[3], u4.z, u4.w);
        float m = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = __fdiv_rn(fmaxf(m, kAmaxFloor), kE4m3Max);
        const int64_t inter = a.N / 2;
        if (lane == 0) a.qs[r * (inter / kBlk) + n0 / kBlk] = s;
        *reinterpret_cast<uint32_t*>(a.q + r * inter + n0 + 4 * lane) =
            quant4(h[0], h[1], h[2], h[3], __frcp_rn(s));
    } else {
#pragma unroll
        for (int c = 0; c < W / 128; ++c) {
            const int64_t n = n0 + c * 128 + 4 * lane;
            const float o[4] = {sum[c].x, sum[c].y, sum[c].z, sum[c].w};
            Out* p = static_cast<Out*>(a.out) + r * a.N + n;
            if constexpr (sizeof(Out) == 4) {
                if (vec && n + 4 <= a.N) {
                    *reinterpret_cast<float4*>(p) = sum[c];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < a.N) p[i] = o[i];
                }
            } else {
                const uint32_t lo = pack2<Out>(o[0], o[1]), hi = pack2<Out>(o[2], o[3]);
                if (vec && n + 4 <= a.N) {
                    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
                } else {
                    uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < a.N) h[i] = (uint16_t)((i < 2 ? lo : hi) >> ((i & 1) * 16));
                }
            }
        }
    }
}

constexpr int kMaxDevices = 64;

inline int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}
// The current device's SM count, asked for once.
inline int sm_count() {
    static std::atomic<int> known[kMaxDevices];
    const int dev = current_device();
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        n = n > 0 ? n : 148;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Tensor maps of both kernels: x rows in boxes of x_box (1: gathered), weight rows as (slab, row,
// byte), a slab being one expert's matrix, or its gate or up half, so that one copy brings a
// tile's gate and up rows.
inline bool make_maps(const Fp8Args& a, int x_box, int w_box, CUtensorMap* tmx, CUtensorMap* tmw) {
    const int64_t slab = a.silu ? a.N / 2 : a.N;
    return make_tma_map_u8(tmx, a.x, (uint64_t)a.x_rows, (uint64_t)a.K, 128, x_box,
                           CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_tma_map_u8_3d(tmw, a.w, (uint64_t)(a.E * a.N / slab), (uint64_t)slab, (uint64_t)a.K,
                              128, a.silu ? 128 : w_box, a.silu ? 2 : 1, CU_TENSOR_MAP_SWIZZLE_128B);
}

// CTAs that share a tile, from the tiles and the K blocks: a cluster of 8 (4) finds room on 15 (33)
// places of the 148 SMs at once, not 18 (37), and a second round costs more than the wider split
// gains (16 tiles of 128 rows x 32 blocks: 16.9 us with 8, 10.0 with 4). Two blocks a CTA at least.
inline int split_for(int64_t tiles, int64_t G) {
    const int sms = sm_count();
    const int room[4] = {sms, sms / 2, sms * 33 / 148, sms * 15 / 148};
    int split = 1;
    for (int i = 1; i < 4; ++i)
        if (tiles <= room[i] && G >= (2 << i)) split = 1 << i;
    return split;
}

inline bool out_vec(const Fp8Args& a) {
    const uintptr_t start = reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.N * (a.out_dtype == 0 ? 4 : 2));
    return start % 16 == 0;
}

// Persistent launch of `tiles` tiles over clusters of t.split CTAs. kEarly: its set-up overlaps the
// end of the stream's work ahead of it, and the next such launch's set-up the end of this one.
template <auto kKernel, bool kEarly, typename... Maps>
int launch_persistent(const TcArgs& t, int64_t tiles, size_t smem, cudaStream_t st, const Maps&... maps) {
    static std::atomic<bool> ready[kMaxDevices];  // this kernel's shared-memory limit is set
    const int dev = current_device();
    cudaError_t e;
    if (!ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        ready[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, std::max(1, sm_count() / t.split)) * t.split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (kEarly) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (t.split > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n++].val.clusterDim = {(unsigned)t.split, 1, 1};
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    e = cudaLaunchKernelEx(&cfg, kKernel, t, maps...);
    return e != cudaSuccess ? (int)e : launch_status();
}

}  // namespace fp8tc
}  // namespace w4a8
