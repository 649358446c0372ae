// gemm_fp8_swap.cu — block-scaled FP8 products for row blocks of up to 64 rows (decode batches, short
// expert runs): the weights on the MMA's M side, the tokens on its N side.
//
// What bounds these is the weight stream, WR rows x 128 bytes a stage. With tokens on the N side an
// MMA costs by their number (M128 x N16 x K32: 50 cycles for 128 weight rows; the other way round
// 147 cycles and 8 times the arithmetic for 256, most of it on rows that do not exist), the
// accumulator is NT columns instead of 256, and the fold and the epilogue shrink with it.
//
// A tile is NT tokens (16, 32 or 64, one row block) x WR weight rows (256: two accumulators, for the
// SiLU form gate and up; or 128). Thread = weight row = tensor-memory lane; per 128-wide block g of K
//     tot[c] += (xs[c, g] * ws[block, g]) * acc[c]
// over its columns (tokens) c, the scale products shared through shared memory by the lanes that
// fetch them. A finished tile is parked in shared memory as [token][weight row] and its rows are
// written by whole warps (fp8_tc.cuh: finish_row).
//
// One persistent CTA per SM, 12 warps: 0 TMA producer (x rows by a 2D box, or by tile::gather4
// through the routing, 4 rows a lane), 1 tensor memory and MMA issue, 2 and 3 write the rows of a
// parked tile while the next is folded (tiles of up to 32 tokens; with the fold warps doing it a
// tile of 4 blocks spent half its time there), 4-11 fold: lane quarter warp % 4, one half of the
// tokens each. With few tiles a cluster of S CTAs shares one along K: token c belongs to CTA c % S,
// every CTA parks its part of it there (distributed shared memory), and after a cluster barrier the
// owner adds the parts in rank order.
//
// Measured: gate_up of 32 tokens over 256 experts (2048 -> 2 x 512, 346 MB) 61 us, 88 % of the
// measured copy bandwidth; down of the same (174 MB) 32.9 us, 82 %: 8.8 tiles a CTA run as 9, and
// padding rows are written too. Dense products of few tiles, replayed from a graph with weights that L2
// does not hold, take 5.7 us (1 x 4096 x 2048), 7.1 (333 x 1001 x 1424) and 8.3 (128 x 2048 x 4096), most
// of it latency: set-up 0.7, first data 0.9, the cluster's join 0.4. The set-up overlaps the end of the
// work ahead in the stream (kEarly); without that they take 6.6, 8.1 and 9.4, and down 33.7 for 32.8.
// Called one by one from Python the same three take 8.9 us each, the host's time for a call.
//
// Waits are bounded as in gemm_fp8_tc.cu: one that gives up leaves NaN in the tile's outputs.
#include "fp8_tc.cuh"

namespace w4a8 {

using namespace fp8tc;

namespace {

template <int NT, int WR>
struct Cfg {
    static constexpr uint32_t kWBytes = WR * 128, kXBytes = NT * 128;
    static constexpr int kSub = WR / 128;      // accumulators per block of K
    static constexpr int kHalf = NT / 2;       // tokens per fold thread
    static constexpr int kAccCols = kSub * NT; // tensor-memory columns of a block of K
    static constexpr int kAcc = 4;
    static constexpr int kPitch = WR + 4;      // floats per token of a parked tile
    static constexpr bool kAside = NT <= 32;   // finished by warps 2 and 3
    static constexpr int kPark = NT * kPitch * 4;
    static constexpr int kFree = 227 * 1024 - 1024 - 2048 - kPark - 2 * kFoldWarps * kSub * kHalf * 4;
    static constexpr int kMost = kFree / (int)(kWBytes + kXBytes);
    // A full memory system is not served faster by more requests, and the scales' own loads queue
    // behind them: down at 32 tokens takes 39.2, 34.8, 34.7 and 36.2 us with 2, 3, 4 and 6 stages of
    // 256 weight rows. Narrow tiles, where a CTA has one, take what there is.
    static constexpr int kCap = WR == 256 ? 4 : 12;
    static constexpr int kStages = kMost < kCap ? kMost : kCap;
    static constexpr uint32_t kTmemCols = kAcc * kAccCols < 32 ? 32 : kAcc * kAccCols;
};

template <int NT, int WR>
struct Smem {
    using C = Cfg<NT, WR>;
    uint8_t ring[C::kStages][C::kWBytes + C::kXBytes];  // 1024-byte aligned
    float park[NT][C::kPitch];
    float scale[2][kFoldWarps][C::kSub][C::kHalf];      // [block parity][warp]: xs * ws of its tokens
    uint64_t full[C::kStages], empty[C::kStages];
    uint64_t tfull[C::kAcc], tempty[C::kAcc];
    uint64_t parked, read;                              // the parked tile, when it is finished aside
    int dead[NT];                                       // tokens whose row is one of zeros
    uint32_t tmem_base;
    int bad;
};

// kHalf columns of this warp's lanes, waited for.
template <int kHalf>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&v)[kHalf]) {
    if constexpr (kHalf == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                       "=r"(v[6]), "=r"(v[7])
                     : "r"(taddr));
    else
#pragma unroll
        for (int j = 0; j < kHalf; j += 16)
            tmem_ld16_nowait(taddr + j, reinterpret_cast<uint32_t(&)[16]>(v[j]));
}
// Keeps the uses of v behind what precedes (the wait for its loads).
template <int kHalf>
__device__ __forceinline__ void pin(uint32_t (&v)[kHalf]) {
#pragma unroll
    for (int j = 0; j < kHalf; j += 8)
        asm volatile("" : "+r"(v[j]), "+r"(v[j + 1]), "+r"(v[j + 2]), "+r"(v[j + 3]), "+r"(v[j + 4]),
                     "+r"(v[j + 5]), "+r"(v[j + 6]), "+r"(v[j + 7]));
}

template <int NT, int WR, typename Out, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_swap_kernel(const TcArgs t, const __grid_constant__ CUtensorMap tmx,
                const __grid_constant__ CUtensorMap tmw) {
    using C = Cfg<NT, WR>;
    constexpr bool SILU = std::is_void<Out>::value;
    extern __shared__ uint8_t smem_raw[];
    Smem<NT, WR>& sm = *reinterpret_cast<Smem<NT, WR>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const Fp8Args& a = t.f;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* bad = &sm.bad;
    const int* some_int = reinterpret_cast<const int*>(a.ws);  // can be read; holds at least one

    const int S = SPLIT ? t.split : 1;
    const int rank = SPLIT ? (int)cluster_rank() : 0;
    const int G = (int)a.G;
    const int g_lo = (int)((int64_t)G * rank / S), g_hi = (int)((int64_t)G * (rank + 1) / S);
    const int n_step = SILU ? 128 : WR;  // outputs per tile
    auto expert_of = [&](int rb) { return a.expert_ids ? fetch(a.expert_ids + rb) : 0; };

    if (tid == 32 * 2) {
        prefetch_map(&tmx);
        prefetch_map(&tmw);
    }
    // The producer sets up its barriers and goes on to its first copies; the others meet when the
    // tensor memory is there too.
    if (warp == 0) {
        if (lane == 0) sm.bad = 0;
        if (lane < C::kStages) {
            mbar_init(&sm.full[lane], 1);
            mbar_init(&sm.empty[lane], 1);
        }
        if (lane < C::kAcc) {
            mbar_init(&sm.tfull[lane], 1);
            mbar_init(&sm.tempty[lane], kFoldWarps);
        }
        if (lane == 0) {
            mbar_init(&sm.parked, kFoldWarps);
            mbar_init(&sm.read, 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem_base)),
                     "r"(C::kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (warp == 0) {
        asm volatile("bar.arrive 8, %0;" ::"n"(kThreads) : "memory");
    } else {
        asm volatile("tcgen05.fence::before_thread_sync;" ::);
        asm volatile("bar.sync 8, %0;" ::"n"(kThreads) : "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::);
    }
    follow_launch();
    const int64_t rows = a.ntp ? max((int64_t)0, min((int64_t)fetch(a.ntp), a.P)) : a.P;
    const int blocks = (int)((rows + NT - 1) / NT);
    const Walk first(blockIdx.x / S, gridDim.x / S, t.n_tiles, blocks);
    if (SPLIT) cluster_arrive();  // awaited before the first part is parked with another CTA

    // One pass runs all of the CTA's tiles; with a split it is one tile, and the cluster meets
    // before the next. Each role keeps its ring positions over the passes.
    Ring<C::kStages> st;
    Ring<C::kAcc> tb;
    uint32_t issued = 0;
    Walk cur = first;
    do {
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            // the routing entries of the tile to enter next are fetched a tile ahead
            int e = -1, slot[4];
            auto look = [&](const Walk& w) {
                if (!w.more()) return;
                e = expert_of(w.rb);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t r = (int64_t)w.rb * NT + 4 * lane + i;
                    slot[i] = a.sorted_ids && 4 * lane < NT && r < rows ? fetch(a.sorted_ids + r) : -1;
                }
            };
            Walk w = cur;
            look(w);
            while (w.more()) {
                const bool present = e >= 0 && e < a.E;
                const int r0 = w.rb * NT, w_row = w.nt * n_step, w_slab = SILU ? 2 * e : e;
                int src[4];  // padding slots read row 0; their columns are dropped at the end
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    src[i] = slot[i] >= 0 && slot[i] < a.num_slots ? slot[i] / a.top_k : 0;
                w.next();
                if (!SPLIT) look(w);
                for (int g = present ? g_lo : g_hi; g < g_hi; ++g) {
                    uint8_t* ws = sm.ring[st.idx];
                    uint8_t* xs = ws + C::kWBytes;
                    uint64_t* fb = &sm.full[st.idx];
                    if (elect_one()) {
                        mbar_wait(&sm.empty[st.idx], st.phase ^ 1, bad);
                        mbar_expect_tx(fb, C::kWBytes + C::kXBytes);
                        tma_load_3d(ws, &tmw, g * 128, w_row, w_slab, fb);
                        if (!a.sorted_ids) tma_load_2d(xs, &tmx, g * 128, r0, fb);
                    }
                    __syncwarp();
                    if (a.sorted_ids && 4 * lane < NT) tma_gather4(xs + lane * 512, &tmx, g * 128, src, fb);
                    st.next();
                    ++issued;
                }
                if (SPLIT) break;
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            if (elect_one()) {
                constexpr uint32_t idesc = umma_idesc(128, NT);
                for (Walk w = cur; w.more(); w.next()) {
                    const int e = expert_of(w.rb);
                    for (int g = e >= 0 && e < a.E ? g_lo : g_hi; g < g_hi; ++g) {
                        mbar_wait(&sm.full[st.idx], st.phase, bad);
                        mbar_wait(&sm.tempty[tb.idx], tb.phase ^ 1, bad);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::);
                        const uint32_t wa = smem_u32(sm.ring[st.idx]);
                        const uint32_t d = sm.tmem_base + tb.idx * C::kAccCols;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint64_t db = desc_sw128(wa + C::kWBytes + kk * 32);
#pragma unroll
                            for (int b = 0; b < C::kSub; ++b) {
                                const uint64_t da = desc_sw128(wa + b * 128 * 128 + kk * 32);
                                asm volatile(
                                    "{\n\t.reg .pred p;\n\t"
                                    "setp.ne.b32 p, %4, 0;\n\t"
                                    "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(
                                        d + b * NT),
                                    "l"(da), "l"(db), "r"(idesc), "r"(kk > 0 ? 1u : 0u));
                            }
                        }
                        asm volatile(
                            "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                            ::"r"(smem_u32(&sm.empty[st.idx])));
                        asm volatile(
                            "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                            ::"r"(smem_u32(&sm.tfull[tb.idx])));
                        st.next();
                        tb.next();
                    }
                    if (SPLIT) break;
                }
            }
            __syncwarp();
        } else if (warp < kFoldWarp0) {
            // ---------------- rows of a parked tile ----------------
            if (C::kAside && !SPLIT) {
                uint32_t turn = 0;
                for (Walk w = cur; w.more(); w.next(), turn ^= 1) {
                    const int64_t r0 = (int64_t)w.rb * NT, n0 = (int64_t)w.nt * n_step;
                    mbar_wait(&sm.parked, turn, bad);
                    for (int c = warp - 2; c < NT && r0 + c < rows; c += 2)
                        finish_row<WR, Out, false>(a, t.out_vec, sm.park[c], 1, 0, r0 + c, n0, sm.dead[c] != 0);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.read);
                }
                __syncwarp();
            }
        } else {
            // ---------------- fold + epilogue ----------------
            const int q = warp & 3, fw = warp - kFoldWarp0, half = fw >> 2;
            const int wrow = q * 32 + lane;                // weight row within a 128-row accumulator
            const int token = half * C::kHalf + lane;      // whose scale this lane fetches
            const bool fetches = lane < C::kHalf;
            const int64_t NB = (a.N + kBlk - 1) / kBlk;
            // With the weights streaming, a load from memory takes as long as a short tile: a tile's
            // first scales are fetched one tile ahead, its routing entries two. The fetches are
            // unconditional (from some address that can be read, where there is nothing to fetch),
            // since a value merged behind a branch is waited for at the merge.
            struct Scales {
                const float *xs, *ws0, *ws1;  // this lane's token's, and its weight blocks'
                float x, w0, w1;              // of the next block of K
                bool present, dead;
            };
            Scales now, ahead;
            uint32_t turn = 0;  // phase of the parked tile
            int next_e = -1, next_slot = -1;
            auto row_of = [&](const Walk& w) { return (int64_t)w.rb * NT + token; };
            auto look = [&](const Walk& w) {
                const int64_t r = row_of(w);
                next_e = fetch(a.expert_ids && w.more() ? a.expert_ids + w.rb : some_int);
                next_slot = fetch(a.sorted_ids && fetches && r < rows ? a.sorted_ids + r : some_int);
            };
            auto enter = [&](const Walk& w, Scales& s) {
                const int e = a.expert_ids ? next_e : 0;
                s.present = w.more() && e >= 0 && e < a.E && g_lo < g_hi;
                const int64_t r = row_of(w);
                int src = fetches && r < rows ? (a.sorted_ids ? next_slot : (int)r) : -1;
                if (a.sorted_ids) src = src >= 0 && src < a.num_slots ? src / a.top_k : -1;
                s.dead = !s.present || src < 0;
                const int64_t b0 = (int64_t)w.nt * n_step / kBlk;
                const float* ws = a.ws + (s.present ? e * NB * G : 0);
                s.xs = a.xs + (s.dead ? 0 : src * (int64_t)G);
                s.ws0 = ws + (s.present ? b0 * G : 0);
                s.ws1 = ws + (s.present ? (SILU ? b0 + a.N / 2 / kBlk : min(b0 + 1, NB - 1)) * G : 0);
                s.x = fetch(s.xs + g_lo);
                s.w0 = fetch(s.ws0 + g_lo);
                s.w1 = C::kSub == 2 ? fetch(s.ws1 + g_lo) : 0.f;
                for (int g = g_lo + 8; g < g_hi; g += 8) {  // 32 bytes at a time
                    if (fetches) prefetch_l2(s.xs + g);
                    if (lane == 0) prefetch_l2(s.ws0 + g);
                    if (C::kSub == 2 && lane == 0) prefetch_l2(s.ws1 + g);
                }
            };
            Walk w = cur, w1 = cur;  // the tile, and the next
            look(w);
            enter(w, now);
            w1.next();
            if (!SPLIT) look(w1);
            while (w.more()) {
                const int64_t r0 = (int64_t)w.rb * NT, n0 = (int64_t)w.nt * n_step;
                const bool is_dead = now.dead;
                w = w1;
                if (!SPLIT) {
                    enter(w, ahead);
                    w1.next();
                    look(w1);
                }
                float tot[C::kSub][C::kHalf];
#pragma unroll
                for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                    for (int c = 0; c < C::kHalf; ++c) tot[b][c] = 0.f;
                if (now.present) {
#pragma unroll 1
                    for (int g = g_lo; g < g_hi; ++g) {
                        float(&sc)[C::kSub][C::kHalf] = sm.scale[g & 1][fw];
                        if (fetches) {
                            sc[0][lane] = now.x * now.w0;
                            if (C::kSub == 2) sc[C::kSub - 1][lane] = now.x * now.w1;
                        }
                        const int next_g = min(g + 1, g_hi - 1);  // behind this block's fold
                        now.x = fetch(now.xs + next_g);
                        now.w0 = fetch(now.ws0 + next_g);
                        if (C::kSub == 2) now.w1 = fetch(now.ws1 + next_g);
                        __syncwarp();
                        mbar_wait(&sm.tfull[tb.idx], tb.phase, bad);
                        __syncwarp();
                        asm volatile("tcgen05.fence::after_thread_sync;" ::);
                        const uint32_t base =
                            sm.tmem_base + ((uint32_t)(q * 32) << 16) + tb.idx * C::kAccCols + half * C::kHalf;
                        uint32_t v[C::kSub][C::kHalf];
#pragma unroll
                        for (int b = 0; b < C::kSub; ++b) tmem_load(base + b * NT, v[b]);
                        tmem_wait_ld();
#pragma unroll
                        for (int b = 0; b < C::kSub; ++b) pin(v[b]);
                        asm volatile("tcgen05.fence::before_thread_sync;" ::);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.tempty[tb.idx]);
                        tb.next();
#pragma unroll
                        for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                            for (int c = 0; c < C::kHalf; c += 4) {
                                const float4 f = *reinterpret_cast<const float4*>(&sc[b][c]);
                                const float2 p0 = ffma2(make_float2(__uint_as_float(v[b][c]), __uint_as_float(v[b][c + 1])),
                                                        make_float2(f.x, f.y), make_float2(tot[b][c], tot[b][c + 1]));
                                const float2 p1 = ffma2(make_float2(__uint_as_float(v[b][c + 2]), __uint_as_float(v[b][c + 3])),
                                                        make_float2(f.z, f.w), make_float2(tot[b][c + 2], tot[b][c + 3]));
                                tot[b][c] = p0.x;
                                tot[b][c + 1] = p0.y;
                                tot[b][c + 2] = p1.x;
                                tot[b][c + 3] = p1.y;
                            }
                    }
                }
                const float poison = *bad ? __int_as_float(0x7fffffff) : 0.f;
                if constexpr (SPLIT) {
                    __syncwarp();
                    cluster_wait();
                    if (q == 0 && fetches) sm.dead[token] = is_dead;
#pragma unroll
                    for (int c = 0; c < C::kHalf; ++c) {
                        const int tok = half * C::kHalf + c, owner = tok & (S - 1);
#pragma unroll
                        for (int b = 0; b < C::kSub; ++b)
                            st_cluster(&sm.park[tok - owner + rank][b * 128 + wrow], owner, tot[b][c] + poison);
                    }
                    break;
                }
                // park the tile once the rows of the one before are written
                if (C::kAside) {
                    mbar_wait(&sm.read, turn ^ 1, bad);
                    turn ^= 1;
                } else {
                    asm volatile("bar.sync 1, %0;" ::"n"(kFoldWarps * 32) : "memory");
                }
                if (q == 0 && fetches) sm.dead[token] = is_dead;
#pragma unroll
                for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                    for (int c = 0; c < C::kHalf; ++c)
                        sm.park[half * C::kHalf + c][b * 128 + wrow] = tot[b][c] + poison;
                if (C::kAside) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.parked);
                } else {
                    asm volatile("bar.sync 2, %0;" ::"n"(kFoldWarps * 32) : "memory");
                    for (int c = fw; c < NT && r0 + c < rows; c += kFoldWarps)
                        finish_row<WR, Out, false>(a, t.out_vec, sm.park[c], 1, 0, r0 + c, n0, sm.dead[c] != 0);
                }
                if (!SPLIT) now = ahead;
            }
            __syncwarp();
        }
        if (SPLIT) {
            // the first wait is the parking warps' own; a cluster without a tile has none of them
            if (warp < kFoldWarp0 || !cur.more()) cluster_wait();
            cluster_sync();
            if (warp >= kFoldWarp0 && cur.more()) {
                const int64_t r0 = (int64_t)cur.rb * NT, n0 = (int64_t)cur.nt * n_step;
                for (int c = rank + S * (warp - kFoldWarp0); c < NT && r0 + c < rows; c += S * kFoldWarps)
                    finish_row<WR, Out, false>(a, t.out_vec, sm.park[c - rank], S, C::kPitch, r0 + c, n0,
                                               sm.dead[c] != 0);
            }
            cur.next();
            if (cur.more()) cluster_arrive();  // this tile is read: awaited before the next is parked
        }
    } while (SPLIT && cur.more());
    // after a wait that gave up: leave no copy in flight
    if (tid == 0 && *bad) {
        const uint64_t t0 = global_ns();
        for (uint32_t j = 0; j < (uint32_t)C::kStages && j < issued; ++j)
            while (!mbar_try(&sm.full[j], ((issued - 1 - j) / C::kStages) & 1) &&
                   global_ns() - t0 < kWaitLimitNs) {
            }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::);
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem_base), "r"(C::kTmemCols));
    }
}

template <int NT, int WR, typename Out, bool SPLIT>
int launch_t(const TcArgs& t, int64_t tiles, cudaStream_t st) {
    static_assert(sizeof(Smem<NT, WR>) + 1024 <= 227 * 1024, "shared memory");
    CUtensorMap tmx, tmw;
    if (!make_maps(t.f, t.f.sorted_ids ? 1 : NT, WR, &tmx, &tmw))
        return set_error("fp8_block: tensor map encoding failed");
    return launch_persistent<fp8_swap_kernel<NT, WR, Out, SPLIT>, true>(
        t, tiles, sizeof(Smem<NT, WR>) + 1024, st, tmx, tmw);
}

template <int NT, typename Out>
int launch_out(const TcArgs& t, bool wide, int64_t tiles, cudaStream_t st) {
    if constexpr (std::is_void<Out>::value)
        return t.split > 1 ? launch_t<NT, 256, Out, true>(t, tiles, st)
                           : launch_t<NT, 256, Out, false>(t, tiles, st);
    else if (wide)
        return launch_t<NT, 256, Out, false>(t, tiles, st);
    else
        return t.split > 1 ? launch_t<NT, 128, Out, true>(t, tiles, st)
                           : launch_t<NT, 128, Out, false>(t, tiles, st);
}

template <int NT>
int launch_nt(TcArgs t, cudaStream_t st) {
    const Fp8Args& a = t.f;
    // row blocks that can hold work: with routing, at most one per slot
    int64_t blocks = (a.P + NT - 1) / NT;
    if (a.sorted_ids) blocks = std::min<int64_t>(blocks, a.num_slots);
    const int64_t n = a.silu ? a.N / 2 : a.N;
    const int64_t tiles256 = blocks * ((n + (a.silu ? 127 : 255)) / (a.silu ? 128 : 256));
    const int64_t tiles128 = blocks * ((n + 127) / 128);
    const bool wide = a.silu || tiles256 >= sm_count();
    const int64_t tiles = wide ? tiles256 : tiles128;
    t.n_tiles = (int)(tiles / blocks);
    t.split = split_for(tiles, a.G);
    if (a.silu) return launch_out<NT, void>(t, wide, tiles, st);
    switch (a.out_dtype) {
        case 0: return launch_out<NT, float>(t, wide, tiles, st);
        case 1: return launch_out<NT, __half>(t, wide, tiles, st);
        default: return launch_out<NT, __nv_bfloat16>(t, wide, tiles, st);
    }
}

}  // namespace

int launch_fp8_swap(const Fp8Args& a, cudaStream_t st) {
    TcArgs t{};
    t.f = a;
    t.out_vec = out_vec(a);
    const int64_t rows = a.expert_ids ? a.block_m : a.P;
    if (rows <= 16) return launch_nt<16>(t, st);
    return rows <= 32 ? launch_nt<32>(t, st) : launch_nt<64>(t, st);
}

}  // namespace w4a8
