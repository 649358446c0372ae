// gemm_fp8_tc.cu — block-scaled FP8 products on the 5th-generation tensor cores.
//
// The kernel for blocks of more than 64 rows (fewer: gemm_fp8_swap.cu). A tile is 128 activation
// rows (the MMA's M side: row = tensor-memory lane) times BN weight rows (its N side). Per 128-wide
// block g of K the tensor core returns acc = x_g w_g^T, and the fold adds it to fp32 registers with
// one scalar per thread,
//     tot[n] += (xs[row, g] * ws[n / 128, g]) * acc[n],
// because a thread owns one row and the columns of one weight-scale block (two for the SiLU form,
// gate and up).
//
// One persistent CTA per SM, 12 warps:
//   warp 0     TMA producer: per stage one 128-byte column slab of the tile's x rows and of BN
//              weight rows, in the 128-byte swizzle that the MMA's K-major descriptors read.
//   warp 1     owns tensor memory; one thread issues 4 x tcgen05.mma.kind::f8f6f4 (K = 32) per
//              block into a ring of fp32 accumulators (512 / BN of them).
//   warps 2, 3 copy the x rows of routed tiles with cp.async instead; warp 3 sends finished 16- and
//              32-bit outputs by TMA.
//   warps 4-11 fold: lane quarter warp % 4, one half of the columns each; then the epilogue. They
//              take registers that the first four warps give back (setmaxnreg: 128 x 64 + 256 x 216
//              = 63,488 of the 384 x 168 = 64,512 that the block was launched with).
//
// When there are fewer tiles than SMs, a cluster of S CTAs shares a tile: each takes a slice of
// the K blocks, parks its fp32 partial tile in shared memory, and after a cluster barrier CTA r
// sums rows r, r + S, ... over the cluster in rank order (distributed shared memory), so the
// result does not depend on timing.
//
// What bounds it: the 1000 W power cap, which takes the clock to 1.6 GHz and below in long runs.
// 8192 x 8192 x 2048 takes 160 us, 1.72 PFLOP/s; gate_up of 4096 tokens over 256 experts (2048 -> 2 x
// 512) 151 us, down of the same 95. In cycles a block of a 128 x 256 tile takes 930: MMA 590, to
// the fold and back 570, fold 400, over two accumulators, while its 48 KB come from L2 in 770 to 840.
// Waits that poll rather than suspend make the way shorter and the runs 3 % longer. A pair of CTAs on
// a tile of 256 x 256 (cta_group::2, 32 KB a block) was slower, 197 us against 173 for the first at
// that point: with a fold after every block only two accumulators fit, and the way from MMA to both
// CTAs' folds and back is 2400 cycles. Two MMAs of 128 columns with barriers of their own read x twice
// from shared memory: 168 us.
//
// Every mbarrier wait is bounded (sm100.cuh). When one gives up, the CTA stops waiting, waits
// (boundedly) for its own copies in flight, writes NaN to the tile's outputs and frees tensor
// memory.
#include "fp8_tc.cuh"

namespace w4a8 {

using namespace fp8tc;

namespace {

constexpr int kRows = 128;  // rows of a tile

// kStaged: outputs leave by TMA from a staging area (not the SiLU form's bytes, nor a split tile).
template <int BN, bool kStaged>
struct Cfg {
    static constexpr uint32_t kABytes = kRows * 128;  // a stage's x slab
    static constexpr uint32_t kBBytes = BN * 128;
    static constexpr int kStages = BN == 256 ? (kStaged ? 3 : 4) : 6;
    static constexpr int kAcc = 512 / BN;
    static constexpr int kCols = BN / 2;   // columns per fold thread
    static constexpr int kLines = kCols / 64;  // 128-byte lines that a warp's staging area holds
    static constexpr int kPitch = BN + 4;  // floats per row of a parked partial tile
};

template <int BN, bool kStaged>
struct Smem {
    using C = Cfg<BN, kStaged>;
    uint8_t ring[C::kStages][C::kABytes + C::kBBytes];  // 1024-byte aligned
    // finished outputs: [column half][line][row] x 128 bytes, 16-byte chunks XORed with row % 8
    uint8_t stage_out[kStaged ? 2 : 0][C::kLines][kRows * 128];
    float amax[kStaged ? 0 : 2][2][kRows];  // SiLU form: row maxima, [tile parity][column half]
    uint64_t full[C::kStages], empty[C::kStages];
    uint64_t tfull[C::kAcc], tempty[C::kAcc];
    uint64_t ofull[2 * C::kLines], ofree[2 * C::kLines];  // staged lines
    int src[kRows];  // x's rows of the gather warps' tile, -1 for none
    uint32_t tmem_base;
    int bad;
    static_assert(kRows * C::kPitch * 4 <= sizeof(ring), "a partial tile fits the ring");
};
static_assert(sizeof(Smem<256, true>) + 1024 <= 227 * 1024, "shared memory");
static_assert(sizeof(Smem<256, false>) + 1024 <= 227 * 1024, "shared memory");
static_assert(sizeof(Smem<128, true>) + 1024 <= 227 * 1024, "shared memory");

// Waits for the loads into v; the operands keep every use of v behind the wait.
__device__ __forceinline__ void tmem_wait16(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                   "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                   "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}

// One block's accumulator into the running totals: columns col(0..kCols) at `base`, the first half
// scaled by f0 and the second by f1; released() runs when the last columns are in registers.
template <int kCols, typename Col, typename Done>
__device__ __forceinline__ void fold_block(uint32_t base, Col col, float f0, float f1,
                                           float (&tot)[kCols], Done released) {
    uint32_t v[2][16];
    tmem_ld16_nowait(base + col(0), v[0]);
    tmem_wait16(v[0]);
#pragma unroll
    for (int j = 0; j < kCols; j += 16) {
        uint32_t(&now)[16] = v[(j / 16) & 1];
        uint32_t(&next)[16] = v[(j / 16 + 1) & 1];
        if (j + 16 < kCols) tmem_ld16_nowait(base + col(j + 16), next);
        else released();
        const float f = j < kCols / 2 ? f0 : f1;
        const float2 f2 = make_float2(f, f);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float2 acc = make_float2(__uint_as_float(now[i]), __uint_as_float(now[i + 1]));
            const float2 p = ffma2(acc, f2, make_float2(tot[j + i], tot[j + i + 1]));
            tot[j + i] = p.x;
            tot[j + i + 1] = p.y;
        }
        if (j + 16 < kCols) tmem_wait16(next);
    }
}

// 32 bytes of one row.
__device__ __forceinline__ void store32(void* p, const uint32_t (&u)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(smem_u32(src))
                 : "memory");
}

// A warp's 32 rows of a staged line to the first `count` rows from r_first on, columns n_first on,
// by plain stores: tiles that TMA cannot store whole, and rows that are not 16-byte aligned.
template <int size>
__device__ __noinline__ void send_line(const Fp8Args& a, bool aligned, const uint8_t* so,
                                       int64_t r_first, int count, int n_first) {
    constexpr int per = 16 / size;
    const int lane = threadIdx.x & 31, r = lane >> 3;
    const int n = n_first + (lane & 7) * per;
    uint8_t* p = static_cast<uint8_t*>(a.out) + ((r_first + r) * a.N + n) * size;
    for (int rr = r; rr < count; rr += 4, p += 4 * a.N * size) {
        const uint4 v = *reinterpret_cast<const uint4*>(so + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
        if (n >= a.N) continue;
        if (aligned) {
            *reinterpret_cast<uint4*>(p) = v;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(&v);
            const int left = (int)min((int64_t)per, a.N - n) * size / 2;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < left) reinterpret_cast<uint16_t*>(p)[k] = h[k];
        }
    }
}

// Out: the output's type; void selects the SiLU form.
template <int BN, typename Out, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_tc_kernel(const TcArgs t, const __grid_constant__ CUtensorMap tmx,
              const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmo) {
    constexpr bool SILU = std::is_void<Out>::value;
    constexpr bool kStaged = !SILU && !SPLIT;
    using C = Cfg<BN, kStaged>;
    extern __shared__ uint8_t smem_raw[];
    Smem<BN, kStaged>& sm = *reinterpret_cast<Smem<BN, kStaged>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const Fp8Args& a = t.f;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* bad = &sm.bad;

    const int S = SPLIT ? t.split : 1;
    const int rank = SPLIT ? (int)cluster_rank() : 0;
    const int64_t rows = a.ntp ? max((int64_t)0, min((int64_t)a.ntp[0], a.P)) : a.P;
    const int blocks = (int)((rows + kRows - 1) / kRows);
    const int per_expert = a.expert_ids ? a.block_m / kRows : 1;
    const int G = (int)a.G;
    const int g_lo = (int)((int64_t)G * rank / S), g_hi = (int)((int64_t)G * (rank + 1) / S);
    const int n_step = SILU ? 128 : BN;                    // outputs per tile
    // rows in routing order come by the gather warps' copies (128 rows of tile::gather4 took 2300
    // cycles of issue a stage, three times the MMAs)
    const bool copy_rows = a.sorted_ids != nullptr;
    constexpr int kGatherWarps = kStaged ? 1 : 2;  // warp 3 then sends the outputs
    // tiles whose 128 rows TMA may store: the rows past the last one in use are not ours
    auto tma_out = [&](int rb) { return t.out_vec && (!a.ntp || (int64_t)(rb + 1) * kRows <= rows); };
    constexpr int kOutSize = SILU ? 1 : sizeof(std::conditional_t<SILU, char, Out>);
    constexpr int kLineCols = 128 / kOutSize;                      // columns of a staged line
    constexpr int kRounds = C::kCols / (C::kLines * kLineCols);    // staging areas per tile
    const Walk first(blockIdx.x / S, gridDim.x / S, t.n_tiles, blocks);
    // expert of w's row block, fetched without a branch (a value merged behind one is waited for at
    // the merge); no expert where there is no such tile
    const int* some_int = reinterpret_cast<const int*>(a.ws);  // can be read; holds at least one
    auto fetch_expert = [&](const Walk& w) {
        return fetch(a.expert_ids && w.more() ? a.expert_ids + w.rb / per_expert : some_int);
    };
    auto expert = [&](int fetched) { return a.expert_ids ? fetched : 0; };

    if (tid == 32 * 2) {
        prefetch_map(&tmx);
        prefetch_map(&tmw);
    }
    // The producer sets up its barriers and goes on to its first copies; the others meet when the
    // tensor memory is there too.
    if (warp == 0) {
        if (lane == 0) sm.bad = 0;
        if (lane < C::kStages) {
            mbar_init(&sm.full[lane], copy_rows ? 1 + 32 * kGatherWarps : 1);
            mbar_init(&sm.empty[lane], 1);
        }
        if (lane < C::kAcc) {
            mbar_init(&sm.tfull[lane], 1);
            mbar_init(&sm.tempty[lane], kFoldWarps);
        }
        if (lane < 2 * C::kLines) {
            mbar_init(&sm.ofull[lane], 4);  // the four lane quarters
            mbar_init(&sm.ofree[lane], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem_base)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (warp == 0) {
        asm volatile("bar.arrive 8, %0;" ::"n"(kThreads) : "memory");
    } else {
        asm volatile("tcgen05.fence::before_thread_sync;" ::);
        asm volatile("bar.sync 8, %0;" ::"n"(kThreads) : "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::);
    }

    // One pass runs all of the CTA's tiles, every role at its own pace; with a split it is one tile,
    // and the cluster meets before the next. Each role keeps its ring positions over the passes.
    uint32_t issued = 0;
    Walk cur = first;
    if (warp < kFoldWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        Ring<C::kStages> st;
        Ring<C::kAcc> tb;
        do {
            if (warp == 0) {
                // ---------------- TMA producer ----------------
                const uint32_t stage_bytes = (copy_rows ? 0u : (uint32_t)kRows * 128) + C::kBBytes;
                Walk w = cur;
                int next_e = fetch_expert(w);
                while (w.more()) {
                    const int e = expert(next_e), r0 = w.rb * kRows, w_row = w.nt * n_step, w_slab = SILU ? 2 * e : e;
                    w.next();
                    if (!SPLIT) next_e = fetch_expert(w);
                    for (int g = e >= 0 && e < a.E ? g_lo : g_hi; g < g_hi; ++g) {
                        uint8_t* xa = sm.ring[st.idx];
                        uint64_t* fb = &sm.full[st.idx];
                        if (elect_one()) {
                            mbar_wait(&sm.empty[st.idx], st.phase ^ 1, bad);
                            mbar_expect_tx(fb, stage_bytes);
                            uint8_t* wb = xa + C::kABytes;
                            tma_load_3d(wb, &tmw, g * 128, w_row, w_slab, fb);
                            if (!a.sorted_ids) tma_load_2d(xa, &tmx, g * 128, r0, fb);
                        }
                        __syncwarp();
                        st.next();
                        ++issued;
                    }
                    if (SPLIT) break;
                }
                __syncwarp();
            } else if (warp == 1) {
                // ---------------- MMA issuer ----------------
                if (elect_one()) {
                    constexpr uint32_t idesc = umma_idesc(128, BN);
                    bool full = false, room = false;  // the next block's barriers were seen complete
                    Walk w = cur;
                    int next_e = fetch_expert(w);
                    while (w.more()) {
                        const int e = expert(next_e);
                        w.next();
                        if (!SPLIT) next_e = fetch_expert(w);
                        for (int g = e >= 0 && e < a.E ? g_lo : g_hi; g < g_hi; ++g) {
                            if (!full) mbar_wait(&sm.full[st.idx], st.phase, bad);
                            // the copied rows were written by the generic proxy, the MMA reads by the other
                            if (copy_rows) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            if (!room) mbar_wait(&sm.tempty[tb.idx], tb.phase ^ 1, bad);
                            asm volatile("tcgen05.fence::after_thread_sync;" ::);
                            const uint32_t xa = smem_u32(sm.ring[st.idx]);
                            const uint32_t d = sm.tmem_base + tb.idx * BN;
                            const uint32_t stage_done = smem_u32(&sm.empty[st.idx]);
                            const uint32_t acc_done = smem_u32(&sm.tfull[tb.idx]);
                            st.next();
                            tb.next();
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                // while MMAs are queued, a look at the next block's barriers is free
                                if (kk == 3) {
                                    full = mbar_test(&sm.full[st.idx], st.phase);
                                    room = mbar_test(&sm.tempty[tb.idx], tb.phase ^ 1);
                                }
                                const uint64_t da = desc_sw128(xa + kk * 32);
                                const uint64_t db = desc_sw128(xa + C::kABytes + kk * 32);
                                asm volatile(
                                    "{\n\t.reg .pred p;\n\t"
                                    "setp.ne.b32 p, %4, 0;\n\t"
                                    "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                                    "l"(da), "l"(db), "r"(idesc), "r"(kk > 0 ? 1u : 0u));
                            }
                            asm volatile(
                                "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                                ::"r"(stage_done));
                            asm volatile(
                                "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                                ::"r"(acc_done));
                        }
                        if (SPLIT) break;
                    }
                }
                __syncwarp();
            } else if (kStaged && warp == 3) {
                // ---------------- output warp: staged lines, 64 x 128 outputs a copy ----------------
                // (a TMA store costs its thread some 500 cycles; the fold warps have none to spare)
                if (lane < 2 * C::kLines) {
                    const int half = lane / C::kLines, line = lane % C::kLines;
                    int turn = 0;
                    for (Walk w = cur; w.more(); w.next()) {
                        if (!tma_out(w.rb)) continue;
                        for (int i = 0; i < kRounds; ++i, turn ^= 1) {
                            const int n = w.nt * n_step + half * C::kCols + (i * C::kLines + line) * kLineCols;
                            mbar_wait(&sm.ofull[lane], turn, bad);
                            if (n < a.N)
                                tma_store_2d(&tmo, n * kOutSize, w.rb * kRows, sm.stage_out[half][line]);
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                            mbar_arrive(&sm.ofree[lane]);
                        }
                    }
                    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
                }
                __syncwarp();
            } else if (copy_rows) {
                // ---------------- gather warps: x rows in routing order ----------------
                // Lane l copies 16-byte chunk l % 8 of rows (l / 8) + 4 (warp index) + 8 i; the stage's
                // barrier hears from each lane when its copies have arrived.
                constexpr int kRowsPer = kRows / (4 * kGatherWarps);
                const int chunk = lane & 7, row0 = (warp - 2) * 4 + (lane >> 3);
                // the routing entries of the tile to enter next, fetched a tile ahead: lane l
                // holds this warp's rows l, l + 32, ...: row groups of 4 are dealt to the warps
                constexpr int kSlots = 4 / kGatherWarps;
                int slot[kSlots], e = -1;
                auto row_of = [&](int i) { return (i >> 2) * 4 * kGatherWarps + (warp - 2) * 4 + (i & 3); };
                auto look = [&](const Walk& w) {
                    e = fetch_expert(w);
#pragma unroll
                    for (int i = 0; i < kSlots; ++i) {
                        const int64_t r = (int64_t)w.rb * kRows + row_of(lane + 32 * i);
                        slot[i] = fetch(r < rows ? a.sorted_ids + r : some_int);
                    }
                };
                Walk w = cur;
                look(w);
                while (w.more()) {
                    const bool present = expert(e) >= 0 && expert(e) < a.E;
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < kSlots; ++i)
                        sm.src[row_of(lane + 32 * i)] =
                            (int64_t)w.rb * kRows + row_of(lane + 32 * i) < rows && slot[i] >= 0 &&
                                    slot[i] < a.num_slots
                                ? slot[i] / a.top_k
                                : -1;
                    __syncwarp();
                    int src[kRowsPer <= 16 ? kRowsPer : 1];  // or from shared memory each time
                    if (kRowsPer <= 16)
#pragma unroll
                        for (int i = 0; i < kRowsPer; ++i)
                            src[i % (kRowsPer <= 16 ? kRowsPer : 1)] = sm.src[row0 + i * 4 * kGatherWarps];
                    w.next();
                    if (!SPLIT) look(w);
                    if (!present) {
                        if (SPLIT) break;
                        continue;
                    }
                    for (int g = g_lo; g < g_hi; ++g) {
                        mbar_wait(&sm.empty[st.idx], st.phase ^ 1, bad);
                        const int64_t k = (int64_t)g * kBlk + chunk * 16;
                        const uint32_t xa = smem_u32(sm.ring[st.idx]);
#pragma unroll
                        for (int i = 0; i < kRowsPer; ++i) {
                            const int tr = row0 + i * 4 * kGatherWarps;
                            // absent rows and columns past K are written as zeros (source size 0)
                            const int sr = kRowsPer <= 16 ? src[i % (kRowsPer <= 16 ? kRowsPer : 1)] : sm.src[tr];
                            const bool ok = sr >= 0 && k < a.K;
                            const uint8_t* p = a.x + (ok ? (int64_t)sr * a.K + k : 0);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                             xa + tr * 128 + ((chunk ^ (tr & 7)) << 4)),
                                         "l"(p), "r"(ok ? 16 : 0)
                                         : "memory");
                        }
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                                         smem_u32(&sm.full[st.idx]))
                                     : "memory");
                        st.next();
                    }
                    if (SPLIT) break;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
            }
            if (SPLIT) {
                cluster_sync();
                cluster_sync();
                cur.next();
            }
        } while (SPLIT && cur.more());
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const uint32_t tmem = sm.tmem_base;
        Ring<C::kAcc> tb;
        do {
            // ---------------- fold + epilogue ----------------
            const int q = warp & 3, fw = warp - kFoldWarp0, half = fw >> 2;
            const int row = q * 32 + lane;
            // column of tot[j]: the plain form's half is contiguous; the SiLU form's holds 64
            // gate columns, then the 64 matching up columns
            auto col = [&](int j) {
                return SILU ? (j < 64 ? half * 64 + j : 128 + half * 64 + j - 64) : half * C::kCols + j;
            };
            const int64_t NB = (a.N + kBlk - 1) / kBlk;
            int done = 0, turn = 0;  // turn: phase of the staging area
            // Scales are fetched a block of K ahead, over the tiles' borders, routing entries a whole
            // tile ahead. The fetches are unconditional, see fetch_expert.
            const float *xs = a.xs, *ws0 = a.ws, *ws1 = a.ws;
            bool present = false, dead = true;  // of the tile that enter() was given
            int next_e = -1, next_slot = -1;    // of the tile to enter next
            auto look = [&](const Walk& w) {
                const int64_t r = (int64_t)w.rb * kRows + row;
                next_e = fetch_expert(w);
                next_slot = fetch(a.sorted_ids && r < rows ? a.sorted_ids + r : some_int);
            };
            auto enter = [&](const Walk& w) {
                const int e = expert(next_e);
                const int64_t r = (int64_t)w.rb * kRows + row;
                present = w.more() && e >= 0 && e < a.E && g_lo < g_hi;
                int src = r < rows ? (a.sorted_ids ? next_slot : (int)r) : -1;
                if (a.sorted_ids) src = src >= 0 && src < a.num_slots ? src / a.top_k : -1;
                dead = !present || src < 0;
                const int64_t n0 = (int64_t)w.nt * n_step;
                const int64_t b0 = SILU ? n0 / kBlk : min((n0 + half * C::kCols) / kBlk, NB - 1);
                xs = a.xs + (dead ? 0 : src * (int64_t)G);
                ws0 = a.ws + (present ? (e * NB + b0) * G : 0);
                ws1 = SILU && present ? ws0 + (a.N / 2 / kBlk) * G : ws0;
            };
            float sx, s0, s1 = 0.f;
            auto scales = [&](int g) {
                sx = fetch(xs + g);
                s0 = fetch(ws0 + g);
                if (SILU) s1 = fetch(ws1 + g);
            };
            Walk w = cur;
            look(w);
            enter(w);
            scales(g_lo);
            bool ready = false;  // the next accumulator was seen complete
            while (w.more()) {
                const int64_t r0 = (int64_t)w.rb * kRows, r = r0 + row;
                const int64_t n0 = (int64_t)w.nt * n_step;
                const bool is_dead = dead, is_present = present;
                w.next();
                if (!SPLIT) look(w);
                float tot[C::kCols];
#pragma unroll
                for (int j = 0; j < C::kCols; ++j) tot[j] = 0.f;
                for (int g = is_present ? g_lo : g_hi; g < g_hi; ++g) {
                    const float f0 = sx * s0, f1 = SILU ? sx * s1 : f0;
                    int next_g = g + 1;
                    if (next_g == g_hi) {
                        next_g = g_lo;
                        if (!SPLIT) enter(w);
                    }
                    scales(next_g);
                    if (!ready) mbar_wait(&sm.tfull[tb.idx], tb.phase, bad);
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::);
                    fold_block(tmem + ((uint32_t)(q * 32) << 16) + tb.idx * BN, col, f0, f1, tot, [&] {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.tempty[tb.idx]);
                        tb.next();
                        ready = mbar_test(&sm.tfull[tb.idx], tb.phase);
                    });
                }
                if (!is_present && !SPLIT) {
                    enter(w);
                    scales(g_lo);
                }
                // rows of zeros are zero whatever the lane's accumulator held: such a lane writes
                // `fill` over its staged row (a wait that gave up makes every row one, of NaN)
                const bool refill = is_dead || *bad;
                const float fill = *bad ? __int_as_float(0x7fffffff) : 0.f;
                if constexpr (SPLIT) {
                    // park the partial tile; the ring is idle once the last accumulator was read
                    float* part = reinterpret_cast<float*>(sm.ring) + row * C::kPitch;
#pragma unroll
                    for (int j = 0; j < C::kCols; j += 4)
                        *reinterpret_cast<float4*>(part + col(j)) =
                            make_float4(tot[j], tot[j + 1], tot[j + 2], tot[j + 3]);
                    if (refill)
#pragma unroll 1
                        for (int j = 0; j < C::kCols; ++j)
                            part[SILU ? (j & 63) + (j >> 6) * 128 + half * 64 : half * C::kCols + j] = fill;
                } else if constexpr (SILU) {
                    float m = 0.f;
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        silu_mul2(tot[j], tot[j + 1], tot[j + 64], tot[j + 65]);
                        m = fmaxf(m, fmaxf(fabsf(tot[j]), fabsf(tot[j + 1])));
                    }
                    if (refill) m = fill;
                    // the row's other 64 outputs are with the warp of the other half
                    float(&amax)[2][kRows] = sm.amax[done & 1];
                    amax[half][row] = m;
                    asm volatile("bar.sync %0, 64;" ::"r"(q + 1) : "memory");
                    m = fmaxf(m, amax[half ^ 1][row]);
                    const float s = __fdiv_rn(fmaxf(m, kAmaxFloor), kE4m3Max);
                    const float rcp = __frcp_rn(s);
                    if (r < rows) {
                        const int64_t inter = a.N / 2;
                        if (half == 0) a.qs[r * (inter / kBlk) + n0 / kBlk] = s;
                        uint8_t* p = a.q + r * inter + n0 + half * 64;
#pragma unroll
                        for (int j = 0; j < 64; j += 32) {
                            uint32_t u[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                u[i] = quant4(tot[j + 4 * i], tot[j + 4 * i + 1], tot[j + 4 * i + 2],
                                              tot[j + 4 * i + 3], rcp);
                            if (refill)
#pragma unroll
                                for (int i = 0; i < 8; ++i) u[i] = fill == 0.f ? 0u : 0x7f7f7f7fu;
                            store32(p + j, u);
                        }
                    }
                } else {
                    const bool by_tma = tma_out((int)(r0 / kRows));
                    const int64_t r_warp = r0 + q * 32;
                    const int count = (int)min(rows - r_warp, (int64_t)32);
                    constexpr int kPer = 16 / sizeof(Out);
#pragma unroll
                    for (int i = 0; i < kRounds; ++i) {
                        uint8_t* so = sm.stage_out[half][0] + q * 4096;
#pragma unroll
                        for (int l = 0; l < C::kLines; ++l)  // the last copy sent from it has read it
                            mbar_wait(&sm.ofree[half * C::kLines + l], turn ^ 1, bad);
#pragma unroll
                        for (int l = 0; l < C::kLines; ++l)
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                uint4 u;
                                const float* v = tot + (i * C::kLines + l) * kLineCols + c * kPer;
                                if constexpr (sizeof(Out) == 4)
                                    u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]),
                                                   __float_as_uint(v[2]), __float_as_uint(v[3]));
                                else
                                    u = make_uint4(pack2<Out>(v[0], v[1]), pack2<Out>(v[2], v[3]),
                                                   pack2<Out>(v[4], v[5]), pack2<Out>(v[6], v[7]));
                                *reinterpret_cast<uint4*>(so + l * (kRows * 128) + lane * 128 +
                                                          ((c ^ (lane & 7)) << 4)) = u;
                            }
                        if (refill) {
                            uint32_t v;
                            if constexpr (sizeof(Out) == 4) v = __float_as_uint(fill);
                            else v = pack2<Out>(fill, fill);
#pragma unroll 1
                            for (int c = 0; c < 8 * C::kLines; ++c)
                                *reinterpret_cast<uint4*>(so + (c >> 3) * (kRows * 128) + lane * 128 +
                                                          (c & 7) * 16) = make_uint4(v, v, v, v);
                        }
                        if (by_tma) {
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                            if (lane < C::kLines) mbar_arrive(&sm.ofull[half * C::kLines + lane]);
                            turn ^= 1;
                        } else {
                            __syncwarp();
                            for (int l = 0; l < C::kLines; ++l)
                                send_line<sizeof(Out)>(a, t.out_vec, so + l * (kRows * 128), r_warp, count,
                                                       (int)n0 + half * C::kCols +
                                                           (i * C::kLines + l) * kLineCols);
                            __syncwarp();
                        }
                    }
                }
                ++done;
                if (SPLIT) break;
            }
            __syncwarp();
            if (SPLIT) {
                cluster_sync();
                // CTA `rank` finishes rows rank, rank + S, ... of the cluster's tile
                if (cur.more()) {
                    const int64_t r0 = (int64_t)cur.rb * kRows, n0 = (int64_t)cur.nt * n_step;
                    const float* part = reinterpret_cast<const float*>(sm.ring);
                    for (int tr = rank + S * (warp - kFoldWarp0); tr < kRows && r0 + tr < rows;
                         tr += S * kFoldWarps)
                        finish_row<BN, Out, true>(a, t.out_vec, part + tr * C::kPitch, S, 0, r0 + tr, n0, false);
                }
                // no CTA leaves, or loads its next tile over the parked one, while that is read
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                cluster_sync();
                cur.next();
            }
        } while (SPLIT && cur.more());
    }
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem_base), "r"(512u));
    }
}

template <int BN, typename Out, bool SPLIT>
int launch_t(TcArgs t, int64_t tiles, cudaStream_t st) {
    constexpr bool kStaged = !std::is_void<Out>::value && !SPLIT;
    const Fp8Args& a = t.f;
    CUtensorMap tmx, tmw, tmo{};
    if (!make_maps(a, a.sorted_ids ? 1 : kRows, BN, &tmx, &tmw))
        return set_error("fp8_block: tensor map encoding failed");
    const int64_t pitch = a.N * (a.out_dtype == 0 ? 4 : 2);
    if (kStaged && pitch > INT32_MAX) t.out_vec = 0;  // beyond a TMA coordinate
    if (kStaged && t.out_vec &&
        !make_tma_map_u8(&tmo, a.out, (uint64_t)a.P, (uint64_t)pitch, 128, kRows, CU_TENSOR_MAP_SWIZZLE_128B))
        return set_error("fp8_block: tensor map encoding failed");
    return launch_persistent<fp8_tc_kernel<BN, Out, SPLIT>, false>(
        t, tiles, sizeof(Smem<BN, kStaged>) + 1024, st, tmx, tmw, tmo);
}

template <typename Out>
int launch_out(const TcArgs& t, bool bn256, int64_t tiles, cudaStream_t st) {
    if constexpr (std::is_void<Out>::value)
        return t.split > 1 ? launch_t<256, Out, true>(t, tiles, st) : launch_t<256, Out, false>(t, tiles, st);
    else if (bn256)
        return launch_t<256, Out, false>(t, tiles, st);
    else
        return t.split > 1 ? launch_t<128, Out, true>(t, tiles, st) : launch_t<128, Out, false>(t, tiles, st);
}

}  // namespace

bool fp8_tc_ok(const Fp8Args& a) {
    return a.K % 16 == 0 && a.x_rows > 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(a.w) & 15) == 0 &&
           (!a.silu || (reinterpret_cast<uintptr_t>(a.q) & 31) == 0);
}

int launch_fp8_tc(const Fp8Args& a, cudaStream_t st) {
    // Up to 64 rows a block the tokens go on the MMA's N side, where they cost by their number.
    const int64_t rows = a.expert_ids ? a.block_m : a.P;
    if (rows <= 64 || (!a.expert_ids && (rows + 63) / 64 * ((a.N + 127) / 128) <= sm_count()))
        return launch_fp8_swap(a, st);
    TcArgs t{};
    t.f = a;
    t.out_vec = out_vec(a);
    // row blocks that can hold work: with routing, at most one per slot and 128 rows of its block
    int64_t blocks = (a.P + kRows - 1) / kRows;
    if (a.sorted_ids) blocks = std::min<int64_t>(blocks, (int64_t)a.num_slots * (a.block_m / kRows));
    const int64_t n = a.silu ? a.N / 2 : a.N;
    // Wide tiles once they fill the GPU; below that, narrow tiles and a cluster along K.
    const int64_t wide = blocks * ((n + (a.silu ? 127 : 255)) / (a.silu ? 128 : 256));
    const int64_t narrow = blocks * ((n + 127) / 128);
    const bool bn256 = a.silu || wide >= sm_count();
    const int64_t tiles = bn256 ? wide : narrow;
    t.n_tiles = (int)(tiles / blocks);
    t.split = split_for(tiles, a.G);
    if (a.silu) return launch_out<void>(t, bn256, tiles, st);
    switch (a.out_dtype) {
        case 0: return launch_out<float>(t, bn256, tiles, st);
        case 1: return launch_out<__half>(t, bn256, tiles, st);
        default: return launch_out<__nv_bfloat16>(t, bn256, tiles, st);
    }
}

}  // namespace w4a8
