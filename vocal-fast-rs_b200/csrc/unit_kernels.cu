// Softmax cross entropy of frames over a codebook of units, and its gradients.
//
//   z[r][v] = scale x_r . w_v + bias_v, lse_r = log sum_v exp z[r][v]
//   loss_r = lse_r - z[r][label_r]  (0 where the label is outside [0, k))
//   G[r][v] = dloss_r (exp(z[r][v] - lse_r) - [v == label_r]), 0 in frames
//   without a label and in units left out (bias -inf)
//   dx = scale G w, dw = scale G^T x, dbias = column sums of G
//
// The logits are never kept.  The forward pass folds each tile of x w^T into
// a running (maximum, sum) per row as it leaves tensor memory; the backward
// pass forms G for a piece of the units at a time in the workspace and takes
// both products of the piece from there.  Large calls are bound by the
// tensor cores (2 rows k width operations a product), calls of few frames by
// reading the units.
//
// All products run on tcgen05 with f32 accumulators: bf16 operands as they
// are, f32 operands as three bf16 terms (24 bits: x = hi + mid + lo, each the
// rounding of what is left) and the six products above 2^-25 of the result.
// hi hi has an accumulator of its own, so the small products do not add to
// its roundings, and both are added up in registers after kChunk blocks of
// depth.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "pdl.cuh"
#include "row_io.cuh"
#include "tc_ptx.cuh"
#include "units.h"
#include "vfr_common.h"

namespace vfr {
namespace {

constexpr int kTileM = 128;      // TMEM lanes
constexpr int kBlockK = 64;      // bf16 elements of one 128-byte swizzled row
constexpr uint32_t kBoxBytes = 64 * kBlockK * 2;  // 64 rows of 128 B
constexpr int kEpiWarps = 16;    // four per lane quarter, each on a quarter of a tile's columns
constexpr int kParts = kEpiWarps / 4;
constexpr int kFirstEpi = 4;     // warps 0 and 2 load A and B, warp 1 issues MMAs, warp 3 only gives up registers
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
// 640 threads launch with 96 registers each: 61,440 = 128 x 64 + 512 x 104.
constexpr int kRoleRegisters = 64, kEpiRegisters = 104;
static_assert(128 * kRoleRegisters + 32 * kEpiWarps * kEpiRegisters <= kThreads * 96, "register split");
constexpr int kGroupM = 16;      // row tiles that share the units they read
constexpr uint32_t kTmemCols = 512;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;

// A bias or log-sum in units of ln 2.  What lies below -2.36e38 (a mask by the
// type's lowest value) stays finite, so that a row of such logits alone is a
// softmax of equal ones, as it is in natural units.
__device__ __forceinline__ float to_log2(float v) { return v == -INFINITY ? v : fmaxf(v * kLog2e, kLowest); }


// 2^v by the hardware's approximation (2 units in the last place of f32 for
// the arguments here, which are not above 0 but by rounding; results below
// 2^-126 are 0).
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// kTerms = 1 (bf16): tiles of 256 columns, 4 stages of A 16 KB + B 32 KB.
// kTerms = 3 (f32): tiles of 128 columns, 2 stages of three A and three B
// tiles of 16 KB; per accumulator buffer 128 columns of hi hi, 128 of the rest.
// kPair (bf16): a cluster of two CTAs on one M = 256, N = 256 MMA.  CTA r
// holds the tile's rows 128 r .. of A and columns 128 r .. of B at the same
// offsets as the other, and its TMEM gets its rows of the result: 32 KB a
// stage and CTA where one CTA alone reads 48 KB, so that L2 keeps up, and
// six stages.  The even CTA leads: it issues the MMAs, and every load of a
// stage counts on its barrier.  The gradients' products take it; the logits'
// do not: their epilogues would hold up two CTAs at a time.
template <int kTerms_, bool kPair_>
struct Shape {
    static constexpr int kTerms = kTerms_;
    static constexpr bool kPair = kPair_;
    static_assert(!kPair || kTerms == 1, "pairs multiply bf16");
    static constexpr int kCtas = kPair ? 2 : 1;
    static constexpr int kTileN = kTerms == 1 ? 256 : 128;
    static constexpr int kStages = kPair ? 6 : kTerms == 1 ? 3 : 2;
    static constexpr uint32_t kABytes = 2 * kBoxBytes;
    static constexpr uint32_t kBBytes = kTileN / kCtas / 64 * kBoxBytes;
    static constexpr uint32_t kStageBytes = kTerms * (kABytes + kBBytes);
    // Logits: per epilogue warp G on its way out, 32 rows of a part's columns,
    // and a tile's bias (f32: in the same place, before G).
    static constexpr uint32_t kStagingBytes = kPair ? 0 : 32 * kTileN / kParts * 2;
    static constexpr uint32_t kStagingOff = kStages * kStageBytes;
    static constexpr bool kBiasApart = kTerms == 1 && !kPair;
    static constexpr uint32_t kBiasBytes = kBiasApart ? 256 : kStagingBytes;
    static constexpr uint32_t kBiasOff = kStagingOff + (kBiasApart ? kEpiWarps * kStagingBytes : 0);
    static constexpr uint32_t kBarOff = kStagingOff + kEpiWarps * (kStagingBytes + (kBiasApart ? kBiasBytes : 0));
    static constexpr size_t kSmem = 1024 + kBarOff + 256;
    static_assert(kSmem <= 232448, "shared memory");
};

// This CTA among those that share its tiles, and the sharing groups.
template <class S>
__device__ __forceinline__ uint32_t tile_rank() { return S::kPair ? blockIdx.x & 1 : 0; }
template <class S>
__device__ __forceinline__ uint32_t tile_group() { return blockIdx.x / S::kCtas; }
template <class S>
__device__ __forceinline__ uint32_t tile_groups() { return gridDim.x / S::kCtas; }

// A tile of a product: rows m0.., columns n0.. (n_cols of them, a multiple of
// 16), depth blocks [k0, k1).  One load brings a block of an operand's term:
// K-major ones are boxes of 64 k by the tile's rows, at (k, row, 0, term);
// MN-major ones 64 columns by 64 k, for each 64 columns of the tile, at
// (0, k, column / 64, term).
struct Tile {
    const CUtensorMap *a, *b;
    bool a_mn, b_mn;
    int32_t m0, n0, n_cols;
    int32_t k0, k1;
};

// Depth blocks summed in tensor memory before f32 registers take over.  The
// accumulator truncates where f32 rounds: at depth 768 in one run a log-sum
// of 20 comes out 1.2e-5 low, in runs of 6 blocks 6e-6, of 4 blocks 4e-6.
// With 6 the tensor cores are a whole tile ahead of the epilogue at depth
// 768, with 4 they wait for it (forward of 30,000 x 16,384 back to back:
// 642 us in one run, 658 by 6, 709 by 4).  The backward pass is held up by
// its epilogue either way and takes 4.  f32 operands, six products a block,
// take 2 and 1: both passes truncate by amounts close to each other, and what
// they differ by goes into gradients whose sums nearly cancel (64 units,
// 30,000 rows of 256, errors of dunits and dbias: 3.8e-5 and 4.6e-5 by 4 and
// 2, 5.2e-5 and 6.5e-5 by 4 and 1, 2.2e-5 and 2.3e-5 by 2 and 1; 4,096 x 4,096
// x 768 takes 134 us against 128 forward, 384 against 371 backward).  Results
// that are rounded to bf16 take one run.
constexpr int kOneRun = 1 << 30;
template <class S, bool kBackward>
constexpr int kLogitRun = S::kTerms == 1 ? (kBackward ? 4 : 6) : (kBackward ? 1 : 2);
constexpr int kGradientRun = 4;

// A bounded wait of a whole warp, the same answer for every lane.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, tc::mbar_wait(bar, parity, kWaitLimitNs));
}

struct Bars {
    uint64_t *full, *empty, *acc_full, *acc_empty;
    uint32_t *tmem_slot;
};

template <class S>
__device__ __forceinline__ Bars bars_at(uint8_t *smem) {
    Bars b;
    b.full = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
    b.empty = b.full + S::kStages;
    b.acc_full = b.empty + S::kStages;
    b.acc_empty = b.acc_full + 2;
    b.tmem_slot = reinterpret_cast<uint32_t *>(b.acc_empty + 2);
    return b;
}

// A loading warp: its operand's blocks of every tile through the stages.  The
// two operands have a warp each: a lane issues a load in some 170 cycles,
// and a stage's MMAs take 512.  `walk.next` gives the CTA's next tile, false
// past the last.
template <class S, bool kB, class Walk>
__device__ __forceinline__ void produce(uint8_t *smem, const Bars &bars, Walk walk) {
    constexpr int kTerms = S::kTerms;
    constexpr uint32_t kBytes = kB ? S::kBBytes : S::kABytes;
    // of both CTAs of a pair
    const uint32_t bytes = kTerms * (kB ? walk.a.tile_n * kBlockK * 2 : S::kCtas * S::kABytes);
    const uint32_t rank = tile_rank<S>();
    smem += kB ? kTerms * S::kABytes : 0;
    const bool leader = tc::elect_one();
    int stage = 0;
    uint32_t phase = 0;
    Tile t, after;
    bool more = walk.next(t), ok = true;
    while (more && ok) {
        const CUtensorMap *map = kB ? t.b : t.a;
        const bool mn = kB ? t.b_mn : t.a_mn;
        const int32_t r = kB ? t.n0 + static_cast<int32_t>(rank) * (S::kTileN / 2) : t.m0;
        for (int k = t.k0; k < t.k1; ++k) {
            ok = warp_wait(&bars.empty[stage], phase ^ 1);
            if (!ok) break;
            if (leader) {
                if (rank == 0) tc::mbar_arrive_expect_tx(&bars.full[stage], bytes);
                uint8_t *dst = smem + stage * S::kStageBytes;
                const int32_t kk = k * kBlockK;
                if constexpr (S::kPair) {
                    tc::tma_load_4d_pair(dst, map, tc::map_to_rank(&bars.full[stage], 0), mn ? 0 : kk, mn ? kk : r,
                                         mn ? r / 64 : 0, 0);
                } else {
#pragma unroll
                    for (int p = 0; p < kTerms; ++p)
                        tc::tma_load_4d(dst + p * kBytes, map, &bars.full[stage], mn ? 0 : kk, mn ? kk : r,
                                        mn ? r / 64 : 0, p);
                }
            }
            __syncwarp();
            if (++stage == S::kStages) {
                stage = 0;
                phase ^= 1;
            }
            if (k == t.k0) more = walk.next(after);  // while this tile's copies are on their way
        }
        t = after;
    }
    // let every issued copy land before the CTA can exit
    for (int s = 0; s < S::kStages; ++s) {
        if (!warp_wait(&bars.empty[stage], phase ^ 1)) break;
        if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
        }
    }
}

// MMA warp, one lane of which issues; the others keep the addresses uniform.
// Accumulator buffer b of a run: TMEM columns 256 b (the product,
// or hi hi) and 256 b + 128 (the other terms' products).
template <class S, int kRun, class Walk>
__device__ __forceinline__ void multiply(uint8_t *smem, const Bars &bars, uint32_t tmem, Walk walk) {
    constexpr int kTerms = S::kTerms;
    const bool leader = tc::elect_one();
    int stage = 0;
    uint32_t phase = 0, acc_count = 0;
    Tile t, after;
    bool more = walk.next(t);
    while (more) {
        const uint32_t idesc = tc::idesc_f16(kTileM * S::kCtas, t.n_cols, 1) | (t.a_mn ? tc::kIdescMnA : 0) |
                               (t.b_mn ? tc::kIdescMnB : 0);
        // descriptors of an operand at shared address 0, and their step (in 16 B) per 16 of depth
        const uint64_t a_base = t.a_mn ? tc::smem_desc_sw128_mn(0, kBoxBytes) : tc::smem_desc_sw128(0);
        const uint64_t b_base = t.b_mn ? tc::smem_desc_sw128_mn(0, kBoxBytes) : tc::smem_desc_sw128(0);
        const uint32_t a_step = t.a_mn ? 2048 >> 4 : 32 >> 4, b_step = t.b_mn ? 2048 >> 4 : 32 >> 4;
        for (int k = t.k0; k < t.k1;) {
            const int stop = t.k1 - k > kRun ? k + kRun : t.k1;
            const uint32_t b = acc_count & 1;
            if (!warp_wait(&bars.acc_empty[b], ((acc_count >> 1) & 1) ^ 1)) return;
            tc::tc_fence_after();
            const uint32_t d = tmem + b * 256;
            uint32_t held = 0;  // whether the accumulators hold a sum
            for (; k < stop; ++k) {
                if (!warp_wait(&bars.full[stage], phase)) return;
                tc::tc_fence_after();
                const uint32_t sa = tc::smem_u32(smem + stage * S::kStageBytes), sb = sa + kTerms * S::kABytes;
                auto product = [&](uint32_t acc, int pa, int pb, uint32_t add) {
                    const uint64_t da = a_base + ((sa + pa * S::kABytes) >> 4);
                    const uint64_t db = b_base + ((sb + pb * S::kBBytes) >> 4);
#pragma unroll
                    for (int kk = 0; kk < kBlockK / 16; ++kk) {
                        if constexpr (S::kPair)
                            tc::mma_f16_pair(acc, da + kk * a_step, db + kk * b_step, idesc, kk ? 1 : add);
                        else tc::mma_f16(acc, da + kk * a_step, db + kk * b_step, idesc, kk ? 1 : add);
                    }
                };
                if (leader) {
                    if constexpr (kTerms == 1) {
                        product(d, 0, 0, held);
                    } else {
                        product(d + 128, 0, 2, held);
                        product(d + 128, 2, 0, 1);
                        product(d + 128, 1, 1, 1);
                        product(d + 128, 0, 1, 1);
                        product(d + 128, 1, 0, 1);
                        product(d, 0, 0, held);
                    }
                    if constexpr (S::kPair) tc::mma_commit_pair(&bars.empty[stage]);
                    else tc::mma_commit(&bars.empty[stage]);
                }
                __syncwarp();
                held = 1;
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
                if (k == t.k0) more = walk.next(after);  // while the tensor cores work
            }
            if (leader) {
                if constexpr (S::kPair) tc::mma_commit_pair(&bars.acc_full[b]);
                else tc::mma_commit(&bars.acc_full[b]);
            }
            __syncwarp();
            ++acc_count;
        }
        t = after;
    }
}

// Epilogue warps' side of the accumulators.  An accumulator is free again as
// soon as it is in registers.  Once a wait gave up (`bad`) the registers are
// not to be used, and every later result is NaN, so that none of a call that
// went wrong looks like one.
template <class S>
struct Drain {
    uint32_t acc_count = 0;
    bool bad = false;

    __device__ __forceinline__ uint32_t wait(const Bars &bars, uint32_t base) {
        if (!bad) bad = !warp_wait(&bars.acc_full[acc_count & 1], (acc_count >> 1) & 1);
        tc::tc_fence_after();
        return base + (acc_count & 1) * 256;
    }
    __device__ __forceinline__ void release(const Bars &bars) {
        tc::tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            if constexpr (S::kPair) tc::mbar_arrive_cluster(tc::map_to_rank(&bars.acc_empty[acc_count & 1], 0));
            else tc::mbar_arrive(&bars.acc_empty[acc_count & 1]);
        }
        ++acc_count;
    }
    template <int kCount>
    static __device__ __forceinline__ void add(float *a, const float (&b)[kCount]) {
#pragma unroll
        for (int i = 0; i < kCount; i += 2) {
            const float2 s = add2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = s.x, a[i + 1] = s.y;
        }
    }
};

// `load` leaves in v this lane's row of the warp's part of the tile, 32 kMax
// columns.  All are read, those past a narrow tile's too: they exist and
// nobody uses them.
template <class S, int kRun>
struct Columns : Drain<S> {
    static constexpr int kTerms = S::kTerms;
    static constexpr int kMax = S::kTileN / kParts / 32;  // 32-column chunks of a part
    float v[kMax][32];

    __device__ __forceinline__ void load(const Bars &bars, uint32_t base, int depth) {
        uint32_t at = this->wait(bars, base);
#pragma unroll
        for (int j = 0; j < kMax; ++j) tc::tmem_ld32_nowait(at + 32 * j, v[j]);
#pragma unroll
        for (int j = 0; j < kMax; ++j) tc::tmem_wait_ld32(v[j]);
        if constexpr (kTerms > 1) add_from(at + 128);
        this->release(bars);
        while (kRun != kOneRun && (depth -= kRun) > 0) {
            at = this->wait(bars, base);
            if constexpr (kTerms > 1) add_from(at + 128);
            add_from(at);
            this->release(bars);
        }
    }

private:
    __device__ __forceinline__ void add_from(uint32_t at) {
#pragma unroll
        for (int j = 0; j < 2 * kMax; ++j) {
            float u[16];
            tc::tmem_ld16_nowait(at + 16 * j, u);
            tc::tmem_wait_ld(u);
            this->add(v[j / 2] + 16 * (j & 1), u);
        }
    }
};

// The same part of the tile as a matrix product's accumulators lie: lane l
// holds, for q < 4, row 16 (q / 2) + 8 (q % 2) + l / 4, and of it columns
// 8 i + 2 (l % 4) and + 1 for i < 4 kMax.  A row's column sums then take 8 lanes
// and not 32, and 8 x 8 tiles go to shared memory as they are.
template <class S, int kRun>
struct Fragments : Drain<S> {
    static constexpr int kTerms = S::kTerms;
    static constexpr int kMax = S::kTileN / kParts / 32;
    static constexpr int kBlocks = 4 * kMax;  // of 8 columns
    float v[2][4 * kBlocks];  // [q / 2][4 i + 2 (q % 2) + e]

    __device__ __forceinline__ float &at(int q, int i, int e) { return v[q >> 1][4 * i + 2 * (q & 1) + e]; }
    __device__ __forceinline__ float2 pair(int q, int i) {
        return make_float2(at(q, i, 0), at(q, i, 1));
    }
    __device__ __forceinline__ void set(int q, int i, float2 p) { at(q, i, 0) = p.x, at(q, i, 1) = p.y; }

    __device__ __forceinline__ void load(const Bars &bars, uint32_t base, int depth) {
        uint32_t from = this->wait(bars, base);
#pragma unroll
        for (int h = 0; h < 2; ++h) tc::tmem_take_rows(from + (static_cast<uint32_t>(16 * h) << 16), v[h]);
        if constexpr (kTerms > 1) add_from(from + 128);
        this->release(bars);
        while ((depth -= kRun) > 0) {
            from = this->wait(bars, base);
            if constexpr (kTerms > 1) add_from(from + 128);
            add_from(from);
            this->release(bars);
        }
    }

private:
    __device__ __forceinline__ void add_from(uint32_t from) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < kMax; ++j) {
                float u[16];
                tc::tmem_take_rows(from + (static_cast<uint32_t>(16 * h) << 16) + 32 * j, u);
                this->add(v[h] + 16 * j, u);
            }
    }
};

// The kernel around the roles: barriers, TMEM, and the epilogue
// `epi(smem, bars, tmem, warp of the epilogue, lane)`.
template <class S, int kRun, class Walk, class Epi>
__device__ __forceinline__ void run_roles(const Walk &walk, Epi epi) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const Bars bars = bars_at<S>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tc::mbar_init(&bars.full[s], 2);
            tc::mbar_init(&bars.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&bars.acc_full[b], 1);
            tc::mbar_init(&bars.acc_empty[b], S::kCtas * kEpiWarps);
        }
        tc::fence_mbarrier_init();
    }
    if (warp == 1) {
        if constexpr (S::kPair) {
            tc::tmem_alloc_pair(bars.tmem_slot, kTmemCols);
            tc::tmem_relinquish_pair();
        } else {
            tc::tmem_alloc(bars.tmem_slot, kTmemCols);
            tc::tmem_relinquish();
        }
    }
    tc::tc_fence_before();
    if constexpr (S::kPair) tc::cluster_sync();  // the leader's barriers exist before the other CTA's loads
    else __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *bars.tmem_slot;
    grid_dependency_wait();
    if (warp < kFirstEpi) {
        tc::registers_down<kRoleRegisters>();
        if (warp == 0) produce<S, false>(smem, bars, walk);
        if (warp == 2) produce<S, true>(smem, bars, walk);
        if (warp == 1 && tile_rank<S>() == 0) multiply<S, kRun>(smem, bars, tmem, walk);
        __syncwarp();
    } else {
        tc::registers_up<kEpiRegisters>();
        epi(smem, bars, tmem, warp, lane);
    }
    tc::tc_fence_before();
    if constexpr (S::kPair) tc::cluster_sync();  // neither CTA leaves while the other may use its memory
    else __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        if constexpr (S::kPair) tc::tmem_dealloc_pair(tmem, kTmemCols);
        else tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------- logits

struct LogitArgs {
    int64_t rows;
    int32_t first, count;  // the units of this launch: [first, first + count)
    int32_t k;             // all units (labels outside [0, k) are none)
    int32_t k_blocks;      // depth blocks
    int32_t tile_n;        // columns of a tile
    int32_t span;          // column tiles of an item
    int32_t splits;        // items of a row tile
    int32_t m_tiles, n_tiles;
    const float *bias;
    const int32_t *labels;
    float scale;
    // forward
    float2 *partial;  // [kParts splits][rows] (maximum, sum), logits in units of ln 2
    float *target;    // [rows] logit of the label, in units of ln 2
    // backward
    const float *lse, *dloss;
    float *column_sums;  // [32-row blocks][count] or null
};

// The CTA's items, then each item's column tiles.  Items are row tiles in
// groups of kGroupM, the items of a group by columns first, so that the CTAs
// of a wave share kGroupM row tiles and few units.  32-bit arithmetic, two
// divisions an item: the loading and the MMA lane walk between tiles.
template <class S>
struct LogitWalk {
    const LogitArgs &a;
    const CUtensorMap *map_x, *map_w;
    uint32_t item, items;
    int m = 0, n = 0, end = 0;

    __device__ __forceinline__ LogitWalk(const LogitArgs &args, const CUtensorMap *x, const CUtensorMap *w)
        : a(args), map_x(x), map_w(w), item(tile_group<S>()),
          items(static_cast<uint32_t>(args.m_tiles) * args.splits) {}
    // Column tiles [n, end) of row tile m.
    __device__ __forceinline__ bool next_item() {
        if (item >= items) return false;
        const uint32_t group = item / (kGroupM * static_cast<uint32_t>(a.splits));
        const uint32_t rest = item - group * kGroupM * a.splits;
        const uint32_t rows = min(static_cast<uint32_t>(kGroupM), a.m_tiles - group * kGroupM);
        const uint32_t split = rest / rows;
        m = static_cast<int>(group * kGroupM + rest - split * rows);
        n = static_cast<int>(split) * a.span;
        end = min(n + a.span, a.n_tiles);
        item += tile_groups<S>();
        return true;
    }
    // This CTA's 128 rows of row tile m.
    __device__ __forceinline__ int block() const { return m * S::kCtas + static_cast<int>(tile_rank<S>()); }
    __device__ __forceinline__ bool next(Tile &t) {
        if (n == end && !next_item()) return false;
        t.a = map_x, t.b = map_w, t.a_mn = t.b_mn = false;
        t.m0 = block() * kTileM;
        t.n0 = n * a.tile_n;  // map_w covers the launch's units
        t.n_cols = S::kPair ? S::kTileN : min(a.tile_n, (a.count - t.n0 + 15) / 16 * 16);
        t.k0 = 0;
        t.k1 = a.k_blocks;
        ++n;
        return true;
    }
};

// The warp's place in the tile: TMEM lane quarter and part of the columns.  A
// tile of 64 columns occupies two parts of 32.
struct Place {
    int quarter, part, part_cols, chunks;
    uint32_t base;
    __device__ __forceinline__ Place(uint32_t tmem, int warp, int tile_n)
        : quarter(warp & 3), part((warp - kFirstEpi) >> 2), part_cols(max(tile_n / kParts, 32)),
          chunks(part * part_cols < tile_n ? part_cols / 32 : 0),
          base(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + part * part_cols) {}
};

// The lane's biases of a part that starts at column `at` - lane of the
// launch's units, -inf past the last.
template <int kMax>
__device__ __forceinline__ void column_bias(const LogitArgs &a, int at, float (&bias)[kMax]) {
#pragma unroll
    for (int j = 0; j < kMax; ++j) {
        const int c = at + 32 * j;
        bias[j] = c >= a.count ? -INFINITY : a.bias ? __ldg(a.bias + a.first + c) : 0.0f;
    }
}

// Forward: per row and item the running (maximum, sum), a row to a lane.
template <class S>
__device__ __forceinline__ void fold_logits(const LogitArgs &a, LogitWalk<S> own, uint8_t *smem, const Bars &bars,
                                            uint32_t tmem, int warp, int lane) {
    constexpr int kRun = kLogitRun<S, false>;
    const Place at(tmem, warp, a.tile_n);
    constexpr int kMax = Columns<S, kRun>::kMax;
    float *bias_slot = reinterpret_cast<float *>(smem + S::kBiasOff + (warp - kFirstEpi) * S::kBiasBytes);
    // logits in units of ln 2, z log2(e): exponentials are powers of two
    const float2 scale = make_float2(a.scale * kLog2e, a.scale * kLog2e);
    Columns<S, kRun> columns;
    auto &v = columns.v;
    while (own.next_item()) {
        const int64_t row = static_cast<int64_t>(own.block()) * kTileM + at.quarter * 32 + lane;
        const bool live = row < a.rows;
        int32_t label = live ? a.labels[row] : -1;
        if (label >= a.k) label = -1;
        float top = -INFINITY, sum = 0.0f;
        float bias[kMax];
        column_bias(a, own.n * a.tile_n + at.part * at.part_cols + lane, bias);
        for (int n = own.n; n < own.end; ++n) {
            const int col0 = n * a.tile_n + at.part * at.part_cols;
            // which columns take no part: units left out and columns past the
            // last, -inf whatever the product is
            uint32_t out[kMax];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kMax; ++j) {
                bias_slot[32 * j + lane] = to_log2(bias[j]);
                out[j] = __ballot_sync(0xFFFFFFFFu, bias[j] == -INFINITY);
            }
            __syncwarp();
            columns.load(bars, at.base, a.k_blocks);
            column_bias(a, col0 + a.tile_n + lane, bias);  // the next tile's, while this one is worked on
#pragma unroll
            for (int j = 0; j < kMax; ++j) {
                if (j >= at.chunks) break;
                const float4 *b4 = reinterpret_cast<const float4 *>(bias_slot + 32 * j);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 b = b4[i / 4];
                    const float2 lo = fma2(make_float2(v[j][i], v[j][i + 1]), scale, make_float2(b.x, b.y));
                    const float2 hi = fma2(make_float2(v[j][i + 2], v[j][i + 3]), scale, make_float2(b.z, b.w));
                    v[j][i] = lo.x, v[j][i + 1] = lo.y, v[j][i + 2] = hi.x, v[j][i + 3] = hi.y;
                }
                if (out[j]) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (out[j] >> i & 1) v[j][i] = -INFINITY;
                }
            }
            const int hit = label - col0;  // the label's column in the part
            if (label >= 0 && hit >= 0 && hit < 32 * at.chunks) {
#pragma unroll
                for (int j = 0; j < kMax; ++j)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * j + i == hit) a.target[row] = v[j][i];
            }
            float m8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) m8[i] = top;
#pragma unroll
            for (int j = 0; j < kMax; ++j) {
                if (j >= at.chunks) break;
#pragma unroll
                for (int i = 0; i < 32; i += 2) m8[i / 2 & 7] = fmaxf(m8[i / 2 & 7], fmaxf(v[j][i], v[j][i + 1]));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) m8[i] = fmaxf(m8[i], m8[i + 4]);
            const float next = fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3]));
            const float from = next == -INFINITY ? 0.0f : next;
            const float2 minus = make_float2(-from, -from);
            float2 s4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) s4[i] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < kMax; ++j) {
                if (j >= at.chunks) break;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 d = add2(make_float2(v[j][i], v[j][i + 1]), minus);
                    s4[i / 2 & 3] = add2(s4[i / 2 & 3], make_float2(exp2_approx(d.x), exp2_approx(d.y)));
                }
            }
            const float2 s = add2(add2(s4[0], s4[1]), add2(s4[2], s4[3]));
            sum = fmaf(sum, exp2_approx(top - from), s.x + s.y);
            top = next;
        }
        if (columns.bad) sum = NAN;
        if (live) a.partial[(own.n / a.span * kParts + at.part) * a.rows + row] = make_float2(top, sum);
    }
}

// Backward: G in bf16 (f32: three terms) to global memory, and its column sums.
template <class S>
__device__ __forceinline__ void store_gradients(const LogitArgs &a, const CUtensorMap *map_g, LogitWalk<S> own,
                                                uint8_t *smem, const Bars &bars, uint32_t tmem, int warp, int lane) {
    constexpr int kTerms = S::kTerms, kRun = kLogitRun<S, true>;
    const Place at(tmem, warp, a.tile_n);
    using Frag = Fragments<S, kRun>;
    constexpr int kMax = Frag::kMax, kBlocks = Frag::kBlocks;
    float *bias_slot = reinterpret_cast<float *>(smem + S::kBiasOff + (warp - kFirstEpi) * S::kBiasBytes);
    uint8_t *staging = smem + S::kStagingOff + (warp - kFirstEpi) * S::kStagingBytes;
    // natural units: where p nears 1 the difference of logit and log-sum is
    // small, and scaling it afterwards loses nothing
    const float2 scale = make_float2(a.scale, a.scale);
    const int pair = 2 * (lane & 3);  // the lane's first column of each 8
    Frag f;
    while (own.next_item()) {
        const int64_t row0 = static_cast<int64_t>(own.block()) * kTileM + at.quarter * 32;
        int32_t label[4];
        float lse[4], grad[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t row = row0 + 16 * (q >> 1) + 8 * (q & 1) + (lane >> 2);
            label[q] = row < a.rows ? a.labels[row] : -1;
            const bool valid = label[q] >= 0 && label[q] < a.k;
            if (!valid) label[q] = -1;
            // Without a label p = exp(-inf) and G = 0 (its frame is a row of
            // zeros); with every unit left out p = exp(-inf - 0)
            lse[q] = !valid ? INFINITY : a.lse[row] == -INFINITY ? 0.0f : a.lse[row];
            grad[q] = valid ? a.dloss[row] : 0.0f;
        }
        float bias[kMax];
        column_bias(a, own.n * a.tile_n + at.part * at.part_cols + lane, bias);
        for (int n = own.n; n < own.end; ++n) {
            const int col0 = n * a.tile_n + at.part * at.part_cols;  // within the launch's units
            // -inf for units left out (rows of zeros) and columns past the last
            if (!S::kBiasApart) tc::bulk_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kMax; ++j) bias_slot[32 * j + lane] = bias[j];
            __syncwarp();
            f.load(bars, at.base, a.k_blocks);
            column_bias(a, col0 + a.tile_n + lane, bias);  // the next tile's, while this one is worked on
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                if (i >= 4 * at.chunks) break;
                const float2 b = *reinterpret_cast<const float2 *>(bias_slot + 8 * i + pair);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 d = add2(fma2(f.pair(q, i), scale, b), make_float2(-lse[q], -lse[q]));
                    const float2 e = mul2(d, make_float2(kLog2e, kLog2e));
                    f.set(q, i, make_float2(exp2_approx(e.x), exp2_approx(e.y)));
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                // the label's column, where the unit takes part
                const int hit = label[q] - a.first - col0;
                if (label[q] >= 0 && hit >= 0 && hit < 32 * at.chunks && (hit & 6) == pair &&
                    bias_slot[hit] != -INFINITY) {
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (8 * i + e + pair == hit) f.at(q, i, e) -= 1.0f;
                }
                const float by = f.bad ? NAN : grad[q];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) f.set(q, i, mul2(f.pair(q, i), make_float2(by, by)));
            }
            if (a.column_sums) {
                // the lane's four rows, then the eight lanes of a column: lane
                // group l / 4 ends with block l / 4 (of 32 columns: l / 4 % 4)
                float2 s[kBlocks];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
                    s[i] = add2(add2(f.pair(0, i), f.pair(1, i)), add2(f.pair(2, i), f.pair(3, i)));
#pragma unroll
                for (int o = kBlocks / 2; o; o >>= 1) {
                    const bool upper = lane & (4 * o);
#pragma unroll
                    for (int i = 0; i < o; ++i) {
                        const float2 keep = upper ? s[i + o] : s[i], send = upper ? s[i] : s[i + o];
                        s[i] = add2(keep, make_float2(__shfl_xor_sync(0xFFFFFFFFu, send.x, 4 * o),
                                                      __shfl_xor_sync(0xFFFFFFFFu, send.y, 4 * o)));
                    }
                }
                if constexpr (kBlocks == 4)
                    s[0] = add2(s[0], make_float2(__shfl_xor_sync(0xFFFFFFFFu, s[0].x, 16),
                                                  __shfl_xor_sync(0xFFFFFFFFu, s[0].y, 16)));
                const int block = lane >> 2, c = col0 + 8 * block + pair;
                if (block < 4 * at.chunks) {
                    float *sums = a.column_sums + row0 / 32 * a.count;
                    if (c < a.count) sums[c] = s[0].x;
                    if (c + 1 < a.count) sums[c + 1] = s[0].y;
                }
            }
            // a factor of its own products, rounded as any operand of theirs;
            // a store takes the part's 64 columns at once, or 32 of a narrow part
            const int units = 4 * at.chunks;  // of 16 bytes in a row of a store
#pragma unroll
            for (int p = 0; p < kTerms; ++p) {
                if (at.chunks == 0) break;
                tc::bulk_wait_read<0>();
                __syncwarp();
                // swizzled as SWIZZLE_128B or SWIZZLE_64B expects; tile l / 8
                // of four: rows + 8 (tile % 2), units + tile / 2
                const int r = lane & 15, turn = kMax == 2 && units == 8 ? r & 7 : r >> 1 & 3;
                const uint32_t to = tc::smem_u32(staging) + r * 16 * units;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < kBlocks; i += 2) {
                        if (i >= units) break;
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int q = 2 * h + (e & 1), block = i + (e >> 1);
                            const float2 x = f.pair(q, block);
                            const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y);
                            w[e] = *reinterpret_cast<const uint32_t *>(&y);
                            if (p + 1 < kTerms) {
                                const float2 z = __bfloat1622float2(y);
                                f.set(q, block, make_float2(x.x - z.x, x.y - z.y));
                            }
                        }
                        tc::store_tiles(to + 256 * units * h + (((i + (lane >> 4)) ^ turn) << 4), w[0], w[1], w[2],
                                        w[3]);
                    }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && col0 < a.count && row0 < a.rows)
                    tc::tma_store_3d(map_g, staging, col0, static_cast<int32_t>(row0), p);
                if (lane == 0) tc::bulk_commit();
            }
        }
    }
    if (lane == 0) tc::bulk_wait_all();
    __syncwarp();
}

// Bound by the tensor cores forward (82% busy at 16,384 x 8,192 x 768 bf16,
// 148 us; f32 76% at 4,096 x 4,096 x 768, 129 us) and, backward, by the
// epilogue that holds them up (58%, 196 us; f32 63%, 153 us).  Tiles of 128
// rows keep a row's sums in one lane's registers; single CTAs, as a pair's
// two epilogues would wait for each other.
template <class S, bool kBackward>
__global__ void __launch_bounds__(kThreads, 1)
    logit_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_g, const LogitArgs a) {
    const LogitWalk<S> walk(a, &map_x, &map_w);
    run_roles<S, kLogitRun<S, kBackward>>(
        walk, [&](uint8_t *smem, const Bars &bars, uint32_t tmem, int warp, int lane) {
            if constexpr (kBackward) store_gradients<S>(a, &map_g, walk, smem, bars, tmem, warp, lane);
            else fold_logits<S>(a, walk, smem, bars, tmem, warp, lane);
        });
}

// Joins the slots of each row: 32 rows a CTA, a warp for every eighth slot.
// Bound by latency (16,384 rows: 7 us, 4 MB read).
__global__ void __launch_bounds__(256) loss_kernel(const float2 *partial, const float *target, const int32_t *labels,
                                                   const float *bias, int64_t rows, int slots, int k, float *loss,
                                                   float *lse) {
    __shared__ float2 joined[8][32];
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float top = -INFINITY, sum = 0.0f;
    auto join = [&](float2 p) {
        const float next = fmaxf(top, p.x);
        const float from = next == -INFINITY ? 0.0f : next;
        sum = sum * exp2_approx(top - from) + p.y * exp2_approx(p.x - from);
        top = next;
    };
    if (row < rows) {
#pragma unroll 4
        for (int s = warp; s < slots; s += 8) join(partial[s * rows + row]);
    }
    joined[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp != 0 || row >= rows) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) join(joined[w][lane]);
    const float l = top == -INFINITY && sum == 0.0f ? top : top + log2f(sum);
    const float natural = l == kLowest ? kLowest : l * kLn2;  // see to_log2
    lse[row] = natural;
    const int32_t t = labels[row];
    if (t < 0 || t >= k) {
        loss[row] = 0.0f;
    } else {
        const float z = target[row];
        loss[row] = z == -INFINITY ? INFINITY : z == kLowest && l > kLowest ? natural - bias[t] : (l - z) * kLn2;
    }
}

// ---------------------------------------------------------------- products

// dx (product 0: G [rows][count] times the units) and dunits (product 1: G^T
// times the frames) of one piece, in one launch.
struct ProductArgs {
    struct One {
        int32_t m_size, m_tiles;  // rows of the result
        int32_t k_blocks, splits, split_blocks;
        uint32_t items;
        void *out;            // the result, where a tile has all of its sum
        float *part;          // else f32 [splits][m_size][width]
        bool add;             // to what `part` holds from the pieces before
        int64_t part_stride;
    } one[2];
    int32_t width, n_tiles, tile_n;
    int32_t first_product;  // whose items come first: the longer ones
    uint32_t odd, extra;    // see ProductWalk
    float scale;
    bool bf16, wide;        // result type; 16-byte stores fit
};

// The CTA's items: the longer product's in turn over the grid, then the
// other's.  Where the longer ones do not come out even, the CTAs that got one
// less (from `odd` on) first take `extra` short items each.
template <class S>
struct ProductWalk {
    const ProductArgs &a;
    const CUtensorMap *map_g, *map_gt, *map_w, *map_x;
    uint32_t item, taken = 0;  // next long item; short items taken
    int which = 0, m = 0, n = 0, split = 0;

    __device__ __forceinline__ ProductWalk(const ProductArgs &args, const CUtensorMap *g, const CUtensorMap *gt,
                                           const CUtensorMap *w, const CUtensorMap *x)
        : a(args), map_g(g), map_gt(gt), map_w(w), map_x(x), item(tile_group<S>()) {}
    __device__ __forceinline__ bool next_item() {
        uint32_t i = item;
        which = a.first_product;
        if (i < a.one[which].items) {
            item += tile_groups<S>();
        } else {
            which ^= 1;
            const uint32_t groups = tile_groups<S>(), own = tile_group<S>(), late = groups - a.odd;
            if (own >= a.odd && taken < a.extra) {
                i = taken * late + own - a.odd;
            } else {
                const uint32_t round = own >= a.odd ? taken - a.extra : taken;
                i = a.extra * late + round * groups + own;
            }
            ++taken;
            if (i >= a.one[which].items) return false;
        }
        // columns first, then splits: neighbours share their rows of G
        const uint32_t rest = i / a.n_tiles;
        n = static_cast<int>(i - rest * a.n_tiles);
        split = static_cast<int>(rest / a.one[which].m_tiles);
        m = static_cast<int>(rest) - split * a.one[which].m_tiles;
        return true;
    }
    // This CTA's 128 rows of row tile m.
    __device__ __forceinline__ int block() const { return m * S::kCtas + static_cast<int>(tile_rank<S>()); }
    __device__ __forceinline__ bool next(Tile &t) {
        if (!next_item()) return false;
        const auto &o = a.one[which];
        t.a = which == 0 ? map_g : map_gt, t.b = which == 0 ? map_w : map_x;
        t.a_mn = which == 1, t.b_mn = true;
        t.m0 = block() * kTileM;
        t.n0 = n * a.tile_n;
        t.n_cols = S::kPair ? S::kTileN : min(a.tile_n, (a.width - t.n0 + 15) / 16 * 16);
        t.k0 = split * o.split_blocks;
        t.k1 = min(o.k_blocks, t.k0 + o.split_blocks);
        return true;
    }
};

// Bound by the tensor cores: 95% busy by pairs (16,384 x 8,192 x 768 bf16,
// both products 287 us, 1,435 TFLOP/s), 78% in f32 (4,096 x 4,096 x 768, 250
// us, six products each).
template <class S>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_gt,
                   const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const ProductArgs a) {
    const ProductWalk<S> walk(a, &map_g, &map_gt, &map_w, &map_x);
    constexpr int kRun = S::kTerms == 1 ? kOneRun : kGradientRun;
    run_roles<S, kRun>(walk, [&](uint8_t *, const Bars &bars, uint32_t tmem, int warp, int lane) {
        const int quarter = warp & 3, part = (warp - kFirstEpi) >> 2;
        const int part_cols = max(a.tile_n / kParts, 32), chunks = part * part_cols < a.tile_n ? part_cols / 32 : 0;
        const uint32_t base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + part * part_cols;
        Columns<S, kRun> columns;
        ProductWalk<S> p = walk;
        while (p.next_item()) {
            const auto &o = a.one[p.which];
            const int k0 = p.split * o.split_blocks;
            columns.load(bars, base, min(o.k_blocks, k0 + o.split_blocks) - k0);
            const int64_t row = static_cast<int64_t>(p.block()) * kTileM + quarter * 32 + lane;
            const float scale = columns.bad ? NAN : a.scale;
#pragma unroll
            for (int j = 0; j < columns.kMax; ++j) {
                if (j >= chunks) break;
                float(&v)[32] = columns.v[j];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= scale;
                const int col = p.n * a.tile_n + part * part_cols + 32 * j;
                if (row >= o.m_size || col >= a.width) continue;
                const int64_t at = row * a.width + col;
                if (o.part == nullptr) {
                    if (a.bf16) {
                        __nv_bfloat16 *q = static_cast<__nv_bfloat16 *>(o.out) + at;
                        if (a.wide) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8)
                                if (col + i < a.width) store_vec<__nv_bfloat16, 8>(q + i, v + i);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (col + i < a.width) q[i] = __float2bfloat16_rn(v[i]);
                        }
                    } else {
                        float *q = static_cast<float *>(o.out) + at;
                        if (a.wide) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                if (col + i < a.width) store_vec<float, 4>(q + i, v + i);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (col + i < a.width) q[i] = v[i];
                        }
                    }
                } else {
                    float *q = o.part + p.split * o.part_stride + at;
                    if (a.wide) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (col + i < a.width) {
                                if (o.add) {
                                    const float4 f = *reinterpret_cast<const float4 *>(q + i);
                                    v[i] += f.x, v[i + 1] += f.y, v[i + 2] += f.z, v[i + 3] += f.w;
                                }
                                store_vec<float, 4>(q + i, v + i);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col + i < a.width) q[i] = o.add ? q[i] + v[i] : v[i];
                    }
                }
            }
        }
    });
}

// What the products of a piece leave to do, in one launch: results whose
// depth was split, out[i] = sum over the splits of part[s][i], and dbias, the
// row blocks' column sums; each in order, the same bits every time.
struct FinishArgs {
    struct Join {
        const float *part;
        int64_t stride, count;
        int splits;
        unsigned blocks;  // CTAs, 0: nothing to join
        void *out;
    } join[2];
    const float *sums;  // [parts][columns]
    int64_t parts;
    int32_t columns;
    unsigned sum_blocks;  // CTAs of 32 columns, 0: no dbias
    float *dbias;
};
constexpr int kFinishThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const FinishArgs a) {
    __shared__ float slots[32][33];
    launch_dependents();
    grid_dependency_wait();
    unsigned block = blockIdx.x;
    if (block < a.sum_blocks) {
        // 32 columns, 32 warps over the row blocks
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int col = block * 32 + lane;
        float s = 0.0f;
        if (col < a.columns) {
#pragma unroll 8
            for (int64_t p = warp; p < a.parts; p += 32) s += a.sums[p * a.columns + col];
        }
        slots[warp][lane] = s;
        __syncthreads();
        s = slots[lane][warp];  // column `warp` of the CTA, part `lane`
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        const int c = block * 32 + warp;
        if (lane == 0 && c < a.columns) a.dbias[c] = s;
        return;
    }
    block -= a.sum_blocks;
    const int which = block < a.join[0].blocks ? 0 : 1;
    const auto &j = a.join[which];
    if (which) block -= a.join[0].blocks;
    for (int64_t i = static_cast<int64_t>(block) * kFinishThreads + threadIdx.x; i < j.count;
         i += static_cast<int64_t>(j.blocks) * kFinishThreads) {
        float s = 0.0f;
        for (int k = 0; k < j.splits; ++k) s += j.part[k * j.stride + i];
        static_cast<T *>(j.out)[i] = from_f32<T>(s);
    }
}

// ---------------------------------------------------------------- operands

// The products' operands: rows of bf16 terms, padded with zeros to 64 columns.
// With `clean`, frames without a label and units left out become zero rows:
// a zero of G times an infinity or a NaN there would reach the gradients.
// A warp a row, each element once (24,576 rows of 768 bf16: 14 us, a third of
// HBM's rate).
struct StageArgs {
    const void *x, *units;
    const float *bias;
    const int32_t *labels;
    int64_t rows;
    int32_t k, width, pitch;
    bool clean, wide;
    __nv_bfloat16 *xs, *ws;  // [terms][rows or k][pitch]
};

template <typename T, int kTerms>
__global__ void __launch_bounds__(256) stage_kernel(StageArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int64_t total = a.rows + a.k;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < total;
         r += static_cast<int64_t>(gridDim.x) * 8) {
        const bool frame = r < a.rows;
        const int64_t own = frame ? r : r - a.rows;
        bool keep = true;
        if (a.clean) {
            if (frame) {
                const int32_t t = a.labels[own];
                keep = t >= 0 && t < a.k;
            } else {
                keep = !a.bias || a.bias[own] != -INFINITY;
            }
        }
        const T *src = static_cast<const T *>(frame ? a.x : a.units) + own * a.width;
        __nv_bfloat16 *dst = (frame ? a.xs : a.ws) + own * a.pitch;
        const int64_t plane = (frame ? a.rows : a.k) * static_cast<int64_t>(a.pitch);
        for (int c = lane * 8; c < a.pitch; c += 256) {
            float v[8];
            if (!keep) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            } else if (a.wide) {
                constexpr int kVec = 16 / sizeof(T);
#pragma unroll
                for (int i = 0; i < 8; i += kVec) {
                    if (c < a.width) load_vec<T, kVec>(src + c + i, v + i);
                    else for (int e = 0; e < kVec; ++e) v[i + e] = 0.0f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = c + i < a.width ? to_f32(src[c + i]) : 0.0f;
            }
#pragma unroll
            for (int p = 0; p < kTerms; ++p) {
                store_vec<__nv_bfloat16, 8>(dst + p * plane + c, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // an infinity is its first term; the others would be NaN
                    const float rest = v[i] - __bfloat162float(__float2bfloat16_rn(v[i]));
                    v[i] = isfinite(v[i]) ? rest : 0.0f;
                }
            }
        }
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
    static EncodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    });
    require(fn != nullptr, "cuTensorMapEncodeTiled is unavailable");
    return fn;
}

// bf16 terms of [rows][pitch], `plane` elements apart; what lies outside
// reads as zero and is not written.
struct Terms {
    const void *base;
    int64_t cols, rows, pitch, plane;
    int count;
};
CUtensorMap encode(const Terms &t, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                   CUtensorMapSwizzle swizzle) {
    require(reinterpret_cast<uintptr_t>(t.base) % 16 == 0 && t.pitch % 8 == 0, "tensor map alignment");
    CUtensorMap map;
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    const CUresult rc = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(t.base), dims,
                                    strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    require(rc == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed");
    return map;
}
// Depth along the columns: boxes of 64 columns by `rows` rows.
CUtensorMap map_k_major(const Terms &t, int rows) {
    const cuuint64_t pitch = t.pitch * 2, plane = t.plane * 2;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(t.cols), static_cast<cuuint64_t>(t.rows), 1,
                                static_cast<cuuint64_t>(t.count)};
    const cuuint64_t strides[3] = {pitch, plane, plane};
    const cuuint32_t box[4] = {kBlockK, static_cast<cuuint32_t>(rows), 1, 1};
    return encode(t, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Depth along the rows: boxes of 64 rows by `cols` columns, 64 of them at a
// time.  The pitch is a multiple of 64, so the last run stays in its row;
// columns past the matrix's own reach only results that nobody stores.
CUtensorMap map_mn_major(const Terms &t, int cols) {
    require(t.pitch % 64 == 0, "tensor map pitch");
    const cuuint64_t pitch = t.pitch * 2, plane = t.plane * 2;
    const cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(t.rows), static_cast<cuuint64_t>((t.cols + 63) / 64),
                                static_cast<cuuint64_t>(t.count)};
    const cuuint64_t strides[3] = {pitch, 128, plane};
    const cuuint32_t box[4] = {64, kBlockK, static_cast<cuuint32_t>(cols / 64), 1};
    return encode(t, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// G's stores: 32 rows by `cols` columns, 32 or 64.
CUtensorMap map_store(const Terms &t, int cols) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(t.cols), static_cast<cuuint64_t>(t.rows),
                                static_cast<cuuint64_t>(t.count)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(t.pitch) * 2, static_cast<cuuint64_t>(t.plane) * 2};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(cols), 32, 1};
    return encode(t, 3, dims, strides, box, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// ---------------------------------------------------------------- plans

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
int terms_of(int dtype) { return dtype == kF32 ? 3 : 1; }

// Columns of a tile: the width whose rounds over the SMs are the shortest, a
// tile costing its columns and some 32 for its start and its end.
int tile_columns(int64_t m_tiles, int64_t cols, int terms, int sms) {
    int best = 0;
    int64_t least = INT64_MAX;
    for (int n = terms == 1 ? 256 : 128; n >= 64; n /= 2) {
        const int64_t cost = ceil_div(m_tiles * ceil_div(cols, n), sms) * (n + 32);
        if (cost < least) {
            least = cost;
            best = n;
        }
    }
    return best;
}

// Whether CTA pairs serve a product of so many rows and columns: a tile of 256
// by 256 for every pair at least, and less than a quarter of the columns'
// tiles empty.  Gradients, width 768, bf16, with pairs and without: 30,000 x
// 16,384 1,723 us and 1,956, 8,192^2 251 and 300, 8,192 x 4,096 140 and 161,
// 5,120^2 122 and 134, 3,500^2 (84 tiles) 101 and 99; below a tile a pair,
// 3,200 x 2,900 (72 tiles) 91 and 67.
bool pairs_fit(int64_t rows, int64_t cols, int terms, int sms) {
    return terms == 1 && ceil_div(rows, 256) * ceil_div(cols, 256) >= sms / 2 && ceil_div(cols, 256) * 192 <= cols;
}

// Column tiles of an item: the shortest rounds of the grid, an item costing a
// quarter of a tile for its start.
int item_span(int64_t m_tiles, int64_t n_tiles, int sms) {
    int64_t best = INT64_MAX, span = 1;
    for (int64_t s = 1; s <= std::min<int64_t>(n_tiles, 64); ++s) {
        const int64_t each = ceil_div(n_tiles, s);
        const int64_t cost = ceil_div(m_tiles * ceil_div(n_tiles, each), sms) * (4 * each + 1);
        if (cost < best) {
            best = cost;
            span = each;
        }
    }
    return static_cast<int>(span);
}

struct ForwardPlan {
    int64_t m_tiles, n_tiles;
    int tile_n, span, splits;
    size_t xs, ws, partial, target, bytes;  // offsets
    int pitch;
};
ForwardPlan plan_forward(int64_t rows, int k, int width, int dtype, int sms) {
    const int terms = terms_of(dtype);
    ForwardPlan p{};
    p.m_tiles = ceil_div(rows, kTileM);
    p.tile_n = tile_columns(p.m_tiles, k, terms, sms);
    p.n_tiles = ceil_div(k, p.tile_n);
    p.span = item_span(p.m_tiles, p.n_tiles, sms);
    p.splits = static_cast<int>(ceil_div(p.n_tiles, p.span));
    p.pitch = (width + 63) / 64 * 64;
    size_t at = 0;
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    p.xs = put(static_cast<size_t>(terms) * rows * p.pitch * 2);
    p.ws = put(static_cast<size_t>(terms) * k * p.pitch * 2);
    p.partial = put(static_cast<size_t>(kParts) * p.splits * rows * sizeof(float2));
    p.target = put(static_cast<size_t>(rows) * sizeof(float));
    p.bytes = at;
    return p;
}

// How many short items (of cost `brief`) the groups that got one long item
// (of cost `slow`) less take first, for the smallest makespan.
int64_t even_out(int64_t slows, int64_t briefs, int64_t slow, int64_t brief, int64_t groups, int64_t *makespan) {
    const int64_t odd = slows % groups, late = groups - odd, each = slows / groups;
    int64_t best = INT64_MAX, extra = 0;
    const int64_t most = odd ? slow / brief + 1 : 0;
    for (int64_t e = std::max<int64_t>(0, most - 1); e <= most; ++e) {
        const int64_t rest = briefs - e * late;
        const int64_t rounds = rest > 0 ? ceil_div(rest, groups) : 0;
        const int64_t early = (each + (odd ? 1 : 0)) * slow + rounds * brief;
        const int64_t other = each * slow + (rest > 0 ? e + rounds : ceil_div(briefs, late)) * brief;
        if (std::max(early, other) < best) {
            best = std::max(early, other);
            extra = e;
        }
    }
    *makespan = best;
    return extra;
}

struct BackwardPlan {
    int64_t piece;  // units of a piece
    bool pair;      // the gradients' products (the logits' goes by the piece)
    int pitch, g_pitch, tile_n;  // tile_n: of the gradients' columns
    int splits[2];
    bool direct[2];
    size_t xs, ws, g, sums, part[2], bytes;
};
// Bytes of G in the workspace, unless 256 units of every frame take more.
constexpr int64_t kPieceBytes = int64_t(1) << 30;

BackwardPlan plan_backward(int64_t rows, int k, int width, int dtype, int sms) {
    const int terms = terms_of(dtype);
    BackwardPlan p{};
    const int64_t fit = kPieceBytes / (std::max<int64_t>(rows, 1) * 2 * terms) / 256 * 256;
    p.piece = std::min<int64_t>(k, std::max<int64_t>(256, fit));
    p.pitch = (width + 63) / 64 * 64;
    p.g_pitch = static_cast<int>((p.piece + 63) / 64 * 64);
    p.tile_n = width > 64 ? (terms == 1 && width > 128 ? 256 : 128) : 64;
    const int64_t n_tiles = ceil_div(width, p.tile_n);
    // both products' rows together: their depths keep the pairs busy
    p.pair = p.tile_n == 256 && pairs_fit(rows + p.piece, width, terms, sms);
    const int64_t tile_m = p.pair ? 2 * kTileM : kTileM, groups = p.pair ? sms / 2 : sms;
    const int64_t tiles[2] = {ceil_div(rows, tile_m) * n_tiles, ceil_div(p.piece, tile_m) * n_tiles};
    const int64_t depth[2] = {ceil_div(p.piece, kBlockK), ceil_div(rows, kBlockK)};
    // Splits of the depth: the smallest makespan in depth blocks, an item
    // costing 6 more for its start and its epilogue and a split 8 more for
    // the join; then the least to join.
    int64_t best = INT64_MAX;
    for (int s0 = 1; s0 <= 64 && s0 <= depth[0]; s0 = s0 < 4 ? s0 + 1 : s0 * 2)
        for (int s1 = 1; s1 <= 64 && s1 <= depth[1]; s1 = s1 < 4 ? s1 + 1 : s1 * 2) {
            const int64_t len[2] = {ceil_div(depth[0], s0), ceil_div(depth[1], s1)};
            const int64_t splits[2] = {ceil_div(depth[0], len[0]), ceil_div(depth[1], len[1])};
            const int64_t n[2] = {tiles[0] * splits[0], tiles[1] * splits[1]};
            const int64_t c[2] = {len[0] + 6 + (splits[0] > 1 ? 8 : 0), len[1] + 6 + (splits[1] > 1 ? 8 : 0)};
            const int f = len[0] >= len[1] ? 0 : 1;
            int64_t cost = 0;
            even_out(n[f], n[f ^ 1], c[f], c[f ^ 1], groups, &cost);
            // what is joined crosses HBM twice in f32: 1 depth block's time for 2 tiles or so
            cost += ((splits[0] > 1 ? n[0] : 0) + (splits[1] > 1 ? n[1] : 0)) / 16;
            if (cost < best) {
                best = cost;
                p.splits[0] = static_cast<int>(splits[0]);
                p.splits[1] = static_cast<int>(splits[1]);
            }
        }
    p.direct[0] = p.splits[0] == 1 && p.piece == k;
    p.direct[1] = p.splits[1] == 1;
    size_t at = 0;
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    p.xs = put(static_cast<size_t>(terms) * rows * p.pitch * 2);
    p.ws = put(static_cast<size_t>(terms) * k * p.pitch * 2);
    p.g = put(static_cast<size_t>(terms) * rows * p.g_pitch * 2);
    p.sums = put(static_cast<size_t>(ceil_div(rows, 256)) * 8 * p.piece * sizeof(float));  // rows of whole pair tiles
    p.part[0] = put(p.direct[0] ? 0 : static_cast<size_t>(p.splits[0]) * rows * width * sizeof(float));
    p.part[1] = put(p.direct[1] ? 0 : static_cast<size_t>(p.splits[1]) * p.piece * width * sizeof(float));
    p.bytes = at;
    return p;
}

// Lets every kernel of this file use its shared memory, once per device.
void allow_smem() {
    static std::mutex lock;
    static uint64_t done = 0;
    int device = 0;
    cuda_check(cudaGetDevice(&device));
    std::lock_guard<std::mutex> held(lock);
    if (device < 64 && (done >> device & 1)) return;
    auto allow = [](auto kernel, size_t bytes) {
        cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    };
    auto shape = [&](auto s) {
        using S = decltype(s);
        allow(logit_kernel<S, false>, S::kSmem);
        allow(logit_kernel<S, true>, S::kSmem);
        allow(product_kernel<S>, S::kSmem);
    };
    shape(Shape<1, false>{});
    shape(Shape<3, false>{});
    allow(product_kernel<Shape<1, true>>, Shape<1, true>::kSmem);
    if (device < 64) done |= uint64_t(1) << device;
}

// Launches a product kernel of shape S with `groups` CTAs or pairs.
template <class S, class Kernel, class... Args>
void launch_groups(Kernel kernel, int64_t groups, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(groups * S::kCtas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = S::kPair ? 2 : 1;
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...));
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, int kTerms>
void stage(const UnitLoss &a, int pitch, bool clean, __nv_bfloat16 *xs, __nv_bfloat16 *ws, int sms,
           cudaStream_t stream) {
    StageArgs s{a.x, a.units, a.bias, a.labels, a.rows, a.k, a.width, pitch, clean, false, xs, ws};
    s.wide = a.width % 8 == 0 && aligned16(a.x) && aligned16(a.units);
    const int64_t grid = std::min<int64_t>(ceil_div(a.rows + a.k, 8), 8 * sms);
    cuda_check(launch_pdl(stage_kernel<T, kTerms>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, s));
}

template <typename T, int kTerms>
void forward(const UnitLoss &a, int sms, cudaStream_t stream) {
    const ForwardPlan p = plan_forward(a.rows, a.k, a.width, a.dtype, sms);
    uint8_t *base = static_cast<uint8_t *>(a.workspace);
    auto *xs = reinterpret_cast<__nv_bfloat16 *>(base + p.xs);
    auto *ws = reinterpret_cast<__nv_bfloat16 *>(base + p.ws);
    const void *x = a.x, *w = a.units;
    int64_t pitch = a.width;
    if (kTerms > 1 || a.width % 8 || !aligned16(x) || !aligned16(w)) {
        stage<T, kTerms>(a, p.pitch, false, xs, ws, sms, stream);
        x = xs, w = ws, pitch = p.pitch;
    }
    const CUtensorMap map_x = map_k_major({x, a.width, a.rows, pitch, a.rows * pitch, kTerms}, kTileM);
    const CUtensorMap map_w = map_k_major({w, a.width, a.k, pitch, a.k * pitch, kTerms}, p.tile_n);
    LogitArgs l{};
    l.rows = a.rows, l.first = 0, l.count = a.k, l.k = a.k;
    l.k_blocks = static_cast<int32_t>(ceil_div(a.width, kBlockK));
    l.tile_n = p.tile_n, l.span = p.span, l.splits = p.splits;
    l.m_tiles = static_cast<int32_t>(p.m_tiles), l.n_tiles = static_cast<int32_t>(p.n_tiles);
    l.bias = a.bias, l.labels = a.labels, l.scale = a.scale;
    l.partial = reinterpret_cast<float2 *>(base + p.partial);
    l.target = reinterpret_cast<float *>(base + p.target);
    allow_smem();
    using S = Shape<kTerms, false>;
    launch_groups<S>(logit_kernel<S, false>, std::min<int64_t>(p.m_tiles * p.splits, sms), stream, map_x, map_w, map_x,
                     l);
    cuda_check(launch_pdl(loss_kernel, dim3(static_cast<unsigned>(ceil_div(a.rows, 32))), dim3(256), 0, stream,
                          static_cast<const float2 *>(l.partial), static_cast<const float *>(l.target), a.labels,
                          a.bias, a.rows, kParts * p.splits, static_cast<int>(a.k), a.loss, a.lse));
}

template <typename T, int kTerms>
void backward(const UnitLoss &a, int sms, cudaStream_t stream) {
    const BackwardPlan p = plan_backward(a.rows, a.k, a.width, a.dtype, sms);
    uint8_t *base = static_cast<uint8_t *>(a.workspace);
    auto *xs = reinterpret_cast<__nv_bfloat16 *>(base + p.xs);
    auto *ws = reinterpret_cast<__nv_bfloat16 *>(base + p.ws);
    stage<T, kTerms>(a, p.pitch, true, xs, ws, sms, stream);
    const int64_t pitch = p.pitch, plane = a.k * pitch;
    const Terms x{xs, a.width, a.rows, pitch, a.rows * pitch, kTerms};
    const CUtensorMap map_x = map_k_major(x, kTileM), map_xt = map_mn_major(x, p.pair ? 128 : p.tile_n);
    allow_smem();
    for (int64_t first = 0; first < a.k; first += p.piece) {
        const int64_t count = std::min<int64_t>(p.piece, a.k - first);
        const Terms g{base + p.g, count, a.rows, p.g_pitch, a.rows * p.g_pitch, kTerms};
        const Terms w{ws + first * pitch, a.width, count, pitch, plane, kTerms};
        LogitArgs l{};
        l.rows = a.rows, l.first = static_cast<int32_t>(first), l.count = static_cast<int32_t>(count), l.k = a.k;
        l.k_blocks = static_cast<int32_t>(ceil_div(a.width, kBlockK));
        l.m_tiles = static_cast<int32_t>(ceil_div(a.rows, kTileM));
        l.tile_n = tile_columns(l.m_tiles, count, kTerms, sms);
        l.n_tiles = static_cast<int32_t>(ceil_div(count, l.tile_n));
        l.span = item_span(l.m_tiles, l.n_tiles, sms);
        l.splits = static_cast<int32_t>(ceil_div(l.n_tiles, l.span));
        l.bias = a.bias, l.labels = a.labels, l.scale = a.scale;
        l.lse = a.lse_in, l.dloss = a.dloss;
        l.column_sums = a.dbias ? reinterpret_cast<float *>(base + p.sums) : nullptr;
        {
            using S = Shape<kTerms, false>;
            launch_groups<S>(logit_kernel<S, true>,
                             std::min<int64_t>(static_cast<int64_t>(l.m_tiles) * l.splits, sms), stream, map_x,
                             map_k_major(w, l.tile_n), map_store(g, l.tile_n == 256 ? 64 : 32), l);
        }
        ProductArgs q{};
        q.width = a.width, q.tile_n = p.tile_n;
        q.n_tiles = static_cast<int32_t>(ceil_div(a.width, p.tile_n));
        q.scale = a.scale, q.bf16 = a.dtype == kBF16;
        const int64_t depth[2] = {ceil_div(count, kBlockK), ceil_div(a.rows, kBlockK)};
        const int64_t size[2] = {a.rows, count};
        T *dunits = static_cast<T *>(a.dunits) + first * a.width;
        void *out[2] = {a.dx, dunits};
        q.wide = a.width % 8 == 0 && aligned16(a.dx) && aligned16(dunits);
        for (int i = 0; i < 2; ++i) {
            auto &o = q.one[i];
            o.m_size = static_cast<int32_t>(size[i]);
            o.m_tiles = static_cast<int32_t>(ceil_div(size[i], p.pair ? 2 * kTileM : kTileM));
            o.k_blocks = static_cast<int32_t>(depth[i]);
            // the last piece is shorter: its splits are too, and all of them exist
            o.splits = static_cast<int32_t>(std::min<int64_t>(p.splits[i], depth[i]));
            o.split_blocks = static_cast<int32_t>(ceil_div(depth[i], o.splits));
            o.splits = static_cast<int32_t>(ceil_div(depth[i], o.split_blocks));
            o.items = static_cast<uint32_t>(o.m_tiles) * q.n_tiles * o.splits;
            o.out = out[i];
            o.part = p.direct[i] ? nullptr : reinterpret_cast<float *>(base + p.part[i]);
            o.add = i == 0 && first > 0;
            o.part_stride = size[i] * a.width;
        }
        q.first_product = q.one[0].split_blocks >= q.one[1].split_blocks ? 0 : 1;
        const int64_t tiles = static_cast<int64_t>(q.one[0].items) + q.one[1].items;
        const int64_t groups = std::min<int64_t>(tiles, p.pair ? sms / 2 : sms);
        const auto &slow = q.one[q.first_product], &brief = q.one[q.first_product ^ 1];
        int64_t makespan = 0;
        q.odd = static_cast<uint32_t>(slow.items % groups);
        q.extra = static_cast<uint32_t>(
            even_out(slow.items, brief.items, slow.split_blocks + 6, brief.split_blocks + 6, groups, &makespan));
        if (p.pair) {
            if constexpr (kTerms == 1) {
                using S = Shape<1, true>;
                launch_groups<S>(product_kernel<S>, groups, stream, map_k_major(g, kTileM),
                                 map_mn_major(g, kTileM), map_mn_major(w, 128), map_xt, q);
            }
        } else {
            using S = Shape<kTerms, false>;
            launch_groups<S>(product_kernel<S>, groups, stream, map_k_major(g, kTileM),
                             map_mn_major(g, kTileM), map_mn_major(w, p.tile_n), map_xt, q);
        }
        FinishArgs f{};
        for (int i = 0; i < 2; ++i) {
            // dx waits for the last piece
            if (p.direct[i] || (i == 0 && first + count < a.k)) continue;
            const int64_t n = size[i] * a.width;
            f.join[i] = {q.one[i].part, q.one[i].part_stride, n, i == 0 ? p.splits[0] : q.one[i].splits,
                         static_cast<unsigned>(std::min<int64_t>(ceil_div(n, kFinishThreads), 4 * sms)), q.one[i].out};
        }
        if (a.dbias) {
            f.sums = l.column_sums, f.parts = ceil_div(a.rows, 32), f.columns = static_cast<int32_t>(count);
            f.sum_blocks = static_cast<unsigned>(ceil_div(count, 32)), f.dbias = a.dbias + first;
        }
        const unsigned blocks = f.sum_blocks + f.join[0].blocks + f.join[1].blocks;
        if (blocks)
            cuda_check(launch_pdl(finish_kernel<T>, dim3(blocks), dim3(kFinishThreads), 0, stream, f));
    }
}

}  // namespace

size_t unit_loss_workspace(int64_t rows, int k, int width, int dtype, bool backward, int sms) {
    return backward ? plan_backward(rows, k, width, dtype, sms).bytes
                    : plan_forward(rows, k, width, dtype, sms).bytes;
}

void launch_unit_loss(const UnitLoss &a, int sms, cudaStream_t stream) {
    if (a.dtype == kF32) forward<float, 3>(a, sms, stream);
    else forward<__nv_bfloat16, 1>(a, sms, stream);
}

void launch_unit_loss_backward(const UnitLoss &a, int sms, cudaStream_t stream) {
    if (a.dtype == kF32) backward<float, 3>(a, sms, stream);
    else backward<__nv_bfloat16, 1>(a, sms, stream);
}

}  // namespace vfr
