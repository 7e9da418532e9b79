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
constexpr int kBox = 64;         // rows of every load's box
constexpr uint32_t kBoxBytes = kBox * kBlockK * 2;
constexpr int kEpiWarps = 8;     // two per lane quarter, each on half of a tile's columns
constexpr int kThreads = 64 + 32 * kEpiWarps;  // warp 0 loads, warp 1 issues MMAs
constexpr int kGroupM = 16;      // row tiles that share the units they read
constexpr uint32_t kTmemCols = 512;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;

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
template <int kTerms>
struct Shape {
    static constexpr int kTileN = kTerms == 1 ? 256 : 128;
    static constexpr int kStages = kTerms == 1 ? 4 : 2;
    static constexpr uint32_t kABytes = 2 * kBoxBytes;
    static constexpr uint32_t kBBytes = kTileN / kBox * kBoxBytes;
    static constexpr uint32_t kStageBytes = kTerms * (kABytes + kBBytes);
    static constexpr uint32_t kStagingOff = kStages * kStageBytes;
    static constexpr uint32_t kBiasOff = kStagingOff + kEpiWarps * 2048;
    static constexpr uint32_t kBarOff = kBiasOff + kEpiWarps * 128;
    static constexpr size_t kSmem = 1024 + kBarOff + 256;
    // Depth blocks summed in tensor memory before f32 registers take over:
    // the accumulator truncates, so f32 results add up short runs.
    static constexpr int kChunk = kTerms == 1 ? 1 << 30 : 8;
    static_assert(kSmem <= 232448, "shared memory");
};

// A tile of a product: rows m0.., columns n0.. (n_cols of them, a multiple of
// 16), depth blocks [k0, k1).  K-major operands are loaded at (k, row),
// MN-major ones at (row, k).
struct Tile {
    const CUtensorMap *a, *b;
    bool a_mn, b_mn;
    int32_t m0, n0, n_cols, a_boxes;
    int32_t k0, k1;
};

struct Bars {
    uint64_t *full, *empty, *acc_full, *acc_empty;
    uint32_t *tmem_slot;
    volatile int *abort_flag;
};

template <int kTerms>
__device__ __forceinline__ Bars bars_at(uint8_t *smem) {
    using S = Shape<kTerms>;
    Bars b;
    b.full = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
    b.empty = b.full + S::kStages;
    b.acc_full = b.empty + S::kStages;
    b.acc_empty = b.acc_full + 2;
    b.tmem_slot = reinterpret_cast<uint32_t *>(b.acc_empty + 2);
    b.abort_flag = reinterpret_cast<volatile int *>(b.tmem_slot + 1);
    return b;
}

// Producer lane: every tile's operand blocks through the stages.  `tile(i, t)`
// gives the CTA's i-th tile, false past the last.
template <int kTerms, class TileAt>
__device__ __forceinline__ void produce(uint8_t *smem, const Bars &bars, TileAt tile) {
    using S = Shape<kTerms>;
    int stage = 0;
    uint32_t phase = 0;
    Tile t;
    for (int64_t i = 0; tile(i, t) && !*bars.abort_flag; ++i) {
        const int b_boxes = (t.n_cols + kBox - 1) / kBox;
        const uint32_t bytes = kTerms * (t.a_boxes + b_boxes) * kBoxBytes;
        for (int k = t.k0; k < t.k1; ++k) {
            if (!tc::mbar_wait(&bars.empty[stage], phase ^ 1, kWaitLimitNs)) {
                *bars.abort_flag = 1;
                break;
            }
            tc::mbar_arrive_expect_tx(&bars.full[stage], bytes);
            uint8_t *sa = smem + stage * S::kStageBytes, *sb = sa + kTerms * S::kABytes;
            const int32_t kk = k * kBlockK;
#pragma unroll
            for (int p = 0; p < kTerms; ++p) {
                for (int j = 0; j < t.a_boxes; ++j) {
                    const int32_t r = t.m0 + j * kBox;
                    tc::tma_load_3d(sa + p * S::kABytes + j * kBoxBytes, t.a, &bars.full[stage], t.a_mn ? r : kk,
                                    t.a_mn ? kk : r, p);
                }
                for (int j = 0; j < b_boxes; ++j) {
                    const int32_t r = t.n0 + j * kBox;
                    tc::tma_load_3d(sb + p * S::kBBytes + j * kBoxBytes, t.b, &bars.full[stage], t.b_mn ? r : kk,
                                    t.b_mn ? kk : r, p);
                }
            }
            if (++stage == S::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    }
    // let every issued copy land before the CTA can exit
    for (int s = 0; s < S::kStages; ++s) {
        if (!tc::mbar_wait(&bars.empty[stage], phase ^ 1, kWaitLimitNs)) break;
        if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
        }
    }
}

// MMA lane.  Accumulator buffer b of a chunk: TMEM columns 256 b (the
// product, or hi hi) and 256 b + 128 (the other terms' products).
template <int kTerms, class TileAt>
__device__ __forceinline__ void multiply(uint8_t *smem, const Bars &bars, uint32_t tmem, TileAt tile) {
    using S = Shape<kTerms>;
    int stage = 0;
    uint32_t phase = 0, acc_count = 0;
    Tile t;
    for (int64_t i = 0; tile(i, t) && !*bars.abort_flag; ++i) {
        const uint32_t idesc = tc::idesc_f16(kTileM, t.n_cols, 1) | (t.a_mn ? tc::kIdescMnA : 0) |
                               (t.b_mn ? tc::kIdescMnB : 0);
        const uint32_t a_step = t.a_mn ? 2048 : 32, b_step = t.b_mn ? 2048 : 32;
        for (int k = t.k0; k < t.k1;) {
            const int chunk = t.k1 - k > S::kChunk ? k + S::kChunk : t.k1;
            const uint32_t b = acc_count & 1;
            if (!tc::mbar_wait(&bars.acc_empty[b], ((acc_count >> 1) & 1) ^ 1, kWaitLimitNs)) {
                *bars.abort_flag = 1;
                return;
            }
            tc::tc_fence_after();
            const uint32_t d = tmem + b * 256;
            uint32_t big = 0, rest = 0;  // whether each accumulator holds a sum
            for (; k < chunk; ++k) {
                if (!tc::mbar_wait(&bars.full[stage], phase, kWaitLimitNs)) {
                    *bars.abort_flag = 1;
                    return;
                }
                tc::tc_fence_after();
                const uint32_t sa = tc::smem_u32(smem + stage * S::kStageBytes), sb = sa + kTerms * S::kABytes;
                auto product = [&](uint32_t acc, int pa, int pb, uint32_t &held) {
#pragma unroll
                    for (int kk = 0; kk < kBlockK / 16; ++kk) {
                        const uint32_t xa = sa + pa * S::kABytes + kk * a_step;
                        const uint32_t xb = sb + pb * S::kBBytes + kk * b_step;
                        tc::mma_f16(acc,
                                    t.a_mn ? tc::smem_desc_sw128_mn(xa, kBoxBytes) : tc::smem_desc_sw128(xa),
                                    t.b_mn ? tc::smem_desc_sw128_mn(xb, kBoxBytes) : tc::smem_desc_sw128(xb), idesc,
                                    held);
                        held = 1;
                    }
                };
                if constexpr (kTerms == 1) {
                    product(d, 0, 0, big);
                } else {
                    product(d + 128, 0, 2, rest);
                    product(d + 128, 2, 0, rest);
                    product(d + 128, 1, 1, rest);
                    product(d + 128, 0, 1, rest);
                    product(d + 128, 1, 0, rest);
                    product(d, 0, 0, big);
                }
                tc::mma_commit(&bars.empty[stage]);
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            tc::mma_commit(&bars.acc_full[b]);
            ++acc_count;
        }
    }
}

// Epilogue warps: `take(j, v)` gives this lane's row, columns 32 j .. of the
// warp's half of the tile; all NaN once a wait gave up, so that no result of
// a call that went wrong looks like one.
template <int kTerms>
struct Columns {
    using S = Shape<kTerms>;
    static constexpr int kMax = S::kTileN / 2 / 32;  // 32-column chunks of a half
    float run[kTerms == 1 ? 1 : S::kTileN / 2];
    uint32_t acc_count = 0;
    bool bad = false;

    // Waits for the tile's accumulator (f32: adds up the tile's chunks).
    __device__ __forceinline__ void open(const Bars &bars, uint32_t tmem, uint32_t half_at, int chunks, int depth) {
        if constexpr (kTerms == 1) {
            wait(bars);
        } else {
#pragma unroll
            for (int i = 0; i < S::kTileN / 2; ++i) run[i] = 0.0f;
            for (int k = 0; k < depth; k += S::kChunk) {
                wait(bars);
                const uint32_t at = tmem + half_at + (acc_count & 1) * 256;
#pragma unroll
                for (int j = 0; j < kMax; ++j) {
                    if (j < chunks) {
                        float v[32];
                        if (!bad) tc::tmem_ld32(at + 32 * j + 128, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) run[32 * j + i] += v[i];
                        if (!bad) tc::tmem_ld32(at + 32 * j, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) run[32 * j + i] += v[i];
                    }
                }
                release(bars);
            }
        }
    }
    __device__ __forceinline__ void take(uint32_t tmem, uint32_t half_at, int j, float (&v)[32]) {
        if constexpr (kTerms == 1) {
            if (!bad) tc::tmem_ld32(tmem + half_at + (acc_count & 1) * 256 + 32 * j, v);
        } else {
#pragma unroll
            for (int c = 0; c < kMax; ++c)
                if (c == j)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = run[32 * c + i];
        }
        if (bad)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = NAN;
    }
    // The tile's last chunk has been taken.
    __device__ __forceinline__ void close(const Bars &bars) {
        if constexpr (kTerms == 1) release(bars);
    }

private:
    __device__ __forceinline__ void wait(const Bars &bars) {
        if (!bad && !tc::mbar_wait(&bars.acc_full[acc_count & 1], (acc_count >> 1) & 1, kWaitLimitNs)) {
            *bars.abort_flag = 1;
            bad = true;
        }
        bad = __any_sync(0xFFFFFFFFu, bad);
        tc::tc_fence_after();
    }
    __device__ __forceinline__ void release(const Bars &bars) {
        tc::tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&bars.acc_empty[acc_count & 1]);
        ++acc_count;
    }
};

// The kernel around the roles: barriers, TMEM, and the epilogue
// `epi(smem, bars, tmem, warp of the epilogue, lane)`.
template <int kTerms, class TileAt, class Epi>
__device__ __forceinline__ void run_roles(TileAt tile, Epi epi) {
    using S = Shape<kTerms>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const Bars bars = bars_at<kTerms>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tc::mbar_init(&bars.full[s], 1);
            tc::mbar_init(&bars.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&bars.acc_full[b], 1);
            tc::mbar_init(&bars.acc_empty[b], kEpiWarps);
        }
        *bars.abort_flag = 0;
        tc::fence_mbarrier_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(bars.tmem_slot, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *bars.tmem_slot;
    grid_dependency_wait();
    if (warp == 0) {
        if (lane == 0) produce<kTerms>(smem, bars, tile);
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) multiply<kTerms>(smem, bars, tmem, tile);
        __syncwarp();
    } else {
        epi(smem, bars, tmem, warp, lane);
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, kTmemCols);
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
    float2 *partial;  // [2 splits][rows] (maximum, sum)
    float *target;    // [rows] logit of the label
    // backward
    const float *lse, *dloss;
    float *column_sums;  // [4 m_tiles][count] or null
};

// Item i: row tiles in groups of kGroupM, the items of a group by columns
// first, so that the CTAs of a wave share kGroupM row tiles and few units.
__device__ __forceinline__ void item_at(const LogitArgs &a, int64_t item, int &m, int &split) {
    const int64_t group = item / (static_cast<int64_t>(kGroupM) * a.splits);
    const int64_t rest = item - group * kGroupM * a.splits;
    const int rows = min(kGroupM, a.m_tiles - static_cast<int>(group) * kGroupM);
    split = static_cast<int>(rest / rows);
    m = static_cast<int>(group) * kGroupM + static_cast<int>(rest % rows);
}

template <int kTerms, bool kBackward>
__global__ void __launch_bounds__(kThreads, 1)
    logit_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_g, const LogitArgs a) {
    using S = Shape<kTerms>;
    const int64_t items = static_cast<int64_t>(a.m_tiles) * a.splits;
    auto tile = [&](int64_t i, Tile &t) {
        const int64_t item = blockIdx.x + (i / a.span) * gridDim.x;
        if (item >= items) return false;
        int m, split;
        item_at(a, item, m, split);
        const int n = split * a.span + static_cast<int>(i % a.span);
        t.a = &map_x, t.b = &map_w, t.a_mn = t.b_mn = false;
        t.m0 = m * kTileM;
        t.a_boxes = a.rows - t.m0 > kBox ? 2 : 1;
        const int at = n * a.tile_n;
        t.n0 = at;  // map_w covers the launch's units
        t.n_cols = min(a.tile_n, (max(a.count - at, 1) + 15) / 16 * 16);
        t.k0 = 0;
        t.k1 = n < a.n_tiles ? a.k_blocks : 0;  // the last item of a row may be short
        return true;
    };
    run_roles<kTerms>(tile, [&](uint8_t *smem, const Bars &bars, uint32_t tmem, int warp, int lane) {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        float *bias_slot = reinterpret_cast<float *>(smem + S::kBiasOff) + (warp - 2) * 32;
        uint8_t *staging = smem + S::kStagingOff + (warp - 2) * 2048;
        const int half_cols = a.tile_n / 2, chunks = half_cols / 32;
        const uint32_t half_at = (static_cast<uint32_t>(quarter * 32) << 16) + half * half_cols;
        Columns<kTerms> columns;
        for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
            int m, split;
            item_at(a, item, m, split);
            const int64_t row = static_cast<int64_t>(m) * kTileM + quarter * 32 + lane;
            const bool live = row < a.rows;
            int32_t label = live ? a.labels[row] : -1;
            if (label >= a.k) label = -1;
            const bool valid = label >= 0;
            float top = -INFINITY, sum = 0.0f;  // forward
            float lse = 0.0f, grad = 0.0f;      // backward
            if constexpr (kBackward) {
                if (valid) {
                    lse = a.lse[row];
                    grad = a.dloss[row];
                }
            }
            for (int n = split * a.span; n < min((split + 1) * a.span, a.n_tiles); ++n) {
                const int col0 = n * a.tile_n + half * half_cols;  // within the launch's units
                float bias[Columns<kTerms>::kMax];
#pragma unroll
                for (int j = 0; j < Columns<kTerms>::kMax; ++j) {
                    const int c = col0 + 32 * j + lane;
                    bias[j] = c >= a.count ? -INFINITY : a.bias ? __ldg(a.bias + a.first + c) : 0.0f;
                }
                columns.open(bars, tmem, half_at, chunks, a.k_blocks);
#pragma unroll
                for (int j = 0; j < Columns<kTerms>::kMax; ++j) {
                    if (j >= chunks) break;
                    const int col = col0 + 32 * j;
                    float v[32];
                    columns.take(tmem, half_at, j, v);
                    if (a.bias) {
                        __syncwarp();
                        bias_slot[lane] = bias[j];
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = fmaf(v[i], a.scale, bias_slot[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= a.scale;
                    }
                    // units left out and columns past the last: -inf whatever the product is
                    const uint32_t out = __ballot_sync(0xFFFFFFFFu, bias[j] == -INFINITY);
                    if (out) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (out >> i & 1) v[i] = -INFINITY;
                    }
                    const int hit = label - a.first - col;  // the label's column in this chunk
                    const bool mine = valid && hit >= 0 && hit < 32;
                    if constexpr (!kBackward) {
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i == hit) a.target[row] = v[i];
                        }
                        float m8[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(fmaxf(v[i], v[i + 8]), fmaxf(v[i + 16], v[i + 24]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) m8[i] = fmaxf(m8[i], m8[i + 4]);
                        const float next = fmaxf(top, fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])));
                        const float base = next == -INFINITY ? 0.0f : next;
                        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < 32; ++i) s4[i & 3] += exp2_approx((v[i] - base) * kLog2e);
                        sum = fmaf(sum, exp2_approx((top - base) * kLog2e), (s4[0] + s4[1]) + (s4[2] + s4[3]));
                        top = next;
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = exp2_approx((v[i] - lse) * kLog2e);
                        if (mine && !(out >> hit & 1)) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i == hit) v[i] -= 1.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= grad;
                        if (!valid) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                        }
                        if (out) {  // 0, also where lse is -inf
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (out >> i & 1) v[i] = 0.0f;
                        }
                        if (a.column_sums) {
                            // lane i ends with column i's sum over the warp's 32 rows
                            float s[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[i] = v[i];
#pragma unroll
                            for (int o = 16; o; o >>= 1) {
                                const bool upper = lane & o;
#pragma unroll
                                for (int i = 0; i < o; ++i) {
                                    const float keep = upper ? s[i + o] : s[i];
                                    s[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, upper ? s[i] : s[i + o], o);
                                }
                            }
                            if (col + lane < a.count)
                                a.column_sums[(static_cast<int64_t>(m) * 4 + quarter) * a.count + col + lane] = s[0];
                        }
                        // G in bf16 (f32: three terms): a factor of its own
                        // products, rounded as any operand of theirs
#pragma unroll
                        for (int p = 0; p < kTerms; ++p) {
                            tc::bulk_wait_read<0>();
                            __syncwarp();
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int i = 8 * c + 2 * e;
                                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[i], v[i + 1]);
                                    w[e] = *reinterpret_cast<const uint32_t *>(&b);
                                    if (p + 1 < kTerms) {
                                        const float2 f = __bfloat1622float2(b);
                                        v[i] -= f.x;
                                        v[i + 1] -= f.y;
                                    }
                                }
                                // 64-byte rows, 16-byte units swizzled as SWIZZLE_64B expects
                                *reinterpret_cast<uint4 *>(staging + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
                                    make_uint4(w[0], w[1], w[2], w[3]);
                            }
                            tc::fence_proxy_async_smem();
                            __syncwarp();
                            const int64_t row0 = static_cast<int64_t>(m) * kTileM + quarter * 32;
                            if (lane == 0 && col < a.count && row0 < a.rows) {
                                tc::tma_store_3d(&map_g, staging, col, static_cast<int32_t>(row0), p);
                                tc::bulk_commit();
                            }
                        }
                    }
                }
                columns.close(bars);
            }
            if constexpr (!kBackward) {
                if (live) a.partial[(static_cast<int64_t>(split) * 2 + half) * a.rows + row] = make_float2(top, sum);
            }
        }
        if constexpr (kBackward) {
            if (lane == 0) tc::bulk_wait_all();
            __syncwarp();
        }
    });
}

// Joins the slots of each row.
__global__ void __launch_bounds__(256) loss_kernel(const float2 *partial, const float *target, const int32_t *labels,
                                                   int64_t rows, int slots, int k, float *loss, float *lse) {
    grid_dependency_wait();
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (row >= rows) return;
    float top = -INFINITY, sum = 0.0f;
    for (int s = 0; s < slots; ++s) {
        const float2 p = partial[static_cast<int64_t>(s) * rows + row];
        const float next = fmaxf(top, p.x);
        const float base = next == -INFINITY ? 0.0f : next;
        sum = sum * exp2_approx((top - base) * kLog2e) + p.y * exp2_approx((p.x - base) * kLog2e);
        top = next;
    }
    const float l = top == -INFINITY && sum == 0.0f ? top : top + logf(sum);
    lse[row] = l;
    const int32_t t = labels[row];
    if (t < 0 || t >= k) {
        loss[row] = 0.0f;
    } else {
        const float z = target[row];
        loss[row] = z == -INFINITY ? INFINITY : l - z;
    }
}

// ---------------------------------------------------------------- products

// dx (product 0: G [rows][count] times the units) and dunits (product 1: G^T
// times the frames) of one piece, in one launch.
struct ProductArgs {
    struct One {
        int32_t m_size, m_tiles;  // rows of the result
        int32_t k_blocks, splits, split_blocks;
        int64_t items;
        void *out;            // the result, where a tile has all of its sum
        float *part;          // else f32 [splits][m_size][width]
        bool add;             // to what `part` holds from the pieces before
        int64_t part_stride;
    } one[2];
    int32_t width, n_tiles, tile_n;
    int32_t first_product;  // whose items come first: the longer ones
    float scale;
    bool bf16, wide;        // result type; 16-byte stores fit
};

struct ProductItem {
    int which, m, n, split;
};
__device__ __forceinline__ bool product_at(const ProductArgs &a, int64_t item, ProductItem &p) {
    p.which = a.first_product;
    if (item >= a.one[p.which].items) {
        item -= a.one[p.which].items;
        p.which ^= 1;
        if (item >= a.one[p.which].items) return false;
    }
    const auto &o = a.one[p.which];
    // columns first, then splits: neighbours share their rows of G
    p.n = static_cast<int>(item % a.n_tiles);
    const int64_t rest = item / a.n_tiles;
    p.m = static_cast<int>(rest % o.m_tiles);
    p.split = static_cast<int>(rest / o.m_tiles);
    return true;
}

template <int kTerms>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_w, const ProductArgs a) {
    auto tile = [&](int64_t i, Tile &t) {
        ProductItem p;
        if (!product_at(a, blockIdx.x + i * gridDim.x, p)) return false;
        const auto &o = a.one[p.which];
        t.a = &map_g, t.b = p.which == 0 ? &map_w : &map_x;
        t.a_mn = p.which == 1, t.b_mn = true;
        t.m0 = p.m * kTileM;
        t.a_boxes = o.m_size - t.m0 > kBox ? 2 : 1;
        t.n0 = p.n * a.tile_n;
        t.n_cols = min(a.tile_n, (a.width - t.n0 + 15) / 16 * 16);
        t.k0 = p.split * o.split_blocks;
        t.k1 = min(o.k_blocks, t.k0 + o.split_blocks);
        return true;
    };
    run_roles<kTerms>(tile, [&](uint8_t *, const Bars &bars, uint32_t tmem, int warp, int lane) {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int half_cols = a.tile_n / 2, chunks = half_cols / 32;
        const uint32_t half_at = (static_cast<uint32_t>(quarter * 32) << 16) + half * half_cols;
        Columns<kTerms> columns;
        ProductItem p;
        for (int64_t item = blockIdx.x; product_at(a, item, p); item += gridDim.x) {
            const auto &o = a.one[p.which];
            const int k0 = p.split * o.split_blocks;
            columns.open(bars, tmem, half_at, chunks, min(o.k_blocks, k0 + o.split_blocks) - k0);
            const int64_t row = static_cast<int64_t>(p.m) * kTileM + quarter * 32 + lane;
#pragma unroll
            for (int j = 0; j < Columns<kTerms>::kMax; ++j) {
                if (j >= chunks) break;
                float v[32];
                columns.take(tmem, half_at, j, v);
                const int col = p.n * a.tile_n + half * half_cols + 32 * j;
                if (row >= o.m_size || col >= a.width) continue;
                const int64_t at = row * a.width + col;
                if (o.part == nullptr) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] *= a.scale;
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
            columns.close(bars);
        }
    });
}

// out[i] = scale * sum over the splits of part[s][i], in split order.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float *part, int64_t stride, int splits, int64_t count,
                                                   float scale, T *out) {
    launch_dependents();
    grid_dependency_wait();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        float s = 0.0f;
        for (int k = 0; k < splits; ++k) s += part[k * stride + i];
        out[i] = from_f32<T>(s * scale);
    }
}

// dbias from the row tiles' column sums, in order: 32 columns a CTA, 8 warps over the rows.
__global__ void __launch_bounds__(256) dbias_kernel(const float *sums, int64_t parts, int32_t count, float *out) {
    __shared__ float slots[8][32];
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < count)
        for (int64_t p = warp; p < parts; p += 8) s += sums[p * count + col];
    slots[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && col < count) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += slots[i][lane];
        out[col] = s;
    }
}

// ---------------------------------------------------------------- operands

// The products' operands: rows of bf16 terms, padded to whole 16-byte units.
// With `clean`, frames without a label and units left out become zero rows:
// a zero of G times an infinity or a NaN there would reach the gradients.
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
                for (int i = 0; i < 8; i += kVec) load_vec<T, kVec>(src + c + i, v + i);
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

// bf16 terms of [rows][pitch], `plane` elements apart, of which `cols`
// columns count; boxes of 64
// rows by 64 columns (loads) or 32 by 32 (G's stores).  What lies outside
// reads as zero and is not written.
CUtensorMap terms_map(const void *base, int64_t cols, int64_t rows, int64_t pitch, int64_t plane, int terms,
                      bool store = false) {
    require(reinterpret_cast<uintptr_t>(base) % 16 == 0 && pitch % 8 == 0, "tensor map alignment");
    CUtensorMap map;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                          static_cast<cuuint64_t>(terms)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch) * 2, static_cast<cuuint64_t>(plane) * 2};
    const cuuint32_t side = store ? 32 : kBox;
    cuuint32_t box[3] = {side, side, 1}, estr[3] = {1, 1, 1};
    const CUresult rc = encode_fn()(
        &map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
        CU_TENSOR_MAP_INTERLEAVE_NONE, store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    require(rc == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed");
    return map;
}

// ---------------------------------------------------------------- plans

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
int terms_of(int dtype) { return dtype == kF32 ? 3 : 1; }

// Columns of a tile: the widest that still gives every SM a tile.
int tile_columns(int64_t m_tiles, int64_t cols, int terms, int sms) {
    int n = terms == 1 ? 256 : 128;
    while (n > 64 && m_tiles * ceil_div(cols, n) < sms) n /= 2;
    return n;
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
    // items of `span` column tiles: the fewest rounds of the grid, then the fewest items
    int64_t best = INT64_MAX;
    for (int64_t s = 1; s <= std::min<int64_t>(p.n_tiles, 64); ++s) {
        const int64_t span = ceil_div(p.n_tiles, s);
        const int64_t cost = ceil_div(p.m_tiles * ceil_div(p.n_tiles, span), sms) * span;
        if (cost < best) {
            best = cost;
            p.span = static_cast<int>(span);
        }
    }
    p.splits = static_cast<int>(ceil_div(p.n_tiles, p.span));
    p.pitch = (width + 7) / 8 * 8;
    size_t at = 0;
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    p.xs = put(static_cast<size_t>(terms) * rows * p.pitch * 2);
    p.ws = put(static_cast<size_t>(terms) * k * p.pitch * 2);
    p.partial = put(static_cast<size_t>(2) * p.splits * rows * sizeof(float2));
    p.target = put(static_cast<size_t>(rows) * sizeof(float));
    p.bytes = at;
    return p;
}

struct BackwardPlan {
    int64_t piece;  // units of a piece
    int64_t m_tiles;
    int pitch, g_pitch, tile_n;  // tile_n: of the gradients' columns
    int splits[2];
    bool direct[2];
    size_t xs, ws, g, sums, part[2], bytes;
};
// Bytes of G in the workspace, unless 256 units of every frame take more.
constexpr int64_t kPieceBytes = int64_t(256) << 20;

BackwardPlan plan_backward(int64_t rows, int k, int width, int dtype, int sms) {
    const int terms = terms_of(dtype);
    BackwardPlan p{};
    const int64_t fit = kPieceBytes / (std::max<int64_t>(rows, 1) * 2 * terms) / 256 * 256;
    p.piece = std::min<int64_t>(k, std::max<int64_t>(256, fit));
    p.m_tiles = ceil_div(rows, kTileM);
    p.pitch = (width + 7) / 8 * 8;
    p.g_pitch = static_cast<int>((p.piece + 63) / 64 * 64);
    p.tile_n = width > 64 ? (terms == 1 && width > 128 ? 256 : 128) : 64;
    const int64_t n_tiles = ceil_div(width, p.tile_n);
    const int64_t tiles[2] = {p.m_tiles * n_tiles, ceil_div(p.piece, kTileM) * n_tiles};
    const int64_t depth[2] = {ceil_div(p.piece, kBlockK), ceil_div(rows, kBlockK)};
    // Splits of the depth: the smallest round-robin makespan in depth blocks,
    // an item costing 6 more for its start and its epilogue and a split 4
    // more for the join.
    int64_t best = INT64_MAX;
    for (int s0 = 1; s0 <= 64 && s0 <= depth[0]; s0 = s0 < 4 ? s0 + 1 : s0 * 2)
        for (int s1 = 1; s1 <= 64 && s1 <= depth[1]; s1 = s1 < 4 ? s1 + 1 : s1 * 2) {
            const int64_t len[2] = {ceil_div(depth[0], s0), ceil_div(depth[1], s1)};
            const int f = len[0] >= len[1] ? 0 : 1;
            const int64_t n[2] = {tiles[0] * ceil_div(depth[0], len[0]), tiles[1] * ceil_div(depth[1], len[1])};
            const int64_t joined[2] = {ceil_div(depth[0], len[0]) > 1 ? 4 : 0, ceil_div(depth[1], len[1]) > 1 ? 4 : 0};
            const int64_t c[2] = {len[0] + 6 + joined[0], len[1] + 6 + joined[1]};
            int64_t cost = 0;
            for (int64_t cta : {int64_t(0), n[f] % sms}) {
                const int64_t own = n[f] > cta ? (n[f] - 1 - cta) / sms + 1 : 0;
                const int64_t all = n[0] + n[1] > cta ? (n[0] + n[1] - 1 - cta) / sms + 1 : 0;
                cost = std::max(cost, own * c[f] + (all - own) * c[f ^ 1]);
            }
            cost = cost * 8 + joined[0] + joined[1];
            if (cost < best) {
                best = cost;
                p.splits[0] = static_cast<int>(ceil_div(depth[0], len[0]));
                p.splits[1] = static_cast<int>(ceil_div(depth[1], len[1]));
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
    p.sums = put(static_cast<size_t>(4) * p.m_tiles * p.piece * sizeof(float));
    p.part[0] = put(p.direct[0] ? 0 : static_cast<size_t>(p.splits[0]) * rows * width * sizeof(float));
    p.part[1] = put(p.direct[1] ? 0 : static_cast<size_t>(p.splits[1]) * p.piece * width * sizeof(float));
    p.bytes = at;
    return p;
}

template <class K>
void allow_smem(K kernel, size_t bytes) {
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
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
    if (kTerms > 1 || a.width % 8 || !aligned16(x) || !aligned16(w)) {
        stage<T, kTerms>(a, p.pitch, false, xs, ws, sms, stream);
        x = xs, w = ws;
    }
    const int64_t plane = static_cast<int64_t>(a.k) * p.pitch;
    const CUtensorMap map_x = terms_map(x, a.width, a.rows, p.pitch, a.rows * p.pitch, kTerms);
    const CUtensorMap map_w = terms_map(w, a.width, a.k, p.pitch, plane, kTerms);
    LogitArgs l{};
    l.rows = a.rows, l.first = 0, l.count = a.k, l.k = a.k;
    l.k_blocks = static_cast<int32_t>(ceil_div(a.width, kBlockK));
    l.tile_n = p.tile_n, l.span = p.span, l.splits = p.splits;
    l.m_tiles = static_cast<int32_t>(p.m_tiles), l.n_tiles = static_cast<int32_t>(p.n_tiles);
    l.bias = a.bias, l.labels = a.labels, l.scale = a.scale;
    l.partial = reinterpret_cast<float2 *>(base + p.partial);
    l.target = reinterpret_cast<float *>(base + p.target);
    allow_smem(logit_kernel<kTerms, false>, Shape<kTerms>::kSmem);
    const int64_t grid = std::min<int64_t>(p.m_tiles * p.splits, sms);
    cuda_check(launch_pdl(logit_kernel<kTerms, false>, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                          Shape<kTerms>::kSmem, stream, map_x, map_w, map_x, l));
    cuda_check(launch_pdl(loss_kernel, dim3(static_cast<unsigned>(ceil_div(a.rows, 256))), dim3(256), 0, stream,
                          static_cast<const float2 *>(l.partial), static_cast<const float *>(l.target), a.labels,
                          a.rows, 2 * p.splits, static_cast<int>(a.k), a.loss, a.lse));
}

template <typename T, int kTerms>
void backward(const UnitLoss &a, int sms, cudaStream_t stream) {
    const BackwardPlan p = plan_backward(a.rows, a.k, a.width, a.dtype, sms);
    uint8_t *base = static_cast<uint8_t *>(a.workspace);
    auto *xs = reinterpret_cast<__nv_bfloat16 *>(base + p.xs);
    auto *ws = reinterpret_cast<__nv_bfloat16 *>(base + p.ws);
    stage<T, kTerms>(a, p.pitch, true, xs, ws, sms, stream);
    const CUtensorMap map_x = terms_map(xs, a.width, a.rows, p.pitch, a.rows * p.pitch, kTerms);
    allow_smem(logit_kernel<kTerms, true>, Shape<kTerms>::kSmem);
    allow_smem(product_kernel<kTerms>, Shape<kTerms>::kSmem);
    const int64_t plane = static_cast<int64_t>(a.k) * p.pitch;
    for (int64_t first = 0; first < a.k; first += p.piece) {
        const int64_t count = std::min<int64_t>(p.piece, a.k - first);
        const CUtensorMap map_g = terms_map(base + p.g, count, a.rows, p.g_pitch, a.rows * p.g_pitch, kTerms);
        const CUtensorMap map_g_store = terms_map(base + p.g, count, a.rows, p.g_pitch, a.rows * p.g_pitch, kTerms, true);
        const CUtensorMap map_w = terms_map(ws + first * p.pitch, a.width, count, p.pitch, plane, kTerms);
        LogitArgs l{};
        l.rows = a.rows, l.first = static_cast<int32_t>(first), l.count = static_cast<int32_t>(count), l.k = a.k;
        l.k_blocks = static_cast<int32_t>(ceil_div(a.width, kBlockK));
        l.m_tiles = static_cast<int32_t>(p.m_tiles);
        l.tile_n = tile_columns(p.m_tiles, count, kTerms, sms);
        l.n_tiles = l.splits = static_cast<int32_t>(ceil_div(count, l.tile_n));
        l.span = 1;
        l.bias = a.bias, l.labels = a.labels, l.scale = a.scale;
        l.lse = a.lse_in, l.dloss = a.dloss;
        l.column_sums = a.dbias ? reinterpret_cast<float *>(base + p.sums) : nullptr;
        int64_t grid = std::min<int64_t>(p.m_tiles * l.splits, sms);
        cuda_check(launch_pdl(logit_kernel<kTerms, true>, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                              Shape<kTerms>::kSmem, stream, map_x, map_w, map_g_store, l));
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
            o.m_tiles = static_cast<int32_t>(ceil_div(size[i], kTileM));
            o.k_blocks = static_cast<int32_t>(depth[i]);
            // the last piece is shorter: its splits are too, and all of them exist
            o.splits = static_cast<int32_t>(std::min<int64_t>(p.splits[i], depth[i]));
            o.split_blocks = static_cast<int32_t>(ceil_div(depth[i], o.splits));
            o.splits = static_cast<int32_t>(ceil_div(depth[i], o.split_blocks));
            o.items = static_cast<int64_t>(o.m_tiles) * q.n_tiles * o.splits;
            o.out = out[i];
            o.part = p.direct[i] ? nullptr : reinterpret_cast<float *>(base + p.part[i]);
            o.add = i == 0 && first > 0;
            o.part_stride = size[i] * a.width;
        }
        q.first_product = q.one[0].split_blocks >= q.one[1].split_blocks ? 0 : 1;
        grid = std::min<int64_t>(q.one[0].items + q.one[1].items, sms);
        cuda_check(launch_pdl(product_kernel<kTerms>, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                              Shape<kTerms>::kSmem, stream, map_g, map_x, map_w, q));
        auto join = [&](int i) {
            const auto &o = q.one[i];
            const int64_t n = size[i] * a.width;
            const int64_t blocks = std::min<int64_t>(ceil_div(n, 256), 16 * sms);
            const int splits = i == 0 ? p.splits[0] : o.splits;
            cuda_check(launch_pdl(join_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                                  static_cast<const float *>(o.part), o.part_stride, splits, n, a.scale,
                                  static_cast<T *>(o.out)));
        };
        if (!p.direct[1]) join(1);
        if (!p.direct[0] && first + count == a.k) join(0);
        if (a.dbias)
            cuda_check(launch_pdl(dbias_kernel, dim3(static_cast<unsigned>(ceil_div(count, 32))), dim3(256), 0,
                                  stream, static_cast<const float *>(l.column_sums), 4 * p.m_tiles,
                                  static_cast<int32_t>(count), a.dbias + first));
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
