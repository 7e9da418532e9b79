// Layer norm of frames and its gradients.
//
//   mean = sum x / w, rstd = (sum (x - mean)^2 / w + eps)^(-1/2)
//   n = (x - mean) rstd, y = n gamma + beta
//   g = dy gamma, dx = rstd (g - mean(g) - n mean(g n))
//   dgamma = sum_rows dy n, dbeta = sum_rows dy
//
// Each matrix crosses HBM once, which bounds f32 and, with the issue of
// instructions, 16-bit types.  A row stays in registers, so the variance is
// the centred sum of squares, not a difference of moments.
// All sums are f32.
#include "norm_rows.cuh"

namespace vfr {
namespace {

// The lane's columns of a parameter vector, `missing` where there is none.
template <class S>
__device__ __forceinline__ void load_columns(const float *p, int width, int warp, int lane, float missing, float *v) {
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
        const int col = S::column(c, warp, lane);
        if (p && col < width) {
            load_params<S::kVec>(p + col, v + c * S::kVec);
        } else {
#pragma unroll
            for (int i = 0; i < S::kVec; ++i) v[c * S::kVec + i] = missing;
        }
    }
}

// A group of kWpr warps walks its rows, each held in registers.  60,000 x 768:
// f32 59 us (HBM 66% busy), bf16 35 us (46%, instructions issued in 58% of
// the cycles); with a checkpoint 68 and 48 us.
template <class S>
__global__ void __launch_bounds__(kRowThreads, 2) norm_forward_kernel(NormForward a, RingPlan plan) {
    using T = typename S::T;
    constexpr int kVec = S::kVec;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[4 * kRowWarps];
    __shared__ RingBars bars;
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int width = a.width;
    const float inv_width = 1.0f / static_cast<float>(width);
    const int64_t blocks = (a.rows + S::kGroups - 1) / S::kGroups;
    RowRing<S::kGroups> ring{plan, &bars, smem, {static_cast<const uint8_t *>(a.x), nullptr}, a.rows};
    typename S::Raw q[S::kChunks];
    float gamma[S::kLane], beta[S::kLane];
    if constexpr (S::kRing) ring.start();
    load_columns<S>(a.gamma, width, warp, lane, 1.0f, gamma);
    load_columns<S>(a.beta, width, warp, lane, 0.0f, beta);
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t row = block * S::kGroups + group;
        const int limit = row < a.rows ? width : 0;
        if constexpr (S::kRing) {
            ring.open();
            S::load(reinterpret_cast<const T *>(ring.row(0, group)), limit, warp, lane, q);
            ring.close(block);
        } else {
            S::load(static_cast<const T *>(a.x) + row * width, limit, warp, lane, q);
        }
        float v[S::kLane];
        float part[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) part[i] = ring.bad ? NAN : 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            q[c].values(v + c * kVec);
            add_to<kVec>(part, v + c * kVec);
        }
        const float mean = row_sum<S::kWpr>(sum_of<kVec>(part), slots, turn, group, warp) * inv_width;
#pragma unroll
        for (int i = 0; i < kVec; ++i) part[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            add_scalar<kVec>(v + c * kVec, -mean);
            if (S::column(c, warp, lane) < limit) fma_to<kVec>(part, v + c * kVec, v + c * kVec);
        }
        const float rstd =
            1.0f / sqrtf(row_sum<S::kWpr>(sum_of<kVec>(part), slots, turn, group, warp) * inv_width + a.eps);
        if (limit && warp == 0 && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        T *y = static_cast<T *>(a.y) + row * width;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float o[kVec];
#pragma unroll
                for (int i = 0; i < kVec; ++i) o[i] = beta[c * kVec + i];
                mul_scalar<kVec>(v + c * kVec, rstd);
                fma_to<kVec>(o, v + c * kVec, gamma + c * kVec);
                store_vec<T, kVec>(y + col, o);
            }
        }
        if (a.packed && limit)
            pack_row<S>(
                [&](int c, float *u) {
                    q[c].values(u);
                    if (ring.bad)
#pragma unroll
                        for (int i = 0; i < kVec; ++i) u[i] = NAN;
                },
                width, warp, lane, a.packed + row * width, a.exponents + row * checkpoint_blocks(width));
    }
}

// x of a row in a lane's registers, as it is or its checkpoint.
template <class S, bool kPacked>
struct Held {
    typename S::Raw q[S::kChunks];
    __device__ __forceinline__ void load(const NormBackward &a, int64_t row, int limit, int warp, int lane) {
        S::load(static_cast<const typename S::T *>(a.x) + row * a.width, limit, warp, lane, q);
    }
    __device__ __forceinline__ void values(int c, float *v) const { q[c].values(v); }
};
template <class S>
struct Held<S, true> {
    PackedBytes<S::kVec> q[S::kChunks];
    uint8_t e[S::kChunks];
    __device__ __forceinline__ void load(const NormBackward &a, int64_t row, int limit, int warp, int lane) {
        const uint8_t *bytes = a.packed + row * a.width, *exps = a.exponents + row * checkpoint_blocks(a.width);
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                q[c] = *reinterpret_cast<const PackedBytes<S::kVec> *>(bytes + col);
                e[c] = exps[col / kCheckpointBlock];
            }
        }
    }
    __device__ __forceinline__ void values(int c, float *v) const {
        unpack_bytes<S::kVec>(q[c], checkpoint_scale(e[c]), v);
    }
};

// A group of kWpr warps walks its rows; the parameter sums stay in registers
// until the last one, then join in shared memory, one partial a CTA.  With a
// ring x and dy are read from shared memory twice, so registers hold only
// the sums and gamma.  60,000 x 768: f32 83 us (HBM 75% busy), bf16 54 us
// (56%, issue 61%); from a checkpoint 71 us (64%) and 64 us (37%, issue 62%).
template <class S, bool kPacked>
__global__ void __launch_bounds__(kRowThreads, 2) norm_backward_kernel(NormBackward a, RingPlan plan) {
    using T = typename S::T;
    constexpr int kVec = S::kVec;
    extern __shared__ __align__(128) uint8_t smem[];  // the ring; at the end the sums [group][2][width]
    __shared__ float slots[4 * kRowWarps];
    __shared__ RingBars bars;
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int width = a.width;
    const float inv_width = 1.0f / static_cast<float>(width);
    const int64_t blocks = (a.rows + S::kGroups - 1) / S::kGroups;
    const uint8_t *x_base = kPacked ? a.packed : static_cast<const uint8_t *>(a.x);
    RowRing<S::kGroups> ring{plan, &bars, smem, {static_cast<const uint8_t *>(a.dy), x_base}, a.rows};
    float dg[S::kLane], db[S::kLane], gamma[S::kLane];
#pragma unroll
    for (int i = 0; i < S::kLane; ++i) dg[i] = db[i] = 0.0f;
    Held<S, kPacked> x;  // without a ring
    typename S::Raw d[S::kChunks];
    float mean = 0.0f, rstd = 0.0f, mean_next = 0.0f, rstd_next = 0.0f;
    auto moments = [&](int64_t block, float &m, float &r) {
        const int64_t row = block * S::kGroups + group;
        m = row < a.rows ? a.mean[row] : 0.0f;
        r = row < a.rows ? a.rstd[row] : 0.0f;
    };
    if constexpr (S::kRing) ring.start();
    load_columns<S>(a.gamma, width, warp, lane, 1.0f, gamma);
    moments(blockIdx.x, mean_next, rstd_next);
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t row = block * S::kGroups + group;
        const int limit = row < a.rows ? width : 0;
        mean = mean_next, rstd = rstd_next;
        moments(block + gridDim.x, mean_next, rstd_next);
        const uint8_t *exps = nullptr;
        if constexpr (S::kRing) {
            if constexpr (kPacked) exps = a.exponents + row * checkpoint_blocks(width);
            ring.open();
            if (ring.bad) mean = NAN;
        } else {
            S::load(static_cast<const T *>(a.dy) + row * width, limit, warp, lane, d);
            x.load(a, row, limit, warp, lane);
        }
        // chunk c: x less the mean, and dy
        auto pair = [&](int c, int col, float *n, float *g) {
            if constexpr (S::kRing) {
                load_vec<T, kVec>(reinterpret_cast<const T *>(ring.row(0, group)) + col, g);
                if constexpr (kPacked)
                    unpack_bytes<kVec>(*reinterpret_cast<const PackedBytes<kVec> *>(ring.row(1, group) + col),
                                       checkpoint_scale(__ldg(exps + col / kCheckpointBlock)), n);
                else
                    load_vec<T, kVec>(reinterpret_cast<const T *>(ring.row(1, group)) + col, n);
            } else {
                d[c].values(g);
                x.values(c, n);
            }
            add_scalar<kVec>(n, -mean);
        };
        float pg[kVec], pgn[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) pg[i] = pgn[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float n[kVec], g[kVec];
                pair(c, col, n, g);
                mul_scalar<kVec>(n, rstd);
                fma_to<kVec>(dg + c * kVec, g, n);
                add_to<kVec>(db + c * kVec, g);
                mul_by<kVec>(g, gamma + c * kVec);
                add_to<kVec>(pg, g);
                fma_to<kVec>(pgn, g, n);
            }
        }
        float sg = sum_of<kVec>(pg), sgn = sum_of<kVec>(pgn);
        row_sums<S::kWpr>(sg, sgn, slots, turn, group, warp);
        // dx = rstd (g - mean(g) - n mean(g n)), n = (x - mean) rstd
        const float shift = -sg * inv_width * rstd, slope = -sgn * inv_width * rstd * rstd;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float n[kVec], g[kVec];
                pair(c, col, n, g);
                mul_by<kVec>(g, gamma + c * kVec);
                fma_scalars<kVec>(g, rstd, shift);
                fma_scalar<kVec>(g, n, slope);
                store_vec<T, kVec>(static_cast<T *>(a.dx) + row * width + col, g);
            }
        }
        if constexpr (S::kRing) ring.close(block);
    }
    launch_dependents();
    if (a.partials == nullptr) return;
    // each group's sums in shared memory, then joined in group order
    float *sums = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
        const int col = S::column(c, warp, lane);
        if (col < width) {
            float *at = sums + static_cast<int64_t>(group) * 2 * width + col;
            store_vec<float, kVec == 1 ? 1 : 4>(at, dg + c * kVec);
            store_vec<float, kVec == 1 ? 1 : 4>(at + width, db + c * kVec);
            if constexpr (kVec == 8) {
                store_vec<float, 4>(at + 4, dg + c * kVec + 4);
                store_vec<float, 4>(at + width + 4, db + c * kVec + 4);
            }
        }
    }
    __syncthreads();
    float *out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * width;
    for (int i = threadIdx.x; i < 2 * width; i += kRowThreads) {
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) s += sums[g * 2 * width + i];
        out[i] = s;
    }
}

// dgamma / dbeta from the CTAs' sums, in order (the same result every time):
// 32 columns a CTA, 32 warps over the partials.  Bound by latency: 7 us for
// 1.8 MB at a width of 768.
__global__ void __launch_bounds__(1024) norm_params_kernel(const float *partials, int parts, int width, float *dgamma,
                                                           float *dbeta) {
    __shared__ float slots[32][33];
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;  // 0 .. 2 width
    float s = 0.0f;
    if (col < 2 * width) {
#pragma unroll 4
        for (int p = warp; p < parts; p += 32) s += partials[static_cast<int64_t>(p) * 2 * width + col];
    }
    slots[warp][lane] = s;
    __syncthreads();
    s = slots[lane][warp];  // column `warp` of the CTA, part `lane`
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    const int c = blockIdx.x * 32 + warp;
    if (lane != 0 || c >= 2 * width) return;
    if (c < width) {
        if (dgamma) dgamma[c] = s;
    } else if (dbeta) {
        dbeta[c - width] = s;
    }
}

// CTAs a SM: with a ring two, whose rings fill its shared memory.
constexpr int kResident = 2, kLaneResident = 4;

}  // namespace

void launch_layer_norm(const NormForward &a, int sms, cudaStream_t stream) {
    if (a.rows == 0) return;
    const size_t row = a.width * dtype_bytes(a.dtype);
    const bool wide = whole_units(row, {a.x, a.y, a.gamma, a.beta}) && packs_wide(a.packed, a.dtype);
    const int groups = row_groups(a.width, wide);
    const RingPlan plan = plan_ring(groups, row, 0, kResident);
    const unsigned grid = row_grid(a.rows, groups, sms, wide ? kResident : kLaneResident);
    with_rows(a.dtype, wide, a.width, [&](auto s) {
        using S = decltype(s);
        launch_rows(norm_forward_kernel<S>, grid, S::kRing ? ring_bytes(plan, groups) : 0, stream, a, plan);
    });
}

// Partials follow the larger grid of the two paths.
size_t norm_backward_workspace(int64_t rows, int width, int sms) {
    const unsigned grid = row_grid(rows, row_groups(width, false), sms, kResident);
    return static_cast<size_t>(grid) * 2 * width * sizeof(float);
}

void launch_layer_norm_backward(const NormBackward &args, int sms, cudaStream_t stream) {
    NormBackward a = args;
    if (!a.dgamma && !a.dbeta) a.partials = nullptr;
    unsigned grid = 0;
    if (a.rows > 0) {
        const size_t row = a.width * dtype_bytes(a.dtype), x_row = a.x ? row : a.width;
        const bool wide = whole_units(row, {a.dy, a.dx, a.gamma}) && whole_units(x_row, {a.x, a.packed});
        const int groups = row_groups(a.width, wide);
        const RingPlan plan = plan_ring(groups, row, x_row, kResident);
        const size_t sums = a.partials ? groups * 2 * a.width * sizeof(float) : 0;
        grid = row_grid(a.rows, groups, sms, kResident);
        with_rows(a.dtype, wide, a.width, [&](auto s) {
            using S = decltype(s);
            launch_rows(a.x ? norm_backward_kernel<S, false> : norm_backward_kernel<S, true>, grid,
                        std::max(sums, S::kRing ? ring_bytes(plan, groups) : 0), stream, a, plan);
        });
    }
    if (a.dgamma || a.dbeta)
        cuda_check(launch_pdl(norm_params_kernel, dim3((2 * a.width + 31) / 32), dim3(1024), 0, stream,
                              static_cast<const float *>(a.partials), static_cast<int>(grid), a.width, a.dgamma,
                              a.dbeta));
}

}  // namespace vfr
