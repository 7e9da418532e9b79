// Layer norm of frames and its gradients.
//
//   mean = sum x / w, rstd = (sum (x - mean)^2 / w + eps)^(-1/2)
//   n = (x - mean) rstd, y = n gamma + beta
//   g = dy gamma, dx = rstd (g - mean(g) - n mean(g n))
//   dgamma = sum_rows dy n, dbeta = sum_rows dy
//
// Bound by HBM: each matrix crosses it once.  A row stays in registers, so
// the variance is the centred sum of squares, not a difference of moments.
// All sums are f32.
#include "norm_rows.cuh"
#include "pdl.cuh"
#include "vfr_common.h"

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

template <class S>
__global__ void __launch_bounds__(kRowThreads, 2) norm_forward_kernel(NormForward a) {
    using T = typename S::T;
    constexpr int kVec = S::kVec;
    __shared__ float slots[4 * kRowWarps];
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int width = a.width;
    const float inv_width = 1.0f / static_cast<float>(width);
    const int64_t step = static_cast<int64_t>(gridDim.x) * S::kGroups;
    typename S::Raw q[S::kChunks];
    float gamma[S::kLane], beta[S::kLane];
    launch_dependents();
    grid_dependency_wait();
    load_columns<S>(a.gamma, width, warp, lane, 1.0f, gamma);
    load_columns<S>(a.beta, width, warp, lane, 0.0f, beta);
    int64_t base = static_cast<int64_t>(blockIdx.x) * S::kGroups;
    S::load(static_cast<const T *>(a.x) + (base + group) * width, base + group < a.rows ? width : 0, warp, lane, q);
    for (; base < a.rows; base += step) {
        const int64_t row = base + group, after = row + step;
        const int limit = row < a.rows ? width : 0;
        typename S::Raw next[S::kChunks];
        S::load(static_cast<const T *>(a.x) + after * width, after < a.rows ? width : 0, warp, lane, next);
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            float v[kVec];
            q[c].values(v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) sum += v[i];
        }
        const float mean = row_sum<S::kWpr>(sum, slots, turn, group, warp) * inv_width;
        float sq = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            if (S::column(c, warp, lane) < limit) {
                float v[kVec];
                q[c].values(v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float d = v[i] - mean;
                    sq += d * d;
                }
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<S::kWpr>(sq, slots, turn, group, warp) * inv_width + a.eps);
        if (limit && warp == 0 && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        T *y = static_cast<T *>(a.y) + row * width;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float v[kVec];
                q[c].values(v);
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                    v[i] = fmaf((v[i] - mean) * rstd, gamma[c * kVec + i], beta[c * kVec + i]);
                store_vec<T, kVec>(y + col, v);
            }
        }
        if (a.packed && limit)
            pack_row<S>(q, width, warp, lane, a.packed + row * width, a.exponents + row * checkpoint_blocks(width));
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) q[c] = next[c];
    }
}

// x of a row in the backward pass: as it is, or its checkpoint.
template <class S, bool kPacked>
struct Source {
    typename S::Raw q[S::kChunks];
    __device__ __forceinline__ void load(const NormBackward &a, int64_t row, int limit, int warp, int lane) {
        S::load(static_cast<const typename S::T *>(a.x) + row * a.width, limit, warp, lane, q);
    }
    __device__ __forceinline__ void values(int c, float *v) const { q[c].values(v); }
};
template <class S>
struct Source<S, true> {
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
            } else {
#pragma unroll
                for (int i = 0; i < S::kVec; ++i) q[c].e[i] = 0;
                e[c] = 127;
            }
        }
    }
    __device__ __forceinline__ void values(int c, float *v) const {
        unpack_bytes<S::kVec>(q[c], checkpoint_scale(e[c]), v);
    }
};

// A group of kWpr warps walks rows group, group + groups, ...; the parameter
// sums stay in registers until its last row, then join in shared memory, one
// partial a CTA.
template <class S, bool kPacked>
__global__ void __launch_bounds__(kRowThreads, 2) norm_backward_kernel(NormBackward a) {
    using T = typename S::T;
    constexpr int kVec = S::kVec;
    constexpr bool kAhead = sizeof(T) == 2;
    extern __shared__ float sums[];  // [2][width]
    __shared__ float slots[4 * kRowWarps];
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int width = a.width;
    const float inv_width = 1.0f / static_cast<float>(width);
    const int64_t step = static_cast<int64_t>(gridDim.x) * S::kGroups;
    float dg[S::kLane], db[S::kLane];
#pragma unroll
    for (int i = 0; i < S::kLane; ++i) dg[i] = db[i] = 0.0f;
    Source<S, kPacked> x, x_next;
    typename S::Raw d[S::kChunks], d_next[S::kChunks];
    float mean = 0.0f, rstd = 0.0f, mean_next = 0.0f, rstd_next = 0.0f;
    auto fetch = [&](int64_t row, Source<S, kPacked> &xs, typename S::Raw(&ds)[S::kChunks], float &m, float &r) {
        const int limit = row < a.rows ? width : 0;
        S::load(static_cast<const T *>(a.dy) + row * width, limit, warp, lane, ds);
        xs.load(a, row, limit, warp, lane);
        m = limit ? a.mean[row] : 0.0f;
        r = limit ? a.rstd[row] : 0.0f;
    };
    launch_dependents();
    grid_dependency_wait();
    float gamma[S::kLane];
    load_columns<S>(a.gamma, width, warp, lane, 1.0f, gamma);
    int64_t base = static_cast<int64_t>(blockIdx.x) * S::kGroups;
    if (kAhead) fetch(base + group, x, d, mean, rstd);
    for (; base < a.rows; base += step) {
        const int64_t row = base + group;
        const int limit = row < a.rows ? width : 0;
        if (kAhead) fetch(row + step, x_next, d_next, mean_next, rstd_next);
        else fetch(row, x, d, mean, rstd);
        float sg = 0.0f, sgn = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float v[kVec], g[kVec];
                x.values(c, v);
                d[c].values(g);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    v[i] = (v[i] - mean) * rstd;
                    dg[c * kVec + i] += g[i] * v[i];
                    db[c * kVec + i] += g[i];
                    g[i] *= gamma[c * kVec + i];
                    sg += g[i];
                    sgn += g[i] * v[i];
                }
            }
        }
        row_sums<S::kWpr>(sg, sgn, slots, turn, group, warp);
        sg *= inv_width, sgn *= inv_width;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float v[kVec], g[kVec];
                x.values(c, v);
                d[c].values(g);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    v[i] = (v[i] - mean) * rstd;
                    g[i] *= gamma[c * kVec + i];
                    g[i] = (g[i] - sg - v[i] * sgn) * rstd;
                }
                store_vec<T, kVec>(static_cast<T *>(a.dx) + row * width + col, g);
            }
        }
        if (kAhead) {
            x = x_next;
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c) d[c] = d_next[c];
            mean = mean_next, rstd = rstd_next;
        }
    }
    if (a.partials == nullptr) return;
    // the CTA's groups one after the other, so the sum's order is fixed
    for (int g = 0; g < S::kGroups; ++g) {
        if (g == group) {
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c) {
                const int col = S::column(c, warp, lane);
                if (col < width) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        float *at = sums + col + i;
                        at[0] = (g ? at[0] : 0.0f) + dg[c * kVec + i];
                        at[width] = (g ? at[width] : 0.0f) + db[c * kVec + i];
                    }
                }
            }
        }
        __syncthreads();
    }
    float *out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * width;
    for (int i = threadIdx.x; i < 2 * width; i += kRowThreads) out[i] = sums[i];
}

// dgamma / dbeta from the CTAs' sums, in order (the same result every time):
// 32 columns a CTA, 32 warps over the partials.
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

constexpr int kForwardResident = 4, kBackwardResident = 2;

}  // namespace

void launch_layer_norm(const NormForward &a, int sms, cudaStream_t stream) {
    if (a.rows == 0) return;
    const bool wide = wide_rows(a.width, a.dtype, {a.x, a.y, a.gamma, a.beta}, a.packed);
    const unsigned grid = row_grid(a.rows, row_groups(a.width), sms, kForwardResident);
    with_rows(a.dtype, wide, a.width, [&](auto s) {
        cuda_check(launch_pdl(norm_forward_kernel<decltype(s)>, dim3(grid), dim3(kRowThreads), 0, stream, a));
    });
}

size_t norm_backward_workspace(int64_t rows, int width, int sms) {
    return static_cast<size_t>(row_grid(rows, row_groups(width), sms, kBackwardResident)) * 2 * width * sizeof(float);
}

void launch_layer_norm_backward(const NormBackward &args, int sms, cudaStream_t stream) {
    NormBackward a = args;
    if (!a.dgamma && !a.dbeta) a.partials = nullptr;
    const unsigned grid = row_grid(a.rows, row_groups(a.width), sms, kBackwardResident);
    if (a.rows > 0) {
        const bool wide = wide_rows(a.width, a.dtype, {a.dy, a.dx, a.x, a.gamma}, a.packed);
        const size_t smem = a.partials ? 2 * a.width * sizeof(float) : 0;
        with_rows(a.dtype, wide, a.width, [&](auto s) {
            using S = decltype(s);
            cuda_check(launch_pdl(a.x ? norm_backward_kernel<S, false> : norm_backward_kernel<S, true>, dim3(grid),
                                  dim3(kRowThreads), smem, stream, a));
        });
    }
    if (a.dgamma || a.dbeta)
        cuda_check(launch_pdl(norm_params_kernel, dim3((2 * a.width + 31) / 32), dim3(1024), 0, stream,
                              static_cast<const float *>(a.partials), static_cast<int>(grid), a.width, a.dgamma,
                              a.dbeta));
}

}  // namespace vfr
