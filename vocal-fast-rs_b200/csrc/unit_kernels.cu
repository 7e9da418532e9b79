// Softmax cross entropy of frames over a codebook of units, and its gradients.
//
//   z[r][v] = scale x_r . w_v + bias_v, lse_r = log sum_v exp z[r][v]
//   loss_r = lse_r - z[r][label_r]  (0 where the label is outside [0, k))
//   G[r][v] = dloss_r (exp(z[r][v] - lse_r) - [v == label_r]), 0 in frames
//   without a label and in units left out (bias -inf)
//   dx = scale G w, dw = scale G^T x, dbias = column sums of G
//
// The logits are never kept: the forward pass folds each tile into a running
// (maximum, sum) per row, the backward pass forms G for a piece of the units
// at a time in the workspace.
#include <algorithm>
#include <cmath>

#include "row_io.cuh"
#include "units.h"

namespace vfr {
namespace {

constexpr int kTile = 64, kStep = 16, kThreads = 256;

// acc[i][j] = sum_k a(row0 + 4 ty + i, k) b(col0 + 4 tx + j, k)
template <class A, class B>
__device__ __forceinline__ void tile_product(A a, B b, int64_t depth, float (&acc)[4][4]) {
    __shared__ float sa[kStep][kTile + 4], sb[kStep][kTile + 4];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    for (int64_t k0 = 0; k0 < depth; k0 += kStep) {
        for (int e = threadIdx.x; e < kTile * kStep; e += kThreads) {
            sa[e % kStep][e / kStep] = a(e / kStep, k0 + e % kStep);
            sb[e % kStep][e / kStep] = b(e / kStep, k0 + e % kStep);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][4 * ty + i] * sb[k][4 * tx + j];
        __syncthreads();
    }
}

template <typename T>
struct Rows {
    const T *p;
    int64_t first, count;
    int width;
    __device__ float operator()(int r, int64_t k) const {
        return first + r < count && k < width ? to_f32(p[(first + r) * width + k]) : 0.0f;
    }
};

__device__ __forceinline__ float logit(const UnitLoss &a, float dot, int64_t v) {
    const float b = a.bias ? a.bias[v] : 0.0f;
    return b == -INFINITY ? b : fmaf(a.scale, dot, b);  // a masked unit's row may hold anything
}

template <typename T>
__global__ void __launch_bounds__(kThreads) loss_kernel(UnitLoss a) {
    __shared__ float z[kTile][kTile + 1], target[kTile];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float top = -INFINITY, sum = 0.0f;  // of row threadIdx.x
    if (threadIdx.x < kTile) target[threadIdx.x] = 0.0f;
    for (int64_t v0 = 0; v0 < a.k; v0 += kTile) {
        float acc[4][4];
        tile_product(Rows<T>{static_cast<const T *>(a.x), row0, a.rows, a.width},
                     Rows<T>{static_cast<const T *>(a.units), v0, a.k, a.width}, a.width, acc);
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int64_t r = row0 + 4 * ty + i, v = v0 + 4 * tx + j;
                const float value = v < a.k ? logit(a, acc[i][j], v) : -INFINITY;
                z[4 * ty + i][4 * tx + j] = value;
                if (r < a.rows && v < a.k && a.labels[r] == v) target[4 * ty + i] = value;
            }
        __syncthreads();
        if (threadIdx.x < kTile) {
            float m = top;
            for (int j = 0; j < kTile; ++j) m = fmaxf(m, z[threadIdx.x][j]);
            if (m > -INFINITY) {
                sum *= expf(top - m);
                for (int j = 0; j < kTile; ++j) sum += expf(z[threadIdx.x][j] - m);
                top = m;
            }
        }
        __syncthreads();
    }
    const int64_t r = row0 + threadIdx.x;
    if (threadIdx.x < kTile && r < a.rows) {
        const float lse = top == -INFINITY ? top : top + logf(sum);
        const int32_t t = a.labels[r];
        a.lse[r] = lse;
        const float zt = target[threadIdx.x];
        a.loss[r] = t < 0 || t >= a.k ? 0.0f : zt == -INFINITY ? INFINITY : lse - zt;
    }
}

// G of the units [first, first + count), row-major with `count` columns.
template <typename T>
__global__ void __launch_bounds__(kThreads) gradient_kernel(UnitLoss a, int64_t first, int64_t count, float *g) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile, v0 = first + static_cast<int64_t>(blockIdx.y) * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4];
    tile_product(Rows<T>{static_cast<const T *>(a.x), row0, a.rows, a.width},
                 Rows<T>{static_cast<const T *>(a.units), v0, a.k, a.width}, a.width, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = row0 + 4 * ty + i, v = v0 + 4 * tx + j;
            if (r >= a.rows || v >= first + count) continue;
            const int32_t t = a.labels[r];
            float value = 0.0f;
            if (t >= 0 && t < a.k && !(a.bias && a.bias[v] == -INFINITY))
                value = (expf(logit(a, acc[i][j], v) - a.lse_in[r]) - (t == v ? 1.0f : 0.0f)) * a.dloss[r];
            g[r * count + (v - first)] = value;
        }
}

__global__ void column_sum_kernel(const float *g, int64_t rows, int64_t count, float *out) {
    const int64_t v = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (v >= count) return;
    float s = 0.0f;
    for (int64_t r = 0; r < rows; ++r) s += g[r * count + v];
    out[v] = s;
}

// dx of the piece, added to `sum` (f32) unless it is the first; the last piece writes dx.
template <typename T>
__global__ void __launch_bounds__(kThreads) dx_kernel(UnitLoss a, int64_t first, int64_t count, const float *g,
                                                      float *sum, bool start, bool last) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile, c0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const T *w = static_cast<const T *>(a.units);
    float acc[4][4];
    tile_product(
        [&](int r, int64_t k) { return row0 + r < a.rows && k < count ? g[(row0 + r) * count + k] : 0.0f; },
        [&](int c, int64_t k) {
            if (c0 + c >= a.width || k >= count || (a.bias && a.bias[first + k] == -INFINITY)) return 0.0f;
            return to_f32(w[(first + k) * a.width + c0 + c]);
        },
        count, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = row0 + 4 * ty + i, c = c0 + 4 * tx + j;
            if (r >= a.rows || c >= a.width) continue;
            const float s = (start ? 0.0f : sum[r * a.width + c]) + acc[i][j];
            if (last) static_cast<T *>(a.dx)[r * a.width + c] = from_f32<T>(s * a.scale);
            else sum[r * a.width + c] = s;
        }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dw_kernel(UnitLoss a, int64_t first, int64_t count, const float *g) {
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * kTile, c0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const T *x = static_cast<const T *>(a.x);
    float acc[4][4];
    tile_product(
        [&](int v, int64_t r) { return v0 + v < count && r < a.rows ? g[r * count + v0 + v] : 0.0f; },
        [&](int c, int64_t r) {
            if (c0 + c >= a.width || r >= a.rows || a.labels[r] < 0 || a.labels[r] >= a.k) return 0.0f;
            return to_f32(x[r * a.width + c0 + c]);
        },
        a.rows, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t v = v0 + 4 * ty + i, c = c0 + 4 * tx + j;
            if (v < count && c < a.width)
                static_cast<T *>(a.dunits)[(first + v) * a.width + c] = from_f32<T>(acc[i][j] * a.scale);
        }
}

unsigned tiles(int64_t n) { return static_cast<unsigned>((n + kTile - 1) / kTile); }
// Units a piece of G covers: 256 MB of G at most, but at least 256 units.
int64_t piece_units(int64_t rows, int k) {
    const int64_t fit = (int64_t(256) << 20) / (std::max<int64_t>(rows, 1) * 4) / 256 * 256;
    return std::min<int64_t>(k, std::max<int64_t>(256, fit));
}

template <typename T>
void backward(const UnitLoss &a, cudaStream_t stream) {
    const int64_t piece = piece_units(a.rows, a.k);
    float *g = static_cast<float *>(a.workspace);
    float *sum = g + a.rows * piece;
    for (int64_t first = 0; first < a.k; first += piece) {
        const int64_t count = std::min<int64_t>(piece, a.k - first);
        if (a.rows > 0) {
            gradient_kernel<T><<<dim3(tiles(a.rows), tiles(count)), kThreads, 0, stream>>>(a, first, count, g);
            dx_kernel<T><<<dim3(tiles(a.rows), tiles(a.width)), kThreads, 0, stream>>>(
                a, first, count, g, sum, first == 0, first + count == a.k);
        }
        dw_kernel<T><<<dim3(tiles(count), tiles(a.width)), kThreads, 0, stream>>>(a, first, count, g);
        if (a.dbias)
            column_sum_kernel<<<static_cast<unsigned>((count + 255) / 256), 256, 0, stream>>>(g, a.rows, count,
                                                                                              a.dbias + first);
    }
}

}  // namespace

size_t unit_loss_workspace(int64_t rows, int k, int width, int, bool backward, int) {
    if (!backward) return 0;
    return static_cast<size_t>(rows) * (piece_units(rows, k) + width) * sizeof(float);
}

void launch_unit_loss(const UnitLoss &a, int, cudaStream_t stream) {
    if (a.rows == 0) return;
    if (a.dtype == kF32) loss_kernel<float><<<tiles(a.rows), kThreads, 0, stream>>>(a);
    else loss_kernel<__nv_bfloat16><<<tiles(a.rows), kThreads, 0, stream>>>(a);
}

void launch_unit_loss_backward(const UnitLoss &a, int, cudaStream_t stream) {
    if (a.dtype == kF32) backward<float>(a, stream);
    else backward<__nv_bfloat16>(a, stream);
}

}  // namespace vfr
