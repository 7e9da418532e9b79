// Layer norm of frames, its gradients, and 8-bit activation checkpoints.
//
//   mean = sum x / w, rstd = (sum (x - mean)^2 / w + eps)^(-1/2)
//   n = (x - mean) rstd, y = n gamma + beta
//   g = dy gamma, dx = rstd (g - mean(g) - n mean(g n))
//   dgamma = sum_rows dy n, dbeta = sum_rows dy
//
// Every kernel is bound by HBM: each matrix crosses it once.  A row stays in
// the registers of one warp (width <= 1,024) or of four, 32 values a lane, so
// the variance is the centred sum of squares, not a difference of moments.
// All sums are f32.
#include <algorithm>

#include "row_io.cuh"
#include "units.h"

namespace vfr {
namespace {

constexpr int kLane = 32;      // values of a row a lane holds at most
constexpr int kThreads = 256;  // 8 rows of one warp or 2 rows of four warps
constexpr int kWarps = kThreads / 32;

// Column of a lane's value i of the chunk c (kVec values): chunks of a warp
// are contiguous, and 128 columns of a checkpoint block belong to one warp.
template <int kVec, int kWpr>
__device__ __forceinline__ int column(int c, int warp, int lane) {
    if constexpr (kVec == 1) return (((c >> 2) * kWpr + warp) << 7) + ((c & 3) << 5) + lane;
    return ((c * kWpr + warp) * 32 + lane) * kVec;
}

// Sum over the warps of a row; `slots` holds kWarps floats and is free again
// when every thread has passed the next call's first barrier.
template <int kWpr>
__device__ __forceinline__ float row_sum(float v, float *slots, int group, int warp) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if constexpr (kWpr > 1) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) slots[group * kWpr + warp] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < kWpr; ++i) v += slots[group * kWpr + i];
    }
    return v;
}

// The 8-bit checkpoint of the values a warp holds: block maxima by lane
// exchange, then e4m3 bytes and one exponent byte a block.
template <int kVec, int kWpr>
__device__ __forceinline__ void pack_row(const float *v, int width, int warp, int lane, uint8_t *packed,
                                         uint8_t *exponents) {
    constexpr int kChunks = kLane / kVec;
    constexpr int kStep = kVec == 1 ? 4 : 1;   // chunks that cover one run of blocks
    constexpr int kSpan = kVec == 8 ? 16 : 32;  // lanes that share a block
#pragma unroll
    for (int c = 0; c < kChunks; c += kStep) {
        const int col = column<kVec, kWpr>(c, warp, lane);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kStep * kVec; ++i) top = max(top, checkpoint_magnitude(v[c * kVec + i]));
        if constexpr (kSpan == 32) {
            top = __reduce_max_sync(0xFFFFFFFFu, top);
        } else {
#pragma unroll
            for (int o = kSpan / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        }
        const uint32_t e = checkpoint_exponent(top);
        const float inverse = checkpoint_inverse(e);
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            const int at = kVec == 1 ? col + 32 * k : col;
            if (at < width) {
                store_packed<kVec>(packed + at, v + (c + k) * kVec, inverse);
                if (at % kCheckpointBlock == 0) exponents[at / kCheckpointBlock] = static_cast<uint8_t>(e);
            }
        }
    }
}

template <typename T, int kVec, int kWpr>
__device__ __forceinline__ void load_row(const T *row, int width, int warp, int lane, float *v) {
#pragma unroll
    for (int c = 0; c < kLane / kVec; ++c) {
        const int col = column<kVec, kWpr>(c, warp, lane);
        if (col < width) {
            load_vec<T, kVec>(row + col, v + c * kVec);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[c * kVec + i] = 0.0f;
        }
    }
}

template <typename T, int kVec, int kWpr>
__global__ void __launch_bounds__(kThreads) norm_forward_kernel(NormForward a) {
    __shared__ float slots[kWarps];
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % kWpr, group = (threadIdx.x >> 5) / kWpr;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / kWpr) + group;
    const bool live = row < a.rows;
    const int width = a.width;
    const int64_t at = row * width;
    float v[kLane];
    load_row<T, kVec, kWpr>(static_cast<const T *>(a.x) + at, live ? width : 0, warp, lane, v);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kLane; ++i) sum += v[i];
    const float mean = row_sum<kWpr>(sum, slots, group, warp) / static_cast<float>(width);
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < kLane / kVec; ++c) {
        if (column<kVec, kWpr>(c, warp, lane) < width) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float d = v[c * kVec + i] - mean;
                sq += d * d;
            }
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<kWpr>(sq, slots, group, warp) / static_cast<float>(width) + a.eps);
    if (!live) return;
    if (warp == 0 && lane == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    T *y = static_cast<T *>(a.y) + at;
#pragma unroll
    for (int c = 0; c < kLane / kVec; ++c) {
        const int col = column<kVec, kWpr>(c, warp, lane);
        if (col < width) {
            float o[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                o[i] = (v[c * kVec + i] - mean) * rstd;
                if (a.gamma) o[i] *= a.gamma[col + i];
                if (a.beta) o[i] += a.beta[col + i];
            }
            store_vec<T, kVec>(y + col, o);
        }
    }
    if (a.packed)
        pack_row<kVec, kWpr>(v, width, warp, lane, a.packed + at, a.exponents + row * checkpoint_blocks(width));
}

// One group of kWpr warps walks rows group, group + groups, ...; the
// parameter sums stay in registers until its last row.
template <typename T, int kVec, int kWpr, bool kPacked>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(NormBackward a) {
    __shared__ float slots[kWarps];
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % kWpr, group = (threadIdx.x >> 5) / kWpr;
    constexpr int kGroups = kWarps / kWpr;
    const int width = a.width, blocks = checkpoint_blocks(width);
    const float inv_width = 1.0f / static_cast<float>(width);
    float dg[kLane], db[kLane];
#pragma unroll
    for (int i = 0; i < kLane; ++i) dg[i] = db[i] = 0.0f;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows;
         base += static_cast<int64_t>(gridDim.x) * kGroups) {
        const int64_t row = base + group;
        const bool live = row < a.rows;
        const int limit = live ? width : 0;
        const int64_t at = row * width;
        float n[kLane], d[kLane];
        load_row<T, kVec, kWpr>(static_cast<const T *>(a.dy) + at, limit, warp, lane, d);
        if constexpr (kPacked) {
#pragma unroll
            for (int c = 0; c < kLane / kVec; ++c) {
                const int col = column<kVec, kWpr>(c, warp, lane);
                if (col < limit) {
                    load_packed<kVec>(a.packed + at + col,
                                      checkpoint_scale(a.exponents[row * blocks + col / kCheckpointBlock]),
                                      n + c * kVec);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) n[c * kVec + i] = 0.0f;
                }
            }
        } else {
            load_row<T, kVec, kWpr>(static_cast<const T *>(a.x) + at, limit, warp, lane, n);
        }
        const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
        float sg = 0.0f, sgn = 0.0f;
#pragma unroll
        for (int c = 0; c < kLane / kVec; ++c) {
            const int col = column<kVec, kWpr>(c, warp, lane);
            if (col < limit) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int j = c * kVec + i;
                    n[j] = (n[j] - mean) * rstd;
                    dg[j] += d[j] * n[j];
                    db[j] += d[j];
                    if (a.gamma) d[j] *= a.gamma[col + i];
                    sg += d[j];
                    sgn += d[j] * n[j];
                }
            }
        }
        sg = row_sum<kWpr>(sg, slots, group, warp) * inv_width;
        sgn = row_sum<kWpr>(sgn, slots, group, warp) * inv_width;
#pragma unroll
        for (int c = 0; c < kLane / kVec; ++c) {
            const int col = column<kVec, kWpr>(c, warp, lane);
            if (col < limit) {
                float o[kVec];
#pragma unroll
                for (int i = 0; i < kVec; ++i) o[i] = (d[c * kVec + i] - sg - n[c * kVec + i] * sgn) * rstd;
                store_vec<T, kVec>(static_cast<T *>(a.dx) + at + col, o);
            }
        }
    }
    if (a.partials == nullptr) return;
    float *out = a.partials + (static_cast<int64_t>(blockIdx.x) * kGroups + group) * 2 * width;
#pragma unroll
    for (int c = 0; c < kLane / kVec; ++c) {
        const int col = column<kVec, kWpr>(c, warp, lane);
        if (col < width) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                out[col + i] = dg[c * kVec + i];
                out[width + col + i] = db[c * kVec + i];
            }
        }
    }
}

// dgamma / dbeta from the groups' sums, in group order (the same result every
// time): 32 columns a CTA, 8 warps over the groups.
__global__ void __launch_bounds__(256) norm_params_kernel(const float *partials, int groups, int width, float *dgamma,
                                                          float *dbeta) {
    __shared__ float sums[8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;  // 0 .. 2 width
    float s = 0.0f;
    if (col < 2 * width)
        for (int g = w; g < groups; g += 8) s += partials[static_cast<int64_t>(g) * 2 * width + col];
    sums[w][lane] = s;
    __syncthreads();
    if (w != 0 || col >= 2 * width) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sums[i][lane];
    if (col < width) {
        if (dgamma) dgamma[col] = s;
    } else if (dbeta) {
        dbeta[col - width] = s;
    }
}

template <typename T, int kVec, int kWpr>
__global__ void __launch_bounds__(kThreads) pack_kernel(const T *x, int64_t rows, int width, uint8_t *packed,
                                                        uint8_t *exponents) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % kWpr, group = (threadIdx.x >> 5) / kWpr;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / kWpr) + group;
    if (row >= rows) return;
    float v[kLane];
    load_row<T, kVec, kWpr>(x + row * width, width, warp, lane, v);
    pack_row<kVec, kWpr>(v, width, warp, lane, packed + row * width, exponents + row * checkpoint_blocks(width));
}

template <typename T, int kVec, int kWpr>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const uint8_t *packed, const uint8_t *exponents,
                                                          int64_t rows, int width, T *x) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % kWpr, group = (threadIdx.x >> 5) / kWpr;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / kWpr) + group;
    if (row >= rows) return;
    const int64_t at = row * width;
    const uint8_t *e = exponents + row * checkpoint_blocks(width);
#pragma unroll
    for (int c = 0; c < kLane / kVec; ++c) {
        const int col = column<kVec, kWpr>(c, warp, lane);
        if (col < width) {
            float v[kVec];
            load_packed<kVec>(packed + at + col, checkpoint_scale(e[col / kCheckpointBlock]), v);
            store_vec<T, kVec>(x + at + col, v);
        }
    }
}

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Calls f(T{}, integral constants kVec, kWpr) for the element type, the
// vector width (16 bytes where `wide`, else single elements) and the warps a row takes.
template <int kVec, int kWpr>
struct Shape {
    static constexpr int vec = kVec, wpr = kWpr;
};
template <typename T, class F>
void with_shape(bool wide, int width, F &&f) {
    constexpr int kWide = 16 / sizeof(T);
    if (width <= 32 * kLane) {
        if (wide) f(T{}, Shape<kWide, 1>{});
        else f(T{}, Shape<1, 1>{});
    } else {
        if (wide) f(T{}, Shape<kWide, 4>{});
        else f(T{}, Shape<1, 4>{});
    }
}
template <class F>
void dispatch(int dtype, bool wide, int width, F &&f) {
    if (dtype == kF32) with_shape<float>(wide, width, f);
    else if (dtype == kBF16) with_shape<__nv_bfloat16>(wide, width, f);
    else with_shape<__half>(wide, width, f);
}
// 16-byte accesses need rows of whole vectors and aligned bases; the packed
// bytes are then read and written 4 or 8 at a time.
bool wide_rows(int width, int dtype, std::initializer_list<const void *> values, const void *packed) {
    const int vec = 16 / static_cast<int>(dtype_bytes(dtype));
    if (width % vec) return false;
    for (const void *p : values)
        if (!aligned(p, 16)) return false;
    return aligned(packed, vec);
}
unsigned row_grid(int64_t rows, int wpr) {
    const int per = kWarps / wpr;
    return static_cast<unsigned>((rows + per - 1) / per);
}

// CTAs of the backward kernel: two per SM keep enough loads in flight, and
// bound the parameter partials.
int backward_grid(int64_t rows, int width, int sms) {
    const int per = kWarps / (width <= 32 * kLane ? 1 : 4);
    return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, 2 * sms));
}

}  // namespace

void launch_layer_norm(const NormForward &a, cudaStream_t stream) {
    if (a.rows == 0) return;
    const bool wide = wide_rows(a.width, a.dtype, {a.x, a.y}, a.packed);
    dispatch(a.dtype, wide, a.width, [&](auto t, auto s) {
        using S = decltype(s);
        norm_forward_kernel<decltype(t), S::vec, S::wpr><<<row_grid(a.rows, S::wpr), kThreads, 0, stream>>>(a);
    });
}

size_t norm_backward_workspace(int64_t rows, int width, int sms) {
    const int per = kWarps / (width <= 32 * kLane ? 1 : 4);
    return static_cast<size_t>(backward_grid(rows, width, sms)) * per * 2 * width * sizeof(float);
}

void launch_layer_norm_backward(const NormBackward &args, int sms, cudaStream_t stream) {
    NormBackward a = args;
    if (!a.dgamma && !a.dbeta) a.partials = nullptr;
    int groups = 0;
    if (a.rows > 0) {
        const bool wide = wide_rows(a.width, a.dtype, {a.dy, a.dx, a.x ? a.x : a.dy}, a.packed);
        const int grid = backward_grid(a.rows, a.width, sms);
        dispatch(a.dtype, wide, a.width, [&](auto t, auto s) {
            using S = decltype(s);
            groups = grid * (kWarps / S::wpr);
            if (a.x) norm_backward_kernel<decltype(t), S::vec, S::wpr, false><<<grid, kThreads, 0, stream>>>(a);
            else norm_backward_kernel<decltype(t), S::vec, S::wpr, true><<<grid, kThreads, 0, stream>>>(a);
        });
    }
    if (a.dgamma || a.dbeta)
        norm_params_kernel<<<(2 * a.width + 31) / 32, 256, 0, stream>>>(a.partials, groups, a.width, a.dgamma,
                                                                        a.dbeta);
}

void launch_checkpoint_pack(const void *x, int64_t rows, int width, int dtype, uint8_t *packed, uint8_t *exponents,
                            cudaStream_t stream) {
    if (rows == 0) return;
    dispatch(dtype, wide_rows(width, dtype, {x}, packed), width, [&](auto t, auto s) {
        using S = decltype(s);
        using T = decltype(t);
        pack_kernel<T, S::vec, S::wpr><<<row_grid(rows, S::wpr), kThreads, 0, stream>>>(
            static_cast<const T *>(x), rows, width, packed, exponents);
    });
}

void launch_checkpoint_unpack(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int width, int dtype,
                              void *x, cudaStream_t stream) {
    if (rows == 0) return;
    dispatch(dtype, wide_rows(width, dtype, {x}, packed), width, [&](auto t, auto s) {
        using S = decltype(s);
        using T = decltype(t);
        unpack_kernel<T, S::vec, S::wpr><<<row_grid(rows, S::wpr), kThreads, 0, stream>>>(packed, exponents, rows,
                                                                                          width, static_cast<T *>(x));
    });
}

}  // namespace vfr
