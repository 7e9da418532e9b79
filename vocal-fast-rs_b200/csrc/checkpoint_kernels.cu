// 8-bit activation checkpoints: e4m3 with one power of two per 128 elements
// of a row.  Bound by HBM: packing reads the values and writes a byte each,
// unpacking the reverse.
#include "norm_rows.cuh"
#include "pdl.cuh"
#include "vfr_common.h"

namespace vfr {
namespace {

template <class S>
__global__ void __launch_bounds__(kRowThreads, 2) pack_kernel(const typename S::T *x, int64_t rows, int width, uint8_t *packed,
                                                              uint8_t *exponents) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int64_t step = static_cast<int64_t>(gridDim.x) * S::kGroups;
    const int blocks = checkpoint_blocks(width);
    launch_dependents();
    grid_dependency_wait();
    int64_t row = static_cast<int64_t>(blockIdx.x) * S::kGroups + group;
    typename S::Raw q[S::kChunks], next[S::kChunks];
    S::load(x + row * width, row < rows ? width : 0, warp, lane, q);
    for (; row < rows; row += step) {
        S::load(x + (row + step) * width, row + step < rows ? width : 0, warp, lane, next);
        pack_row<S>(q, width, warp, lane, packed + row * width, exponents + row * blocks);
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) q[c] = next[c];
    }
}

template <class S>
__global__ void __launch_bounds__(kRowThreads, 2) unpack_kernel(const uint8_t *packed, const uint8_t *exponents,
                                                                int64_t rows, int width, typename S::T *x) {
    constexpr int kVec = S::kVec;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int64_t step = static_cast<int64_t>(gridDim.x) * S::kGroups;
    const int blocks = checkpoint_blocks(width);
    launch_dependents();
    grid_dependency_wait();
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * S::kGroups + group; row < rows; row += step) {
        const uint8_t *bytes = packed + row * width, *exps = exponents + row * blocks;
        PackedBytes<kVec> q[S::kChunks];
        uint8_t e[S::kChunks];
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < width) {
                q[c] = *reinterpret_cast<const PackedBytes<kVec> *>(bytes + col);
                e[c] = exps[col / kCheckpointBlock];
            }
        }
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < width) {
                float v[kVec];
                unpack_bytes<kVec>(q[c], checkpoint_scale(e[c]), v);
                store_vec<typename S::T, kVec>(x + row * width + col, v);
            }
        }
    }
}

constexpr int kResident = 4;

}  // namespace

void launch_checkpoint_pack(const void *x, int64_t rows, int width, int dtype, uint8_t *packed, uint8_t *exponents,
                            int sms, cudaStream_t stream) {
    if (rows == 0) return;
    const unsigned grid = row_grid(rows, row_groups(width), sms, kResident);
    with_rows(dtype, wide_rows(width, dtype, {x}, packed), width, [&](auto s) {
        using S = decltype(s);
        cuda_check(launch_pdl(pack_kernel<S>, dim3(grid), dim3(kRowThreads), 0, stream,
                              static_cast<const typename S::T *>(x), rows, width, packed, exponents));
    });
}

void launch_checkpoint_unpack(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int width, int dtype,
                              void *x, int sms, cudaStream_t stream) {
    if (rows == 0) return;
    const unsigned grid = row_grid(rows, row_groups(width), sms, kResident);
    with_rows(dtype, wide_rows(width, dtype, {x}, packed), width, [&](auto s) {
        using S = decltype(s);
        cuda_check(launch_pdl(unpack_kernel<S>, dim3(grid), dim3(kRowThreads), 0, stream, packed, exponents, rows,
                              width, static_cast<typename S::T *>(x)));
    });
}

}  // namespace vfr
