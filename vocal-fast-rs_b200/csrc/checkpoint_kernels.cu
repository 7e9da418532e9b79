// 8-bit activation checkpoints: e4m3 with one power of two per 128 elements
// of a row.  Packing reads the values and writes a byte each, unpacking the
// reverse.  60,000 x 768: packing f32 39 us (HBM 67% busy), bf16 27 us (46%,
// instructions issued in 63% of the cycles), unpacking to f32 36 us (59%).
#include "norm_rows.cuh"

namespace vfr {
namespace {

template <class S>
__global__ void __launch_bounds__(kRowThreads, 2)
    pack_kernel(const typename S::T *x, int64_t rows, int width, uint8_t *packed, uint8_t *exponents, RingPlan plan) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RingBars bars;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int64_t blocks = (rows + S::kGroups - 1) / S::kGroups;
    RowRing<S::kGroups> ring{plan, &bars, smem, {reinterpret_cast<const uint8_t *>(x), nullptr}, rows};
    typename S::Raw q[S::kChunks];
    if constexpr (S::kRing) ring.start();
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t row = block * S::kGroups + group;
        const int limit = row < rows ? width : 0;
        if constexpr (S::kRing) {
            ring.open();
            S::load(reinterpret_cast<const typename S::T *>(ring.row(0, group)), limit, warp, lane, q);
            ring.close(block);
        } else {
            S::load(x + row * width, limit, warp, lane, q);
        }
        if (limit)
            pack_row<S>(
                [&](int c, float *v) {
                    q[c].values(v);
                    if (ring.bad)
#pragma unroll
                        for (int i = 0; i < S::kVec; ++i) v[i] = NAN;
                },
                width, warp, lane, packed + row * width, exponents + row * checkpoint_blocks(width));
    }
}

template <class S>
__global__ void __launch_bounds__(kRowThreads, 2)
    unpack_kernel(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int width, typename S::T *x,
                  RingPlan plan) {
    constexpr int kVec = S::kVec;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RingBars bars;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % S::kWpr, group = (threadIdx.x >> 5) / S::kWpr;
    const int64_t blocks = (rows + S::kGroups - 1) / S::kGroups;
    RowRing<S::kGroups> ring{plan, &bars, smem, {packed, nullptr}, rows};
    if constexpr (S::kRing) ring.start();
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t row = block * S::kGroups + group;
        const int limit = row < rows ? width : 0;
        const uint8_t *exps = exponents + row * checkpoint_blocks(width);
        PackedBytes<kVec> q[S::kChunks];
        uint8_t e[S::kChunks];
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                e[c] = exps[col / kCheckpointBlock];
                if (!S::kRing) q[c] = *reinterpret_cast<const PackedBytes<kVec> *>(packed + row * width + col);
            }
        }
        if constexpr (S::kRing) {
            ring.open();
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c) {
                const int col = S::column(c, warp, lane);
                if (col < limit) q[c] = *reinterpret_cast<const PackedBytes<kVec> *>(ring.row(0, group) + col);
            }
            ring.close(block);
        }
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int col = S::column(c, warp, lane);
            if (col < limit) {
                float v[kVec];
                unpack_bytes<kVec>(q[c], ring.bad ? NAN : checkpoint_scale(e[c]), v);
                store_vec<typename S::T, kVec>(x + row * width + col, v);
            }
        }
    }
}

// CTAs a SM.  Measured at 30,000 x 4,096 bf16: pack 78 us with two, 68 with
// three, 65 with four; unpack 116, 102, 109.
constexpr int kPackResident = 4, kUnpackResident = 3, kLaneResident = 4;

}  // namespace

void launch_checkpoint_pack(const void *x, int64_t rows, int width, int dtype, uint8_t *packed, uint8_t *exponents,
                            int sms, cudaStream_t stream) {
    if (rows == 0) return;
    const size_t row = width * dtype_bytes(dtype);
    const bool wide = whole_units(row, {x}) && packs_wide(packed, dtype);
    const int groups = row_groups(width, wide);
    const RingPlan plan = plan_ring(groups, row, 0, kPackResident);
    const unsigned grid = row_grid(rows, groups, sms, wide ? kPackResident : kLaneResident);
    with_rows(dtype, wide, width, [&](auto s) {
        using S = decltype(s);
        launch_rows(pack_kernel<S>, grid, S::kRing ? ring_bytes(plan, groups) : 0, stream,
                    static_cast<const typename S::T *>(x), rows, width, packed, exponents, plan);
    });
}

void launch_checkpoint_unpack(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int width, int dtype,
                              void *x, int sms, cudaStream_t stream) {
    if (rows == 0) return;
    const bool wide = whole_units(width, {packed}) && whole_units(width * dtype_bytes(dtype), {x});
    const int groups = row_groups(width, wide);
    const RingPlan plan = plan_ring(groups, width, 0, kUnpackResident);
    const unsigned grid = row_grid(rows, groups, sms, wide ? kUnpackResident : kLaneResident);
    with_rows(dtype, wide, width, [&](auto s) {
        using S = decltype(s);
        launch_rows(unpack_kernel<S>, grid, S::kRing ? ring_bytes(plan, groups) : 0, stream, packed, exponents, rows,
                    width, static_cast<typename S::T *>(x), plan);
    });
}

}  // namespace vfr
