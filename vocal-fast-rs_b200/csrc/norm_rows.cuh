// How the norm and checkpoint kernels hold rows: a row belongs to a group of
// one to eight warps, 8 to 24 values a lane in chunks of kVec, and the CTA's
// groups walk blocks of rows, one row each.
//
// The rows of a block are one run of memory.  Where every row starts and
// ends on 16 bytes, kVec is 16 bytes and one thread brings whole blocks into
// a ring in shared memory with bulk copies, several blocks ahead: what is in
// flight takes no registers.   Other rows are loaded by their lanes, element
// by element (kVec = 1).
#pragma once

#include <algorithm>
#include <initializer_list>

#include "pdl.cuh"
#include "row_io.cuh"
#include "tc_ptx.cuh"
#include "units.h"
#include "vfr_common.h"

namespace vfr {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

template <typename Type, int kVec_, int kWpr_, int kLane_>
struct RowShape {
    using T = Type;
    static constexpr int kVec = kVec_, kWpr = kWpr_, kLane = kLane_;
    static constexpr int kChunks = kLane / kVec;
    static constexpr bool kRing = kVec > 1;
    static constexpr int kGroups = kRowWarps / kWpr;  // rows a CTA works on
    using Raw = RawVec<T, kVec>;

    // First column of the lane's chunk c: a warp's chunks are contiguous, and
    // the 128 columns of a checkpoint block belong to one warp.
    static __device__ __forceinline__ int column(int c, int warp, int lane) {
        if constexpr (kVec == 1) return (((c >> 2) * kWpr + warp) << 7) + ((c & 3) << 5) + lane;
        return ((c * kWpr + warp) * 32 + lane) * kVec;
    }
    static __device__ __forceinline__ void load(const T *row, int limit, int warp, int lane, Raw (&q)[kChunks]) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int col = column(c, warp, lane);
            if (col < limit) {
                q[c] = *reinterpret_cast<const Raw *>(row + col);
            } else {
                q[c].clear();
            }
        }
    }
};

// The ring of a CTA: up to two operands of row_bytes each, `stages` blocks of
// kGroups rows.  A wait that gives up makes the ring `bad`: nothing more is
// copied or waited for, and the kernels write NaN.
struct RingPlan {
    int stages;
    uint32_t row_bytes[2];   // 0: no second operand
};
constexpr int kMaxStages = 8;
struct RingBars {
    uint64_t full[kMaxStages], empty[kMaxStages];
};
constexpr uint64_t kRowWaitNs = 2000000000ull;

template <int kGroups>
struct RowRing {
    RingPlan plan;
    RingBars *bars;
    uint8_t *smem;
    const uint8_t *base[2];
    int64_t rows;
    int stage = 0;
    uint32_t phase = 0;
    bool bad = false;

    __device__ __forceinline__ uint32_t block_bytes() const {
        return kGroups * (plan.row_bytes[0] + plan.row_bytes[1]);
    }
    __device__ __forceinline__ void copy(int64_t block, int s) {
        if (block * kGroups >= rows) return;
        const uint32_t n = static_cast<uint32_t>(rows - block * kGroups < kGroups ? rows - block * kGroups : kGroups);
        tc::mbar_arrive_expect_tx(&bars->full[s], n * (plan.row_bytes[0] + plan.row_bytes[1]));
        uint8_t *dst = smem + s * block_bytes();
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            if (plan.row_bytes[o])
                tc::bulk_load(dst, base[o] + block * kGroups * plan.row_bytes[o], n * plan.row_bytes[o],
                              &bars->full[s]);
            dst += kGroups * plan.row_bytes[o];
        }
    }
    // Every thread of the CTA.
    __device__ __forceinline__ void start() {
        if (threadIdx.x == 0) {
            for (int s = 0; s < plan.stages; ++s) {
                tc::mbar_init(&bars->full[s], 1);
                tc::mbar_init(&bars->empty[s], kRowWarps);
            }
            tc::fence_mbarrier_init();
        }
        __syncthreads();
        if (threadIdx.x == 0)
            for (int s = 0; s < plan.stages; ++s) copy(blockIdx.x + static_cast<int64_t>(s) * gridDim.x, s);
    }
    // The present block has landed: operand o of group g's row.
    __device__ __forceinline__ void open() {
        if (!bad) bad = !__all_sync(0xFFFFFFFFu, tc::mbar_wait(&bars->full[stage], phase, kRowWaitNs));
    }
    __device__ __forceinline__ const uint8_t *row(int o, int group) const {
        return smem + stage * block_bytes() + (o ? kGroups * plan.row_bytes[0] : 0) + group * plan.row_bytes[o];
    }
    // This warp has read its part of block `block`; the first thread fills the
    // stage again once every warp has.
    __device__ __forceinline__ void close(int64_t block) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&bars->empty[stage]);
        if (threadIdx.x == 0 && !bad) {
            const int64_t next = block + static_cast<int64_t>(plan.stages) * gridDim.x;
            if (next * kGroups < rows) {
                if (tc::mbar_wait(&bars->empty[stage], phase, kRowWaitNs)) {
                    tc::fence_proxy_async_smem();
                    copy(next, stage);
                } else {
                    bad = true;
                }
            }
        }
        __syncwarp();
        bad = __any_sync(0xFFFFFFFFu, bad);
        if (++stage == plan.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

// Host: the ring for rows of these sizes (second operand 0: none) where
// `resident` CTAs share a SM's shared memory.  A block is 32 KB at most (two
// operands: two CTAs a SM) or 24 KB, so two stages always fit.
constexpr size_t kRingRoom = 208 * 1024;
inline RingPlan plan_ring(int groups, size_t row_a, size_t row_b, int resident) {
    const size_t stages = std::min<size_t>(kMaxStages, kRingRoom / resident / (groups * (row_a + row_b)));
    return {static_cast<int>(stages), {static_cast<uint32_t>(row_a), static_cast<uint32_t>(row_b)}};
}
inline size_t ring_bytes(const RingPlan &p, int groups) {
    return static_cast<size_t>(p.stages) * groups * (p.row_bytes[0] + p.row_bytes[1]);
}

// Sums of a and b over the warps of a row.  `slots` holds two sets of
// 2 kRowWarps floats, used in turn: a warp can be at most one call ahead of
// the slowest of its group.
template <int kWpr>
__device__ __forceinline__ void row_sums(float &a, float &b, float *slots, int &turn, int group, int warp) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if constexpr (kWpr > 1) {
        float2 *s = reinterpret_cast<float2 *>(slots) + turn * kRowWarps + group * kWpr;
        if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * kWpr) : "memory");
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < kWpr; ++i) a += s[i].x, b += s[i].y;
        turn ^= 1;
    }
}
template <int kWpr>
__device__ __forceinline__ float row_sum(float a, float *slots, int &turn, int group, int warp) {
    float unused = 0.0f;
    row_sums<kWpr>(a, unused, slots, turn, group, warp);
    return a;
}

// The 8-bit checkpoint of the values a warp holds (converged, zeros past the
// width): block maxima by lane exchange, then e4m3 bytes and one exponent
// byte a block.
template <class S, class Values>
__device__ __forceinline__ void pack_row(Values values, int width, int warp, int lane, uint8_t *packed,
                                         uint8_t *exponents) {
    constexpr int kVec = S::kVec;
    constexpr int kStep = kVec == 1 ? 4 : 1;  // chunks that cover one run of blocks
#pragma unroll
    for (int c = 0; c < S::kChunks; c += kStep) {
        float v[kStep * kVec];
#pragma unroll
        for (int k = 0; k < kStep; ++k) values(c + k, v + k * kVec);
        float top = 0.0f;  // NaN takes no part in a maximum
#pragma unroll
        for (int i = 0; i < kStep * kVec; ++i) top = fmaxf(top, fabsf(v[i]));
        auto block_max = [](float m) {
            // a block is 32 lanes, or the 16 lanes that hold 8 elements each
            if constexpr (kVec != 8) return __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
#pragma unroll
            for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            return __float_as_uint(m);
        };
        uint32_t bits = block_max(top);
        if (__any_sync(0xFFFFFFFFu, bits == 0x7F800000u)) {
            // infinities take no part either, and become NaN
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < kStep * kVec; ++i) {
                if (isinf(v[i])) v[i] = NAN;
                top = fmaxf(top, fabsf(v[i]));
            }
            bits = block_max(top);
        }
        const uint32_t e = checkpoint_exponent(bits);
        const float inverse = checkpoint_inverse(e);
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            const int at = S::column(c + k, warp, lane);
            if (at < width) {
                store_packed<kVec>(packed + at, v + k * kVec, inverse);
                if (at % kCheckpointBlock == 0) exponents[at / kCheckpointBlock] = static_cast<uint8_t>(e);
            }
        }
    }
}

// Whether rows of `bytes` bytes from these bases (null: not used) all start
// and end on 16 bytes.
inline bool whole_units(size_t bytes, std::initializer_list<const void *> bases) {
    for (const void *p : bases)
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return bytes % 16 == 0;
}
// Packed bytes are written kVec at a time.
inline bool packs_wide(const void *packed, int dtype) {
    return reinterpret_cast<uintptr_t>(packed) % (16 / dtype_bytes(dtype)) == 0;
}

// Calls f(RowShape) for the element type, the access width and the warps a
// row takes. 
template <typename T, int kVec, class F>
void with_row_warps(int width, F &&f) {
    if (width <= 256) f(RowShape<T, kVec, 1, 8>{});
    else if (width <= 512) f(RowShape<T, kVec, 1, 16>{});
    else if (kVec > 1 && width <= 768) f(RowShape<T, kVec, 1, (kVec > 1 ? 24 : 16)>{});
    else if (width <= 1024) f(RowShape<T, kVec, 2, 16>{});
    else if (width <= 2048) f(RowShape<T, kVec, 4, 16>{});
    else f(RowShape<T, kVec, 8, 16>{});
}
template <typename T, class F>
void with_row_shape(bool wide, int width, F &&f) {
    if (wide) with_row_warps<T, 16 / sizeof(T)>(width, f);
    else with_row_warps<T, 1>(width, f);
}
template <class F>
void with_rows(int dtype, bool wide, int width, F &&f) {
    if (dtype == kF32) with_row_shape<float>(wide, width, f);
    else if (dtype == kBF16) with_row_shape<__nv_bfloat16>(wide, width, f);
    else with_row_shape<__half>(wide, width, f);
}
inline int row_groups(int width, bool wide) {
    return width <= (wide ? 768 : 512) ? 8 : width <= 1024 ? 4 : width <= 2048 ? 2 : 1;
}

// CTAs for `rows` rows: what the rows fill, or `resident` a SM.
inline unsigned row_grid(int64_t rows, int groups, int sms, int resident) {
    return static_cast<unsigned>(std::min<int64_t>((rows + groups - 1) / groups, static_cast<int64_t>(resident) * sms));
}

// Launches a row kernel, not as a dependent of the one before: CTAs that came
// early beside those of another grid would not spread evenly over the SMs, and
// their shares of the rows are fixed (30,000 x 4,096 bf16 packed and unpacked:
// 250 us so, 196 us in order).
template <class Kernel, class... Args>
void launch_rows(Kernel kernel, unsigned grid, size_t smem, cudaStream_t stream, const Args &...args) {
    if (smem > 40 * 1024)  // 48 KB with the kernels' static arrays need no leave
        cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom / 2));
    kernel<<<grid, kRowThreads, smem, stream>>>(args...);
    cuda_check(cudaGetLastError());
}

}  // namespace vfr
