// How the norm and checkpoint kernels hold rows: a row belongs to a group of
// one to eight warps, 8 or 16 values a lane in chunks of kVec (16 bytes, or
// single elements where rows or bases fit no 16-byte access), and the group
// walks the rows with the next row's loads in flight while it works on the
// present one.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "row_io.cuh"
#include "units.h"

namespace vfr {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

template <typename Type, int kVec_, int kWpr_, int kLane_>
struct RowShape {
    using T = Type;
    static constexpr int kVec = kVec_, kWpr = kWpr_, kLane = kLane_;
    static constexpr int kChunks = kLane / kVec;
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
#pragma unroll
                for (int i = 0; i < kVec; ++i) q[c].e[i] = T(0.0f);
            }
        }
    }
};

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
template <class S>
__device__ __forceinline__ void pack_row(const typename S::Raw (&q)[S::kChunks], int width, int warp, int lane,
                                         uint8_t *packed, uint8_t *exponents) {
    constexpr int kVec = S::kVec;
    constexpr int kStep = kVec == 1 ? 4 : 1;  // chunks that cover one run of blocks
#pragma unroll
    for (int c = 0; c < S::kChunks; c += kStep) {
        float v[kStep * kVec];
#pragma unroll
        for (int k = 0; k < kStep; ++k) q[c + k].values(v + k * kVec);
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

inline bool aligned_to(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// 16-byte accesses need rows of whole vectors and aligned bases (null: not
// used); packed bytes are then read and written kVec at a time.
inline bool wide_rows(int width, int dtype, std::initializer_list<const void *> values, const void *packed) {
    const int vec = 16 / static_cast<int>(dtype_bytes(dtype));
    if (width % vec) return false;
    for (const void *p : values)
        if (!aligned_to(p, 16)) return false;
    return aligned_to(packed, vec);
}

// Calls f(RowShape) for the element type, the access width and the warps a
// row takes.
template <typename T, int kVec, class F>
void with_row_warps(int width, F &&f) {
    if (width <= 256) f(RowShape<T, kVec, 1, 8>{});
    else if (width <= 512) f(RowShape<T, kVec, 1, 16>{});
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
inline int row_groups(int width) { return width <= 512 ? 8 : width <= 1024 ? 4 : width <= 2048 ? 2 : 1; }

// CTAs for `rows` rows: what the rows fill, or `resident` a SM.
inline unsigned row_grid(int64_t rows, int groups, int sms, int resident) {
    return static_cast<unsigned>(std::min<int64_t>((rows + groups - 1) / groups, static_cast<int64_t>(resident) * sms));
}

}  // namespace vfr
