// Row loads and stores of f32 / bf16 / f16 values as f32, one element or 16
// bytes at a time, and the e4m3 checkpoint encoding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace vfr {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// kVec consecutive elements as loaded: kVec * sizeof(T) bytes, aligned to that size.
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) RawVec {
    T e[kVec];
    __device__ __forceinline__ void values(float *v) const {
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = to_f32(e[i]);
    }
};
template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T *p, float *v) {
    if constexpr (kVec == 1) {
        v[0] = to_f32(*p);
    } else {
        struct alignas(sizeof(T) * kVec) Pack {
            T e[kVec];
        };
        const Pack q = *reinterpret_cast<const Pack *>(p);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = to_f32(q.e[i]);
    }
}
// kVec f32 parameters, 16-byte aligned where kVec > 1.
template <int kVec>
__device__ __forceinline__ void load_params(const float *p, float *v) {
    if constexpr (kVec == 1) {
        v[0] = __ldg(p);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4 *>(p + i));
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    }
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
    if constexpr (kVec == 1) {
        *p = from_f32<T>(v[0]);
    } else {
        struct alignas(sizeof(T) * kVec) Pack {
            T e[kVec];
        } q;
#pragma unroll
        for (int i = 0; i < kVec; ++i) q.e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<Pack *>(p) = q;
    }
}

// ---- 8-bit checkpoints
// A block of 128 elements of a row shares the power of two 2^s, s the
// smallest (not below -127) that brings the block's largest finite magnitude
// to at most 448, e4m3's largest value.  A power of two costs no precision in
// a floating format, x 2^-s is exact wherever e4m3 can hold it, and every
// host and device gets the same bytes.  Stored as the byte s + 127.
// `top` holds the largest finite magnitude's f32 bits (0 for an all-zero block).
__device__ __forceinline__ uint32_t checkpoint_exponent(uint32_t top) {
    const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u);
    return e > 0 ? e : 0;
}
// 2^-s for the byte s + 127 <= 247 (2^-120 .. 2^127, all normal).
__device__ __forceinline__ float checkpoint_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^s; the byte 0 stands for 2^-127, a subnormal.
__device__ __forceinline__ float checkpoint_scale(uint32_t byte) {
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x400000u);
}
// Two values already multiplied by 2^-s to e4m3 bytes (first in the low
// byte), to nearest even; NaN becomes the format's NaN, infinities its
// largest value.
__device__ __forceinline__ uint32_t checkpoint_pair(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float checkpoint_value(uint8_t q) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

// kVec e4m3 bytes as loaded.
template <int kVec>
struct alignas(kVec) PackedBytes {
    uint8_t e[kVec];
};
template <int kVec>
__device__ __forceinline__ void unpack_bytes(const PackedBytes<kVec> &q, float scale, float *v) {
    if constexpr (kVec == 1) {
        v[0] = checkpoint_value(q.e[0]) * scale;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
                static_cast<__nv_fp8x2_storage_t>(q.e[i] | (q.e[i + 1] << 8)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            v[i] = f.x * scale;
            v[i + 1] = f.y * scale;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void store_packed(uint8_t *p, const float *v, float inverse) {
    PackedBytes<kVec> q;
    if constexpr (kVec == 1) {
        q.e[0] = static_cast<uint8_t>(checkpoint_pair(v[0] * inverse, 0.0f));
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const uint32_t r = checkpoint_pair(v[i] * inverse, v[i + 1] * inverse);
            q.e[i] = static_cast<uint8_t>(r);
            q.e[i + 1] = static_cast<uint8_t>(r >> 8);
        }
    }
    *reinterpret_cast<PackedBytes<kVec> *>(p) = q;
}

}  // namespace vfr
