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

// Two f32 operations at a time.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// Elementwise on kVec values, two at a time where they come in pairs.
template <int kVec>
__device__ __forceinline__ void add_to(float *a, const float *b) {  // a += b
    if constexpr (kVec == 1) {
        a[0] += b[0];
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = add2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = r.x, a[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void add_scalar(float *a, float s) {  // a += s
    if constexpr (kVec == 1) {
        a[0] += s;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = add2(make_float2(a[i], a[i + 1]), make_float2(s, s));
            a[i] = r.x, a[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void mul_by(float *a, const float *b) {  // a *= b
    if constexpr (kVec == 1) {
        a[0] *= b[0];
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = mul2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = r.x, a[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void mul_scalar(float *a, float s) {  // a *= s
    if constexpr (kVec == 1) {
        a[0] *= s;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = mul2(make_float2(a[i], a[i + 1]), make_float2(s, s));
            a[i] = r.x, a[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void fma_to(float *acc, const float *a, const float *b) {  // acc += a b
    if constexpr (kVec == 1) {
        acc[0] = fmaf(a[0], b[0], acc[0]);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]),
                                  make_float2(acc[i], acc[i + 1]));
            acc[i] = r.x, acc[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void fma_scalars(float *a, float m, float s) {  // a = a m + s
    if constexpr (kVec == 1) {
        a[0] = fmaf(a[0], m, s);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(m, m), make_float2(s, s));
            a[i] = r.x, a[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ void fma_scalar(float *acc, const float *a, float s) {  // acc += a s
    if constexpr (kVec == 1) {
        acc[0] = fmaf(a[0], s, acc[0]);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(s, s), make_float2(acc[i], acc[i + 1]));
            acc[i] = r.x, acc[i + 1] = r.y;
        }
    }
}
template <int kVec>
__device__ __forceinline__ float sum_of(const float *a) {
    float s = a[0];
#pragma unroll
    for (int i = 1; i < kVec; ++i) s += a[i];
    return s;
}

// Two 16-bit values at a time.
__device__ __forceinline__ float2 pair_f32(uint32_t q, __nv_bfloat16) {
    return make_float2(__uint_as_float(q << 16), __uint_as_float(q & 0xFFFF0000u));
}
__device__ __forceinline__ float2 pair_f32(uint32_t q, __half) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&q));
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, __half) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// kVec consecutive elements as loaded: kVec * sizeof(T) bytes, aligned to that size.
template <typename T, int kVec>
struct RawVec {
    static_assert(sizeof(T) * kVec == 16, "16 bytes or one element");
    uint4 w;
    __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void values(float *v) const {
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(q[i]);
            } else {
                const float2 f = pair_f32(q[i], T());
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float *v) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) q[i] = __float_as_uint(v[i]);
            else q[i] = pair_bits(v[2 * i], v[2 * i + 1], T());
        }
        w = make_uint4(q[0], q[1], q[2], q[3]);
    }
};
template <typename T>
struct RawVec<T, 1> {
    T w;
    __device__ __forceinline__ void clear() { w = T(0.0f); }
    __device__ __forceinline__ void values(float *v) const { v[0] = to_f32(w); }
    __device__ __forceinline__ void set(const float *v) { w = from_f32<T>(v[0]); }
};
template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T *p, float *v) {
    const RawVec<T, kVec> q = *reinterpret_cast<const RawVec<T, kVec> *>(p);
    q.values(v);
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
    RawVec<T, kVec> q;
    q.set(v);
    *reinterpret_cast<RawVec<T, kVec> *>(p) = q;
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
struct PackedBytes;
template <>
struct PackedBytes<1> {
    uint8_t w;
};
template <>
struct PackedBytes<4> {
    uint32_t w;
};
template <>
struct PackedBytes<8> {
    uint2 w;
};
__device__ __forceinline__ void unpack_word(uint32_t w, float *v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
template <int kVec>
__device__ __forceinline__ void unpack_bytes(const PackedBytes<kVec> &q, float scale, float *v) {
    if constexpr (kVec == 1) {
        v[0] = checkpoint_value(q.w) * scale;
    } else {
        if constexpr (kVec == 4) {
            unpack_word(q.w, v);
        } else {
            unpack_word(q.w.x, v);
            unpack_word(q.w.y, v + 4);
        }
        mul_scalar<kVec>(v, scale);
    }
}
__device__ __forceinline__ uint32_t pack_word(const float *v) {
    return checkpoint_pair(v[0], v[1]) | checkpoint_pair(v[2], v[3]) << 16;
}
template <int kVec>
__device__ __forceinline__ void store_packed(uint8_t *p, const float *v, float inverse) {
    float s[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) s[i] = v[i];
    mul_scalar<kVec>(s, inverse);
    PackedBytes<kVec> q;
    if constexpr (kVec == 1) q.w = static_cast<uint8_t>(checkpoint_pair(s[0], 0.0f));
    else if constexpr (kVec == 4) q.w = pack_word(s);
    else q.w = make_uint2(pack_word(s), pack_word(s + 4));
    *reinterpret_cast<PackedBytes<kVec> *>(p) = q;
}

}  // namespace vfr
