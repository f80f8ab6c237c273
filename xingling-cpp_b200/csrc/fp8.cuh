// e4m3 rounding and typed 8-element accesses of the 8-bit serving operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged.h"
#include "xl_kernels.h"

namespace xl {

constexpr float kFp8Max = 448.0f;    // largest e4m3 value
constexpr uint8_t kFp8NaN = 0x7f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two floats to the low and high half of a word.
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 consecutive elements of a 16-byte aligned address, as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = u;
    }
}
// 8 elements as they lie in memory, so that several loads can be under way before the first is converted.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};
// VEC: all 8 (a 16-byte aligned address) or, with live 0, zeros.  Else the first `live`, zeros for the others.
template <bool VEC, typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p, int live) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (VEC) {
        if (live) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
        }
    } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) e[i] = p[i];
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float (&v)[8]) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
}

// 8 floats rounded to T, as they lie in memory.
template <typename T>
__device__ __forceinline__ Raw8<T> round_raw8(const float (&v)[8]) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 4) {
        float* e = reinterpret_cast<float*>(&r);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = v[i];
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_pair(v[2 * i], v[2 * i + 1], T{});
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store_raw8(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

// Two floats to two e4m3 bytes (the first in the low byte), to nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The e4m3 value nearest to v, in one rounding: v goes to 32 bits rounded to
// odd (truncated, the last bit set where anything was cut), which keeps it on
// its side of every e4m3 border, and then to 8 bits.
__device__ __forceinline__ uint32_t e4m3_of(double v) {
    float f = __double2float_rz(v);
    if (static_cast<double>(f) != v) f = __uint_as_float(__float_as_uint(f) | 1u);
    return e4m3x2(f, 0.0f) & 0xffu;
}

// Quotients of the fast path are off by less than kQuotientError of
// themselves and then raised by it, so they lie 0 to 16 units in the last
// place above the exact ones: a quotient on the other side of a border between
// two e4m3 values than the exact one, or on a border, is one of the 16 floats
// from the border on.  From 2^-6 on borders are where the 4th bit after the
// leading one is set and nothing follows: bits 4 .. 19 are those of 0x80000,
// and this is 0.
constexpr float kQuotientError = 4.76837158203125e-7f;  // 2^-21
__device__ __forceinline__ uint32_t border_bits(float q) { return (__float_as_uint(q) & 0xffff0u) ^ 0x80000u; }
// Below 2^-6 (steps of 2^-9) they are the odd multiples of 2^-10.
__device__ __forceinline__ bool near_border_small(float q) {
    const float m = fabsf(q) * 1024.0f, r = rintf(m);
    return m <= 16.5f && fabsf(m - r) < 4e-5f && (static_cast<int>(r) & 1);
}

}  // namespace xl
