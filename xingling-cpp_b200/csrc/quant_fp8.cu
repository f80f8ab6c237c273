// e4m3 quantisation with a scale per 128 columns, alone (activations: one row
// a scale; weights: 128 rows a scale) and behind the residual addition and
// RMSNorm of a sublayer's input.
//
//   a = max |y| over the group, s = fl32(a / 448), q = e4m3(y / s)
//
// A group of zeros has s = 0 and q = 0; a group that holds a value that is
// not finite has s = NaN and q = NaN, so what it stands for shows it.
//
// The quotients are formed in 32 bits and checked against the borders between
// e4m3 values; the few that lie next to one are formed again in 64 bits.  So
// q is the nearest e4m3 value to the exact y / s, whatever the rounding of
// the fast path, and does not depend on how the work is split.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fp8.cuh"
#include "xl_device.cuh"
#include "xl_kernels.h"

namespace xl {

namespace {

constexpr int kLanesPerGroup = 16;  // lanes that share a group: 8 columns each
constexpr double kNormEps = 1e-6;   // as the engine's RMSNorm

// What divides a group's values: the stored scale and its reciprocal (raised, see kQuotientError).
struct GroupScale {
    float s, inv;
    bool exact_only;  // the reciprocal overflows (a scale near the smallest floats)
};
__device__ __forceinline__ GroupScale group_scale(float s) {
    GroupScale g;
    g.s = s;
    g.exact_only = s > 0.0f && s < 1e-30f;
    g.inv = s > 0.0f ? __fdividef(1.0f + kQuotientError, s) : 0.0f;  // within 2 ulp: s is below 2^126
    return g;
}

// Bytes of 8 quotients; y(i) is the exact value in 64 bits, fast(i) its quotient by the scale in 32.
template <typename Fast, typename Exact>
__device__ __forceinline__ uint2 quantise8(const GroupScale& g, Fast fast, Exact y) {
    float q[8], least = INFINITY;
    uint32_t bits = 1u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = fast(i);
        bits = min(bits, border_bits(q[i]));
        least = fminf(least, fabsf(q[i]));
    }
    bool close = g.exact_only || bits == 0u;
    if (least < 0.015625f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) close |= near_border_small(q[i]);
    }
    uint2 out;
    out.x = e4m3x2(q[0], q[1]) | e4m3x2(q[2], q[3]) << 16;
    out.y = e4m3x2(q[4], q[5]) | e4m3x2(q[6], q[7]) << 16;
    if (close && g.s > 0.0f) {
        out = make_uint2(0u, 0u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = e4m3_of(y(i) / static_cast<double>(g.s));
            if (i < 4) out.x |= b << (8 * i);
            else out.y |= b << (8 * (i - 4));
        }
    }
    if (!(g.s >= 0.0f)) out.x = out.y = kFp8NaN * 0x01010101u;
    return out;
}

__device__ __forceinline__ void store_bytes(uint8_t* p, uint2 b, int live) {
    if (live >= 8) {
        *reinterpret_cast<uint2*>(p) = b;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) p[i] = static_cast<uint8_t>((i < 4 ? b.x : b.y) >> (8 * (i & 3)));
    }
}

// Magnitudes compare as unsigned integers, with NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned long long abs_bits(double v) {
    return static_cast<unsigned long long>(__double_as_longlong(v)) & 0x7fffffffffffffffull;
}
template <typename U>
__device__ __forceinline__ U umax(U a, U b) { return a > b ? a : b; }

__device__ __forceinline__ float scale_of(uint32_t a) {
    return a < 0x7f800000u ? __fdiv_rn(__uint_as_float(a), kFp8Max) : __uint_as_float(0x7fffffffu);
}

template <typename T>
__device__ __forceinline__ uint2 quantise_plain(const float (&v)[8], const GroupScale& g) {
    return quantise8(
        g, [&](int i) { return v[i] * g.inv; }, [&](int i) { return static_cast<double>(v[i]); });
}

// One scale per row and 128 columns: 16 lanes a group, 8 columns a lane.  Bound
// by its bytes where there are many (151669 x 1536 fp32: 220 us, 5.3 TB/s), by
// the launch where there are few (8 x 1536: 1.7 us).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, size_t ldx, uint8_t* __restrict__ q,
                                                            size_t ldq, float* __restrict__ scale, uint32_t groups,
                                                            FastDiv per_row, int k) {
    const uint32_t stride = gridDim.x * (256 / kLanesPerGroup);
    const int sub = threadIdx.x % kLanesPerGroup;
    // whole warps stay in the loop: the reductions shuffle across the half-warp only, but name the warp
    const uint32_t first = blockIdx.x * (256 / kLanesPerGroup) + (threadIdx.x / 32) * 2;
    for (uint32_t base = first; base < groups; base += stride) {
        const uint32_t gi = base + (threadIdx.x / kLanesPerGroup) % 2;
        const bool on = gi < groups;
        const uint32_t row = on ? per_row.div(gi) : 0u;
        const int c = static_cast<int>(gi - row * per_row.d) * kFp8Block + sub * 8;
        const int live = on ? max(0, min(8, k - c)) : 0;
        float v[8];
        to_floats(load_raw8<VEC>(x + row * ldx + (live ? c : 0), live), v);
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = umax(a, abs_bits(v[i]));
#pragma unroll
        for (int o = kLanesPerGroup / 2; o; o >>= 1) a = umax(a, __shfl_xor_sync(0xffffffffu, a, o));
        const GroupScale g = group_scale(scale_of(a));
        const uint2 b = quantise_plain<T>(v, g);
        if (live) store_bytes(q + row * ldq + c, b, live);
        if (on && sub == 0) scale[gi] = g.s;
    }
}

// One scale per block of 128 x 128: a CTA keeps the block in registers, so it
// is read once (64 values a thread, 16 loads of 16 bytes in flight for fp32).
// Bound by its bytes: 151669 x 1536 fp32 in 197 us, 5.9 TB/s.  bf16 blocks are
// not (26620 x 2072: 87 us, 1.9 TB/s): 8-bit values meet exact borders often and
// a warp then takes the 64-bit path, though borders decided by a remainder's
// sign instead took as long, so that may not be all of it.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* __restrict__ x, size_t ldx, uint8_t* __restrict__ q,
                                                              size_t ldq, float* __restrict__ scale, FastDiv per_row,
                                                              int n, int k) {
    __shared__ uint32_t red[8];
    const uint32_t rb = per_row.div(blockIdx.x);
    const int c = static_cast<int>(blockIdx.x - rb * per_row.d) * kFp8Block + (threadIdx.x % kLanesPerGroup) * 8;
    const int live = max(0, min(8, k - c));
    const long long r0 = static_cast<long long>(rb) * kFp8Block + threadIdx.x / kLanesPerGroup;
    Raw8<T> raw[8];
    float v[8][8];
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long r = r0 + 16 * j;
        const bool on = r < n && live;
        raw[j] = load_raw8<VEC>(x + (on ? r * ldx + c : 0), on ? live : 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) to_floats(raw[j], v[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) a = umax(a, abs_bits(v[j][i]));
#pragma unroll
    for (int o = 16; o; o >>= 1) a = umax(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) a = umax(a, red[w]);
    const GroupScale g = group_scale(scale_of(a));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long r = r0 + 16 * j;
        if (r < n && live) store_bytes(q + r * ldq + c, quantise_plain<T>(v[j], g), live);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = g.s;
}

// 1 / sqrt(v) in 64 bits: Newton's iteration y (3 - v y^2) / 2 from the 32-bit
// function, whose 2^-22 two steps square down below 2^-80.
__device__ __forceinline__ double inverse_root(double v) {
    if (!(v < 1e37)) return 1.0 / sqrt(v);
    double y = rsqrtf(static_cast<float>(v));
    y *= fma(-0.5 * v * y, y, 1.5);
    return y * fma(-0.5 * v * y, y, 1.5);
}

// r = fl_T(residual + delta) (stored where there is a delta), rs =
// 1 / sqrt(mean(r^2) + eps), y = r gamma rs, e4m3 per row and 128 columns.
// One row a CTA, kept in registers (CHUNKS x 8 columns a thread), so each
// input is read once.  The sum of squares is 64-bit and the largest |r gamma|
// of a group is taken with the remainder of its fp32 product, the largest among
// those that round to the same (rounding keeps the order, but not strictly), so
// that a group's scale is the rounded exact one.  fp32 rows are
// bound by their bytes (4095 x 8192: 77 us, 5.7 TB/s), bf16 rows by some 40
// instructions a value (60 us, 3.9 TB/s); 8 x 1536 takes 2.4 us, a row's chain.
template <typename T, int CHUNKS, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1) add_rmsnorm_fp8_kernel(const T* __restrict__ delta, const T* residual, T* sum,
                                                                  const float* __restrict__ gamma,
                                                                  uint8_t* __restrict__ q, size_t ldq,
                                                                  float* __restrict__ scale, int k) {
    __shared__ double red[32];
    const size_t row = blockIdx.x;
    const int warp = threadIdx.x >> 5;
    const double per_k = 1.0 / k;
    Raw8<T> raw_r[CHUNKS], raw_d[CHUNKS];
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = static_cast<int>(threadIdx.x + j * blockDim.x) * 8;
        const int live = max(0, min(8, k - c));
        const size_t at = row * k + (live ? c : 0);
        raw_r[j] = load_raw8<VEC>(residual + at, live);
        raw_d[j] = load_raw8<VEC>(delta + at, delta ? live : 0);
    }
    float r[CHUNKS][8];
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        to_floats(raw_r[j], r[j]);
        if (delta) {
            const int c = static_cast<int>(threadIdx.x + j * blockDim.x) * 8;
            const int live = max(0, min(8, k - c));
            const size_t at = row * k + (live ? c : 0);
            float d[8];
            to_floats(raw_d[j], d);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] += d[i];
            if constexpr (sizeof(T) == 2) {
                const Raw8<T> rounded = round_raw8<T>(r[j]);
                to_floats(rounded, r[j]);
                if (VEC && live) store_raw8(sum + at, rounded);
            } else {
                if (VEC && live) store8(sum + at, r[j]);
            }
            if (!VEC) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < live) sum[at + i] = from_float<T>(r[j][i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double x = r[j][i];
            ss = fma(x, x, ss);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 31) == 0) red[warp] = ss;
    __syncthreads();
    ss = 0.0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) ss += red[w];
    const double rs = inverse_root(fma(ss, per_k, kNormEps));
    const double rs448 = rs * (1.0 / static_cast<double>(kFp8Max));
    const float rs_hi = static_cast<float>(rs448), rs_lo = static_cast<float>(rs448 - static_cast<double>(rs_hi));
    const int per_row = (k + kFp8Block - 1) / kFp8Block;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = static_cast<int>(threadIdx.x + j * blockDim.x) * 8;
        const int live = max(0, min(8, k - c));
        float w[8], p[8];
        to_floats(load_raw8<VEC>(gamma + (live ? c : 0), live), w);
        float own = 0.0f;  // the lane's largest product (NaN if there is one)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = r[j][i] * w[i];
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(own) : "f"(fabsf(p[i])));
        }
        const uint32_t mine = __float_as_uint(own);
        uint32_t a = mine;
#pragma unroll
        for (int o = kLanesPerGroup / 2; o; o >>= 1) a = umax(a, __shfl_xor_sync(0xffffffffu, a, o));
        // the group's largest product, exactly: its rounded value and the largest remainder among those that round to it
        const float top = __uint_as_float(a);
        float rest = -INFINITY;
        if (mine == a) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (fabsf(p[i]) == top) rest = fmaxf(rest, fmaf(fabsf(r[j][i]), fabsf(w[i]), -top));
        }
#pragma unroll
        for (int o = kLanesPerGroup / 2; o; o >>= 1) rest = fmaxf(rest, __shfl_xor_sync(0xffffffffu, rest, o));
        // top / 448 / root to 2^-46, then rounded once
        const float t = top * rs_hi;
        float s = t + (fmaf(top, rs_hi, -t) + fmaf(top, rs_lo, rest * rs_hi));
        // out of the range where these are exact (and for a group of zeros, where nothing is lost): 64 bits
        const bool far = !(top < 1e30f) || top < 1e-20f || !(rs_hi > 1e-15f);
        if (__any_sync(0xffffffffu, far)) {
            unsigned long long e = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) e = umax(e, abs_bits(static_cast<double>(r[j][i]) * static_cast<double>(w[i])));
#pragma unroll
            for (int o = kLanesPerGroup / 2; o; o >>= 1) e = umax(e, __shfl_xor_sync(0xffffffffu, e, o));
            if (far) s = static_cast<float>(__longlong_as_double(static_cast<long long>(e)) * rs448);
        }
        if (!(s <= 3.4e38f)) s = __uint_as_float(0x7fffffffu);
        GroupScale g;
        g.s = s;
        // 448 (1 + error) / top, within 4 ulp of rs / s: the products are at most top
        g.inv = s > 0.0f ? __fdividef(rs_hi * (kFp8Max * (1.0f + kQuotientError)), s) : 0.0f;
        g.exact_only = far;
        const uint2 b = quantise8(
            g, [&](int i) { return p[i] * g.inv; },
            [&](int i) { return static_cast<double>(r[j][i]) * static_cast<double>(w[i]) * rs; });
        if (live) {
            store_bytes(q + row * ldq + c, b, live);
            if (threadIdx.x % kLanesPerGroup == 0) scale[row * per_row + c / kFp8Block] = s;
        }
    }
}

template <typename T, bool VEC>
cudaError_t launch_norm_typed(const void* delta, const void* residual, void* sum, const float* gamma, uint8_t* q,
                              size_t ldq, float* scale, int n, int k, int num_sms, cudaStream_t s) {
    const int chunks = (k + 7) / 8;
    const T *d = static_cast<const T*>(delta), *r = static_cast<const T*>(residual);
    T* o = static_cast<T*>(sum);
    count_launch();
    auto threads = [&](int per) { return ((chunks + per - 1) / per + 31) / 32 * 32; };
    // Few rows: as many threads as a row has chunks, for the shortest chain; many: more columns a thread, so that an
    // SM holds more rows at different points of theirs.
    const bool few = n <= 2 * num_sms;
    if (chunks <= 256 && (few || chunks <= 64))
        add_rmsnorm_fp8_kernel<T, 1, 256, VEC><<<n, threads(1), 0, s>>>(d, r, o, gamma, q, ldq, scale, k);
    else if (chunks <= 512)
        add_rmsnorm_fp8_kernel<T, 2, 256, VEC><<<n, threads(2), 0, s>>>(d, r, o, gamma, q, ldq, scale, k);
    else if (chunks <= 1024)
        add_rmsnorm_fp8_kernel<T, 4, 256, VEC><<<n, threads(4), 0, s>>>(d, r, o, gamma, q, ldq, scale, k);
    else
        add_rmsnorm_fp8_kernel<T, 4, 1024, VEC><<<n, threads(4), 0, s>>>(d, r, o, gamma, q, ldq, scale, k);
    return cudaGetLastError();
}

template <typename T, bool VEC>
cudaError_t launch_quantize_typed(const T* x, size_t ldx, uint8_t* q, size_t ldq, float* scale, int n, int k, int rows,
                                  int num_sms, cudaStream_t s) {
    const uint32_t per_row = static_cast<uint32_t>((k - 1) / kFp8Block + 1);
    count_launch();
    if (rows == 1) {
        const uint32_t groups = static_cast<uint32_t>(n) * per_row;
        const uint32_t ctas = (groups + 15) / 16, most = static_cast<uint32_t>(num_sms) * 32;
        quantize_rows_kernel<T, VEC><<<ctas < most ? ctas : most, 256, 0, s>>>(x, ldx, q, ldq, scale, groups,
                                                                               FastDiv(per_row), k);
    } else {
        const uint32_t blocks = static_cast<uint32_t>((n - 1) / kFp8Block + 1) * per_row;
        quantize_blocks_kernel<T, VEC><<<blocks, 256, 0, s>>>(x, ldx, q, ldq, scale, FastDiv(per_row), n, k);
    }
    return cudaGetLastError();
}

// Whole 16-byte loads: k in eights, rows that stay aligned.
template <typename T>
cudaError_t launch_quantize_typed(const void* xv, size_t ldx, uint8_t* q, size_t ldq, float* scale, int n, int k,
                                  int rows, int num_sms, cudaStream_t s) {
    const T* x = static_cast<const T*>(xv);
    const bool vec = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * sizeof(T)) % 16 == 0;
    return vec ? launch_quantize_typed<T, true>(x, ldx, q, ldq, scale, n, k, rows, num_sms, s)
               : launch_quantize_typed<T, false>(x, ldx, q, ldq, scale, n, k, rows, num_sms, s);
}
template <typename T>
cudaError_t launch_norm_typed(const void* delta, const void* residual, void* sum, const float* gamma, uint8_t* q,
                              size_t ldq, float* scale, int n, int k, int num_sms, cudaStream_t s) {
    return k % 8 == 0 ? launch_norm_typed<T, true>(delta, residual, sum, gamma, q, ldq, scale, n, k, num_sms, s)
                      : launch_norm_typed<T, false>(delta, residual, sum, gamma, q, ldq, scale, n, k, num_sms, s);
}

}  // namespace

cudaError_t launch_quantize_fp8(int dtype, const void* x, size_t ldx, uint8_t* q, size_t ldq, float* scale, int n, int k,
                                int rows, int num_sms, cudaStream_t s) {
    switch (dtype) {
        case kF32: return launch_quantize_typed<float>(x, ldx, q, ldq, scale, n, k, rows, num_sms, s);
        case kBF16: return launch_quantize_typed<__nv_bfloat16>(x, ldx, q, ldq, scale, n, k, rows, num_sms, s);
        case kF16: return launch_quantize_typed<__half>(x, ldx, q, ldq, scale, n, k, rows, num_sms, s);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_add_rmsnorm_fp8(int dtype, const void* delta, const void* residual, void* sum, const float* gamma,
                                   uint8_t* q, size_t ldq, float* scale, int n, int k, int num_sms, cudaStream_t s) {
    switch (dtype) {
        case kF32: return launch_norm_typed<float>(delta, residual, sum, gamma, q, ldq, scale, n, k, num_sms, s);
        case kBF16: return launch_norm_typed<__nv_bfloat16>(delta, residual, sum, gamma, q, ldq, scale, n, k, num_sms, s);
        case kF16: return launch_norm_typed<__half>(delta, residual, sum, gamma, q, ldq, scale, n, k, num_sms, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace xl
