// Matrix product in e4m3 with a scale for each block of 128, fp32 sums.
//
//   Y[i][j] = sum_b sx[i][b] sw[j / 128][b] sum_{c in block b} xq[i][c] wq[j][c] + bias[j]
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.cuh"
#include "xl_device.cuh"
#include "xl_kernels.h"

namespace xl {

namespace {

constexpr int kT = 16;

// One output a thread, 16 x 16 outputs a CTA; operands pass through shared memory one block of 128 columns at a time.
template <typename T>
__global__ void __launch_bounds__(256) linear_fp8_kernel(int mode, const uint8_t* __restrict__ xq, size_t ldx,
                                                         const float* __restrict__ xs, const uint8_t* __restrict__ wq,
                                                         size_t ldw, const float* __restrict__ ws,
                                                         const float* __restrict__ bias, T* y, int n, int m, int k) {
    __shared__ float sx[kT][kFp8Block + 1], sw[kT][kFp8Block + 1];
    const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
    const int tiles_m = (m + kT - 1) / kT;
    const int i0 = static_cast<int>(blockIdx.x / tiles_m) * kT, j0 = static_cast<int>(blockIdx.x % tiles_m) * kT;
    const int i = i0 + ty, j = j0 + tx, blocks = (k + kFp8Block - 1) / kFp8Block;
    float acc = 0.0f;
    for (int b = 0; b < blocks; ++b) {
        for (int e = threadIdx.x; e < kT * kFp8Block; e += 256) {
            const int r = e / kFp8Block, c = e % kFp8Block, col = b * kFp8Block + c;
            __nv_fp8_e4m3 v;
            v.__x = i0 + r < n && col < k ? xq[(i0 + r) * ldx + col] : 0;
            sx[r][c] = static_cast<float>(v);
            v.__x = j0 + r < m && col < k ? wq[(j0 + r) * ldw + col] : 0;
            sw[r][c] = static_cast<float>(v);
        }
        __syncthreads();
        float part = 0.0f;
        for (int c = 0; c < kFp8Block; ++c) part = fmaf(sx[ty][c], sw[tx][c], part);
        if (i < n && j < m)
            acc = fmaf(xs[static_cast<size_t>(i) * blocks + b] * ws[static_cast<size_t>(j / kFp8Block) * blocks + b], part, acc);
        __syncthreads();
    }
    if (j < m && bias) acc += bias[j];
    const float partner = __shfl_xor_sync(0xffffffffu, acc, 1);
    if (i >= n || j >= m) return;
    if (mode == kGemvSwiGLU) {
        if (!(j & 1)) y[static_cast<size_t>(i) * (m / 2) + j / 2] = from_float<T>(silu(acc) * partner);
    } else {
        T* dst = y + static_cast<size_t>(i) * m + j;
        *dst = from_float<T>(mode == kGemvResidual ? to_float(*dst) + acc : acc);
    }
}

}  // namespace

cudaError_t launch_linear_fp8(int mode, int dtype, const uint8_t* xq, size_t ldx, const float* xs, const uint8_t* wq,
                              size_t ldw, const float* ws, const float* bias, void* y, int n, int m, int k, int num_sms,
                              cudaStream_t s) {
    const long long tiles = static_cast<long long>((n + kT - 1) / kT) * ((m + kT - 1) / kT);
    if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
    const int grid = static_cast<int>(tiles);
    count_launch();
    switch (dtype) {
        case kF32:
            linear_fp8_kernel<<<grid, 256, 0, s>>>(mode, xq, ldx, xs, wq, ldw, ws, bias, static_cast<float*>(y), n, m, k);
            break;
        case kBF16:
            linear_fp8_kernel<<<grid, 256, 0, s>>>(mode, xq, ldx, xs, wq, ldw, ws, bias, static_cast<__nv_bfloat16*>(y), n,
                                                   m, k);
            break;
        case kF16:
            linear_fp8_kernel<<<grid, 256, 0, s>>>(mode, xq, ldx, xs, wq, ldw, ws, bias, static_cast<__half*>(y), n, m, k);
            break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace xl
