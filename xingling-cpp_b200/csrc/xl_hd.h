// Marks arithmetic that kernels share with the checks that run on the host.
#pragma once

#ifdef __CUDACC__
#define XL_HD __host__ __device__ __forceinline__
#else
#define XL_HD inline
#endif
