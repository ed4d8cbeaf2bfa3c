// Marks functions that both the kernels and a plain C++ compiler take (the parts
// of a kernel's plan that are checked without a GPU).
#pragma once

#ifdef __CUDACC__
#define VMPS_HD __host__ __device__ __forceinline__
#else
#define VMPS_HD inline
#endif
