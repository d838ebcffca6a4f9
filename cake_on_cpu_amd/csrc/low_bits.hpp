// low_bits.hpp -- the element types of the operators beyond fp32 and the vector types their
// kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "cake_hip.h"

namespace cake {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

inline __host__ __device__ int type_bytes(int type) { return type == CAKE_HIP_F32 ? 4 : 2; }

template <int TYPE> struct Element;
template <> struct Element<CAKE_HIP_F32> { typedef float T; };
template <> struct Element<CAKE_HIP_F16> { typedef _Float16 T; };
template <> struct Element<CAKE_HIP_BF16> { typedef __bf16 T; };

// element i of an array whose type is known at run time (the same for every lane)
__device__ __forceinline__ float load_as_float(const void* p, size_t i, int type)
{
    if (type == CAKE_HIP_F32) return static_cast<const float*>(p)[i];
    if (type == CAKE_HIP_F16) return (float)static_cast<const _Float16*>(p)[i];
    return (float)static_cast<const __bf16*>(p)[i];
}
// one rounding, to nearest, ties to even
__device__ __forceinline__ void store_from_float(void* p, size_t i, int type, float v)
{
    if (type == CAKE_HIP_F32) static_cast<float*>(p)[i] = v;
    else if (type == CAKE_HIP_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
    else static_cast<__bf16*>(p)[i] = (__bf16)v;
}

}  // namespace cake
