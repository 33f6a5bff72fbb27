// Values of the three floating types that the operators around a stack take, computed with in 32 bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "cbm_b200.h"

namespace cbm {

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// Calls `f` with a value of the type that `type` names; false where it names none.
template <class F>
bool with_type(int32_t type, F&& f) {
    switch (type) {
        case CBM_B200_FP32: f(float()); return true;
        case CBM_B200_BF16: f(__nv_bfloat16()); return true;
        case CBM_B200_FP16: f(__half()); return true;
        default: return false;
    }
}
inline int size_of_type(int32_t type) { return type == CBM_B200_FP32 ? 4 : 2; }

}  // namespace cbm
