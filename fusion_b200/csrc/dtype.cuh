// Element types of the kernels that take bf16, fp16 and fp32 (FUS_DT_*), with fp32 arithmetic.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace fus {

FUS_DEVICE float to_f(float v) { return v; }
FUS_DEVICE float to_f(__half v) { return __half2float(v); }
FUS_DEVICE float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
FUS_DEVICE T from_f(float v);
template <>
FUS_DEVICE float from_f<float>(float v) { return v; }
template <>
FUS_DEVICE __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
FUS_DEVICE __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline bool dtype_known(int dtype) {
  return dtype == FUS_DT_BF16 || dtype == FUS_DT_F16 || dtype == FUS_DT_F32;
}
inline int dtype_size(int dtype) { return dtype == FUS_DT_F32 ? 4 : 2; }

}  // namespace fus
