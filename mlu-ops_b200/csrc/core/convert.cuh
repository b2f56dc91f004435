// Device helpers shared by the operators: conversions between a storage type and
// float, and moves of several consecutive values at once.
#ifndef MLUOP_B200_CORE_CONVERT_CUH_
#define MLUOP_B200_CORE_CONVERT_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mluop {

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T fromFloat(float v);
template <>
__device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values, moved as vectors of up to 16 bytes; the address is aligned to them.
template <int N, typename T>
struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) Pack {
  T v[N];
};
template <int N, typename T>
__device__ __forceinline__ Pack<N, T> loadPack(const T *p) { return *reinterpret_cast<const Pack<N, T> *>(p); }
template <int N, typename T>
__device__ __forceinline__ void storePack(T *p, const Pack<N, T> &v) { *reinterpret_cast<Pack<N, T> *>(p) = v; }

}  // namespace mluop

#endif  // MLUOP_B200_CORE_CONVERT_CUH_
