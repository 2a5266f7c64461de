// vx_ops.cuh — what the stand-alone serving operators share: element types, argument
// refusals, the status word and bounded waits.
//
// These operators run on the caller's device memory and belong to no handle, so a kernel
// that meets a bad index or a wait that expires reports it in the caller's status word
// (nullable), with the codes of DevError; the first one stays.
#pragma once
#include <cuda_bf16.h>

#include "vx_common.cuh"

namespace vx {
namespace ops {

template <typename T> struct Elem;
template <> struct Elem<__half> {
  static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static constexpr uint32_t kIdescType = 0;   // tcgen05 kind::f16 operand format F16
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static constexpr uint32_t kIdescType = 1;   // BF16
};
template <> struct Elem<float> {
  static __device__ __forceinline__ float to_f32(float v) { return v; }
  static __device__ __forceinline__ float from_f32(float v) { return v; }
};

__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// Wait on an mbarrier phase, bounded: after kSpinLimit polls, or once another wait of the
// CTA has given up (*abort), it returns false and the caller unwinds.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* status, int code) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *abort) return false;
  }
  *abort = 1;
  report(status, code);
  return false;
}
// The same for copies in flight, which always land: another wait's failure does not end it.
__device__ __forceinline__ void wait_landed(uint64_t* bar, uint32_t parity, int32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; ++i)
    if (mbar_try_wait(bar, parity)) return;
  report(status, kDevTimeoutDrain);
}

}  // namespace ops
}  // namespace vx
