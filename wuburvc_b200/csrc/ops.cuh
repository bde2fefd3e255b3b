// ops.cuh — what the transformer training operators (act8.cu, resnorm.cu, attention*.cu) share: element
// types, 16-byte loads and stores as floats, and the host-side checks.
#pragma once
#include <atomic>
#include <cstdio>

#include "../../include/wuburvc_b200.h"
#include "common.cuh"

namespace wb {

// The operators' device status word (one per device, see wubu_b200_ops_sync); nullptr on a CUDA error.
int* ops_status_word();
int ops_sms();  // SMs of the current device; 0 without one

// Raises a kernel's dynamic shared-memory limit, once per device (`devices`: the ones done).
inline bool ops_smem_limit(const void* kernel, int bytes, std::atomic<uint64_t>& devices) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (devices.load() >> dev & 1) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  devices.fetch_or(uint64_t(1) << dev);
  return true;
}

inline int ops_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return WUBU_B200_OK;
  fprintf(stderr, "wuburvc_b200: %s launch failed: %s\n", what, cudaGetErrorString(e));
  return WUBU_B200_ERR_CUDA;
}

// Launches a kernel that may start while its predecessor on the stream still runs (it waits for it with
// griddep_wait before it touches what that wrote).
template <typename... Args, typename... Given>
int ops_launch_after(void (*kernel)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char* what,
                     Given... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, Args(args)...);
  if (e == cudaSuccess) return WUBU_B200_OK;
  cudaGetLastError();
  fprintf(stderr, "wuburvc_b200: %s launch failed: %s\n", what, cudaGetErrorString(e));
  return WUBU_B200_ERR_CUDA;
}

inline bool ops_dtype_ok(int dtype) {
  return dtype == WUBU_B200_F32 || dtype == WUBU_B200_BF16 || dtype == WUBU_B200_F16;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

WB_DEV float to_float(float x) { return x; }
WB_DEV float to_float(bf16 x) { return __bfloat162float(x); }
WB_DEV float to_float(f16 x) { return __half2float(x); }
template <typename T>
WB_DEV T from_float(float x);
template <>
WB_DEV float from_float<float>(float x) { return x; }
template <>
WB_DEV bf16 from_float<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
WB_DEV f16 from_float<f16>(float x) { return __float2half_rn(x); }

// 8 values from 16-byte aligned memory (one 16-byte load, two for float), and back.
WB_DEV void load8(const float* p, float* v) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
WB_DEV void load8(const bf16* p, float* v) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
WB_DEV void load8(const f16* p, float* v) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
WB_DEV uint32_t pack2(float a, float b, bf16) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
WB_DEV uint32_t pack2(float a, float b, f16) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
WB_DEV void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
WB_DEV void store8(T* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                                            pack2(v[6], v[7], T()));
}

// Two float32 operations in one instruction.
WB_DEV uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
WB_DEV void each(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
WB_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
WB_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
WB_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Calls f(T()) with the element type of `dtype`.
template <typename F>
inline void with_dtype(int dtype, F f) {
  if (dtype == WUBU_B200_BF16) f(bf16());
  else if (dtype == WUBU_B200_F16) f(f16());
  else f(float());
}

}  // namespace wb
