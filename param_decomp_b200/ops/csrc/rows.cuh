// Helpers of the kernels that walk rows of bf16 or fp32 elements: eight columns at a time as 16-byte words, warp sums,
// and launches that overlap their set-up with the end of the kernel before them.
#pragma once

#include <atomic>

#include "common.cuh"

namespace pd {

template <typename T>
struct Raw8 {  // eight elements as they lie in memory
  uint4 q[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {  // p is 16-byte aligned
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.q[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(r.q[i].x);
    v[4 * i + 1] = __uint_as_float(r.q[i].y);
    v[4 * i + 2] = __uint_as_float(r.q[i].z);
    v[4 * i + 3] = __uint_as_float(r.q[i].w);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
// One rounding to the element type (to nearest, ties to even).
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16_2(pk2(v[0], v[1])), pack_bf16_2(pk2(v[2], v[3])),
                                            pack_bf16_2(pk2(v[4], v[5])), pack_bf16_2(pk2(v[6], v[7])));
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A kernel's dynamic shared memory, asked for once a device: a bit each in a word that belongs to the kernel.
inline bool make_room(std::atomic<unsigned long long>& asked, const void* kern, int bytes) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (device & 63);
  if (asked.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  asked.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// A kernel launched with `launch_after` may begin before the kernel ahead of it in the stream has ended: it calls
// `wait_for_previous` before it touches memory, and the kernel ahead calls `let_next_start` once its blocks need no
// more of the machine than they hold.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T>
struct Same {
  using type = T;  // the kernel alone decides the argument types
};
template <typename... A>
inline cudaError_t launch_after(void (*kern)(A...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                typename Same<A>::type... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace pd
