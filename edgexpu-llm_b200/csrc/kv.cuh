// kv.cuh -- the paged cache of edgexpu_cuda_kv_cache as kernels see it, and its checks (kvcache.cu,
// kvattn.cu).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/edgexpu_cuda.h"
#include "common.cuh"

namespace ex {

struct KvView {
  uint16_t* k;
  uint16_t* v;
  long long layer_stride, page_stride;  // elements
  int n_layers, n_pages, ps_shift, n_kv, hd, n_seqs, max_pages;
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  int32_t* work;
  uint32_t* status;
};

// The descriptor as a view; 0 with a message naming `who` when it is not a cache.
int kv_view(const edgexpu_cuda_kv_cache* c, const char* who, KvView* view);

__device__ __forceinline__ int kv_pages_of(const KvView& c, int len) {  // len >= 0
  return (len >> c.ps_shift) + ((len & ((1 << c.ps_shift) - 1)) != 0 ? 1 : 0);
}

// 16 bits of type T from fp32, to nearest even.
template <typename T>
__device__ __forceinline__ uint16_t round16(float x);
template <>
__device__ __forceinline__ uint16_t round16<__half>(float x) {
  return __half_as_ushort(__float2half_rn(x));
}
template <>
__device__ __forceinline__ uint16_t round16<__nv_bfloat16>(float x) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack16<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

template <typename T>
__host__ __device__ constexpr uint32_t exponent16();  // the bits of the exponent, all ones in infinities and NaN
template <>
__host__ __device__ constexpr uint32_t exponent16<__half>() {
  return 0x7C00u;
}
template <>
__host__ __device__ constexpr uint32_t exponent16<__nv_bfloat16>() {
  return 0x7F80u;
}

// Two weights >= 0 as a coarse number of the type each and the rest, which is never below 0: the coarse one is
// rounded from a little less than the weight.  Together they hold it to 2^-15 (bf16), or to 2^-20 or, below 2^-5,
// 2^-25 (f16).  Down to 2^-115 (bf16) or 2^-14 (f16: with P_SHIFT 2^-24 of the row's largest) both are above 0, so
// that their products with an infinity have its sign; a smaller weight may make NaN of it.
template <typename T>
__device__ __forceinline__ void split16(float p0, float p1, uint32_t& coarse, uint32_t& rest) {
  constexpr float LESS = exponent16<T>() == 0x7C00u ? 1.0f - 1.0f / 1024 : 1.0f - 1.0f / 256;
  coarse = pack16<T>(p0 * LESS, p1 * LESS);
  const float2 c = unpack16<T>(coarse);
  rest = pack16<T>(p0 - c.x, p1 - c.y);
}

// Let the next grid of the stream launch, and wait until the one before has completed.
__device__ __forceinline__ void pdl_enter_grid() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The same where the next grid runs beside this one: what came before is complete first, so that the next
// grid need not wait for it.  That grid, in turn, waits for this one before it ends.
__device__ __forceinline__ void pdl_enter_pair() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename F>
cudaError_t allow_smem(F* kern, size_t bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace ex
