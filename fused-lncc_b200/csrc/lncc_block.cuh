// Shared by the token-block operators (layer_norm.cu, gated_scan.cu, gated_ffn.cu): element types, 16-byte vectors,
// warp sums, argument checks, and the host side of the bounds-checked build. Every type is loaded into fp32 registers,
// all arithmetic is fp32, and a value is rounded to its type once, on the store.
#pragma once

#include "lncc.h"
#include "lncc_check.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace lncc {
namespace blk {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// V elements moved as one access (V * sizeof(T) a power of two up to 16 bytes, address aligned to it)
template <typename T, int V> struct alignas(sizeof(T) * V) Vec {
  T e[V];
};
template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; i++) out[i] = to_f(v.e[i]);
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; i++) v.e[i] = from_f<T>(in[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// two fp32 numbers a packed instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 A, B;\n\tmov.b64 A, {%2, %3};\n\tmov.b64 B, {%4, %5};\n\tadd.rn.f32x2 A, A, B;\n\tmov.b64 {%0, %1}, A;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 A, B;\n\tmov.b64 A, {%2, %3};\n\tmov.b64 B, {%4, %5};\n\tmul.rn.f32x2 A, A, B;\n\tmov.b64 {%0, %1}, A;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 A, B, C;\n\tmov.b64 A, {%2, %3};\n\tmov.b64 B, {%4, %5};\n\tmov.b64 C, {%6, %7};\n\tfma.rn.f32x2 A, A, B, C;\n\t"
      "mov.b64 {%0, %1}, A;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

inline bool valid_dtype(int dtype) { return dtype == LNCC_F32 || dtype == LNCC_BF16 || dtype == LNCC_F16; }
inline int elem_size(int dtype) { return dtype == LNCC_F32 ? 4 : 2; }
inline bool aligned(const void* p, uintptr_t n) { return uintptr_t(p) % n == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// SMs of the current device (148 where it cannot be asked), read once per device.
inline int sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = counts[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// The devices that were asked for a kernel's shared memory, marked by any thread. Asking twice does no harm.
struct Asked {
  std::atomic<uint64_t> devices{0};
  bool has(int dev) const { return dev < 64 && devices.load(std::memory_order_relaxed) >> dev & 1; }
  void mark(int dev) {
    if (dev < 64) devices.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
};

// In the bounds-checked build: zero this file's violation counter before a call's launches, and turn a count into
// LNCC_ERR_CHECK after them. In the normal build both cost nothing. Static: each source file has a counter of its own, and one
// function for all of them would read one file's.
static inline int check_begin() {
#ifdef LNCC_CHECKED
  const unsigned long long z = 0;
  return cudaMemcpyToSymbol(g_check_violations, &z, sizeof(z)) == cudaSuccess ? LNCC_OK : LNCC_ERR_CUDA;
#else
  return LNCC_OK;
#endif
}
static inline int check_end(cudaStream_t stream) {
  if (cudaGetLastError() != cudaSuccess) return LNCC_ERR_LAUNCH;
#ifdef LNCC_CHECKED
  unsigned long long n = 0;
  if (cudaStreamSynchronize(stream) != cudaSuccess ||
      cudaMemcpyFromSymbol(&n, g_check_violations, sizeof(n)) != cudaSuccess)
    return LNCC_ERR_CUDA;
  return n ? LNCC_ERR_CHECK : LNCC_OK;
#else
  (void)stream;
  return LNCC_OK;
#endif
}

}  // namespace blk
}  // namespace lncc
