// What the stand-alone kernels of a serving step share: conversions, row geometry of the paged batch, error texts.
#ifndef MK_SERVING_CUH
#define MK_SERVING_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <initializer_list>

#include "../../include/b200mk.h"

namespace mk_serving {

constexpr int kHeadDim = 128;
constexpr unsigned kAll = 0xffffffffu;

// text of the last refused or failed call of this thread (mk_op_error)
char* error_text();
constexpr int kErrorBytes = 512;
inline int fail(int code, const char* fmt, ...) noexcept {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(error_text(), kErrorBytes, fmt, ap);
  va_end(ap);
  return code;
}
inline int launched(const char* what) noexcept {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(MK_E_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
}
// Lets a kernel have so much dynamic shared memory on the current device, once (a call of the driver takes a microsecond).
template <auto kernel> cudaError_t allow_shared(int bytes) noexcept {
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}
// Multiprocessors of the current device (the value of a device does not change).
int sm_count();

// What a call reads or writes of one tensor: entries of `reach` bytes, at `at` plus multiples of the strides (bytes), size[i] of each.
struct Memory {
  const char* name;
  const void* at;
  long long reach;
  int dims;
  long long size[3], stride[3];
};
inline Memory list_of(const char* name, const void* at, long long n, int bytes) { return {name, at, n * bytes, 0, {}, {}}; }
// Whether two of them have a byte in common.  Exactly, where the strides nest as those of slices and permutations of a tensor do; where
// the search would take long, true.
bool share_memory(const Memory& a, const Memory& b);
// The first pair of the `n` that shares memory, the first `written` of them with any other: an error that names them (0: none).
int refuse_shared(const char* what, const Memory* m, int written, int n);

// An address that is no multiple of its element's size: an error that names it (0: none).  torch's own tensors have none, an address from elsewhere may.
struct Address {
  const char* name;
  const void* at;
  int bytes;
};
int refuse_misaligned(const char* what, std::initializer_list<Address> all);

inline bool aligned16(const void* p) { return (((uintptr_t)p) & 15) == 0; }

// ---- 16-bit types
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
// two floats in one word, a in the low half
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// two fp32 values in a register pair
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// First of the entries 0 <= i < n with first(i + 1) > x, where first() does not fall; one thread.
template <typename F> __device__ __forceinline__ int find_owner(int n, long long x, const F& first) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (first(mid + 1) > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}
// The same by a converged warp: 32 probes at a time, so that a table in global memory costs a round trip per factor of 32.
template <typename F> __device__ __forceinline__ int find_owner_warp(int n, long long x, const F& first) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int at = min(lo + (lane + 1) * step, hi) - 1;  // last entry of this lane's share
    const unsigned over = __ballot_sync(kAll, first(at + 1) > x);
    const int k = over ? __ffs(over) - 1 : 31;
    const int l = min(lo + k * step, n - 1);
    hi = min(lo + (k + 1) * step, hi);
    lo = l;
    if (hi <= lo) return lo;
  }
  return lo;
}

}  // namespace mk_serving

#endif
