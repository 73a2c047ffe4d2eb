// mk_rotate_append: what stands between the QKV projection and attention in a serving step.
//
//   q'[t, h] = rope(norm(q[t, h]))          k'[t, h] = rope(norm(k[t, h])) -> k_cache[slot t, h]        v[t, h] -> v_cache[slot t, h]
//   norm(x) = w x / sqrt(mean(x^2) + eps)   rope(x)[i] = x[i] cos[i] - x[i + 64] sin[i],  rope(x)[i + 64] = x[i + 64] cos[i + 64] + x[i] sin[i + 64]
//
// in fp32 from the inputs to the one rounding at the end.  Every row of a head is read once and written once: bound by HBM
// (2 x 256 bytes a row) from a few hundred tokens on, by the launch below.  Eight lanes hold a row, each 8 elements of its
// lower half and the 8 that they turn with, so that the loads are 16 bytes wide, the norm is three shuffles and the rotation none.
#include "mk_serving.cuh"

namespace mk_serving {
namespace {

constexpr int kRowLanes = 8;
constexpr int kRotThreads = 256;

template <typename T, bool WIDE> __device__ __forceinline__ void load8(const T* p, float* f) {
  if constexpr (WIDE && sizeof(T) == 2) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = unpack2<T>(w[i]);
      f[2 * i] = d.x;
      f[2 * i + 1] = d.y;
    }
  } else if constexpr (WIDE) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float(p[i]);
  }
}
template <typename T, bool WIDE> __device__ __forceinline__ void store8(T* p, const float* f) {
  if constexpr (WIDE) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(f[i]);
  }
}

// T: rows and caches, A: rotary tables; WIDE: every row starts at a multiple of 16 bytes
template <typename T, typename A, bool WIDE>
__global__ void __launch_bounds__(kRotThreads) rotate_append_kernel(const __grid_constant__ mk_rotate_append_args a) {
  const int heads = a.q_heads + 2 * a.kv_heads;
  const long long row = ((long long)blockIdx.x * kRotThreads + threadIdx.x) / kRowLanes;
  const int l = threadIdx.x % kRowLanes;
  const bool in = row < (long long)a.tokens * heads;  // the norm's shuffles take whole warps
  const int t = in ? (int)(row / heads) : 0, h = in ? (int)(row - (long long)t * heads) : 0;
  const long long slot = in ? a.slots[t] : -1;
  const int pos = in ? a.positions[t] : 0;
  const bool live = slot >= 0 && slot < (long long)a.pages * a.page_size && pos >= 0 && pos < a.table_rows;
  const int kind = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;  // q, k, v
  const int head = kind == 0 ? h : kind == 1 ? h - a.q_heads : h - a.q_heads - a.kv_heads;
  const T* src = kind == 0 ? (const T*)a.q + t * a.q_stride[0] + head * a.q_stride[1]
               : kind == 1 ? (const T*)a.k + t * a.k_stride[0] + head * a.k_stride[1]
                           : (const T*)a.v + t * a.v_stride[0] + head * a.v_stride[1];
  float lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.f;
  if (live) {
    load8<T, WIDE>(src + 8 * l, lo);
    load8<T, WIDE>(src + 64 + 8 * l, hi);
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq += lo[i] * lo[i] + hi[i] * hi[i];
#pragma unroll
  for (int o = 1; o < kRowLanes; o <<= 1) sq += __shfl_xor_sync(kAll, sq, o);  // (by whole warps: rows of v and rows without a slot too)
  if (!live) return;
  if (kind < 2) {
    const T* norm = (const T*)(kind == 0 ? a.q_norm : a.k_norm);
    float c[8], s[8];
    if (norm) {
      const float scale = rsqrtf(sq * (1.f / kHeadDim) + a.eps);
      load8<T, WIDE>(norm + 8 * l, c);
      load8<T, WIDE>(norm + 64 + 8 * l, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] *= scale * c[i];
        hi[i] *= scale * s[i];
      }
    }
    const A* cs = (const A*)a.cos + pos * a.table_stride[0];
    const A* sn = (const A*)a.sin + pos * a.table_stride[1];
    float x[8];
    load8<A, WIDE>(cs + 8 * l, c);
    load8<A, WIDE>(sn + 8 * l, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = lo[i] * c[i] - hi[i] * s[i];
    load8<A, WIDE>(cs + 64 + 8 * l, c);
    load8<A, WIDE>(sn + 64 + 8 * l, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      hi[i] = hi[i] * c[i] + lo[i] * s[i];
      lo[i] = x[i];
    }
  }
  const long long pg = slot / a.page_size, in_page = slot - pg * a.page_size;
  T* dst = kind == 0 ? (T*)a.out + t * a.out_stride[0] + head * a.out_stride[1]
         : kind == 1 ? (T*)a.k_cache + pg * a.k_cache_stride[0] + in_page * a.k_cache_stride[1] + head * a.k_cache_stride[2]
                     : (T*)a.v_cache + pg * a.v_cache_stride[0] + in_page * a.v_cache_stride[1] + head * a.v_cache_stride[2];
  store8<T, WIDE>(dst + 8 * l, lo);
  store8<T, WIDE>(dst + 64 + 8 * l, hi);
}

template <typename T, typename A> int launch(const mk_rotate_append_args& a, bool wide, cudaStream_t s) {
  const long long rows = (long long)a.tokens * (a.q_heads + 2 * a.kv_heads), per = kRotThreads / kRowLanes;
  const unsigned grid = (unsigned)((rows + per - 1) / per);
  if (wide) rotate_append_kernel<T, A, true><<<grid, kRotThreads, 0, s>>>(a);
  else rotate_append_kernel<T, A, false><<<grid, kRotThreads, 0, s>>>(a);
  return launched("rotate_append");
}

}  // namespace
}  // namespace mk_serving

extern "C" int mk_rotate_append(const mk_rotate_append_args* args, void* stream) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "rotate_append: null arguments");
  const mk_rotate_append_args& a = *args;
  if (!a.q || !a.k || !a.v || !a.cos || !a.sin || !a.positions || !a.slots || !a.k_cache || !a.v_cache || !a.out)
    return fail(MK_E_INVALID, "rotate_append: null pointer");
  if (a.dtype != MK_BF16 && a.dtype != MK_F16) return fail(MK_E_INVALID, "rotate_append: rows and caches are bf16 or fp16");
  if (a.table_dtype != a.dtype && a.table_dtype != MK_F32) return fail(MK_E_INVALID, "rotate_append: cos and sin have the rows' type or fp32");
  if (a.tokens < 0 || a.q_heads < 1 || a.kv_heads < 1 || a.page_size < 1 || a.pages < 1 || a.table_rows < 1)
    return fail(MK_E_INVALID, "rotate_append: sizes must be positive");
  if ((long long)a.tokens * (a.q_heads + 2 * a.kv_heads) > (1ll << 36)) return fail(MK_E_TOO_LARGE, "rotate_append: too many rows");
  if (a.tokens == 0) return 0;
  bool wide = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos) && aligned16(a.sin) && aligned16(a.k_cache) &&
              aligned16(a.v_cache) && aligned16(a.out) && aligned16(a.q_norm) && aligned16(a.k_norm);
  for (int i = 0; i < 2; ++i) wide = wide && !((a.q_stride[i] | a.k_stride[i] | a.v_stride[i] | a.out_stride[i] | a.table_stride[i]) & 7);
  for (int i = 0; i < 3; ++i) wide = wide && !((a.k_cache_stride[i] | a.v_cache_stride[i]) & 7);
  const cudaStream_t s = (cudaStream_t)stream;
  const bool f32 = a.table_dtype == MK_F32;
  if (a.dtype == MK_BF16) return f32 ? launch<__nv_bfloat16, float>(a, wide, s) : launch<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
  return f32 ? launch<__half, float>(a, wide, s) : launch<__half, __half>(a, wide, s);
}
