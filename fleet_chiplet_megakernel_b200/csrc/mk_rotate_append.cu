// mk_rotate_append: what stands between the QKV projection and attention in a serving step.
//
//   q'[t, h] = rope(norm(q[t, h]))          k'[t, h] = rope(norm(k[t, h])) -> k_cache[slot t, h]        v[t, h] -> v_cache[slot t, h]
//   norm(x) = w x / sqrt(mean(x^2) + eps)   rope(x)[i] = x[i] cos[i] - x[i + 64] sin[i],  rope(x)[i + 64] = x[i + 64] cos[i + 64] + x[i] sin[i + 64]
//
// in fp32 from the inputs to the one rounding at the end.  Every row of a head is read once and written once: bound by HBM
// (2 x 256 bytes a row) from a few hundred tokens on, by the launch below.  Eight lanes hold a row, each 8 elements of its
// lower half and the 8 that they turn with, so that the loads are 16 bytes wide, the norm is three shuffles and the rotation none.
// 4000 tokens of 32 q and 8 kv heads: 24 us, 4.1 TB/s; a copy of as many bytes takes 16.  What lacks is loads in flight: four rows a
// lane group are 127 registers, 16 warps an SM (two or three rows, with more warps, and six or eight are slower).
#include "mk_serving.cuh"

namespace mk_serving {
namespace {

constexpr int kRowLanes = 8;
constexpr int kRotThreads = 128;
constexpr int kRows = 4;  // of a lane on their way together

// Eight elements as they lie in memory, so that several rows can be on their way in few registers.
template <typename T> struct Raw {
  uint4 w[sizeof(T) / 2];
  template <bool WIDE> __device__ __forceinline__ void load(const T* p) {
    if constexpr (WIDE) {
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) w[k] = reinterpret_cast<const uint4*>(p)[k];
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(uint64_t (&f)[4]) const {  // as pairs of fp32
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
      const uint32_t v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          const float2 d = unpack2<T>(v[i]);
          f[i] = pair(d.x, d.y);
        } else if (i < 2) {
          f[2 * k + i] = pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        }
      }
    }
  }
  template <bool WIDE> __device__ __forceinline__ void store(T* p) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(p)[k] = w[k];
    } else {
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = e[i];
    }
  }
  __device__ __forceinline__ void put(const uint64_t (&f)[4]) {  // (16-bit types)
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = unpair(f[i]);
      v[i] = pack2<T>(d.x, d.y);
    }
    w[0] = make_uint4(v[0], v[1], v[2], v[3]);
  }
};

// T: rows and caches, A: rotary tables; WIDE: every row starts at a multiple of 16 bytes; ROWS heads of a token, next to each other, to eight
// lanes: the token's slot, position and rotary row are looked up once for them, and their loads are on their way together.
template <typename T, typename A, bool WIDE, int ROWS>
__global__ void __launch_bounds__(kRotThreads, 4) rotate_append_kernel(const __grid_constant__ mk_rotate_append_args a) {
  const int heads = a.q_heads + 2 * a.kv_heads, l = threadIdx.x % kRowLanes, groups = (heads + ROWS - 1) / ROWS;
  const unsigned group = (blockIdx.x * kRotThreads + threadIdx.x) / kRowLanes;  // (fewer than 2^31: the launch sees to it)
  const int t = (int)(group / (unsigned)groups), h0 = (int)(group - (unsigned)t * (unsigned)groups) * ROWS;
  if (t >= a.tokens) return;  // (eight lanes together, and so below: the norm's shuffles are theirs alone)
  const unsigned lanes = 0xffu << (threadIdx.x & 24);
  const long long slot = __ldg(a.slots + t);
  const int pos = __ldg(a.positions + t);
  if (slot < 0 || slot >= (long long)a.pages * a.page_size || pos < 0 || pos >= a.table_rows) return;
  auto kind_of = [&](int h) { return h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2; };  // q, k, v
  auto head_of = [&](int h, int kind) { return kind == 0 ? h : kind == 1 ? h - a.q_heads : h - a.q_heads - a.kv_heads; };
  Raw<T> lo[ROWS], hi[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int h = h0 + j, kind = kind_of(h), head = head_of(h, kind);
    if (h >= heads) break;
    const T* src = 8 * l + (kind == 0 ? (const T*)a.q + t * a.q_stride[0] + head * a.q_stride[1]
                          : kind == 1 ? (const T*)a.k + t * a.k_stride[0] + head * a.k_stride[1]
                                      : (const T*)a.v + t * a.v_stride[0] + head * a.v_stride[1]);
    lo[j].template load<WIDE>(src);
    hi[j].template load<WIDE>(src + 64);
  }
  long long pg, in_page;
  if ((unsigned long long)slot >> 31) {
    pg = slot / a.page_size;
    in_page = slot - pg * a.page_size;
  } else {
    pg = (unsigned)slot / (unsigned)a.page_size;
    in_page = (unsigned)slot - (unsigned)pg * (unsigned)a.page_size;
  }
  // the lane's 8 + 8 elements of the rotary row (rows of v need none)
  uint64_t c0[4], c1[4], s0[4], s1[4];
  if (kind_of(h0) < 2) {
    const A* cs = (const A*)a.cos + pos * a.table_stride[0] + 8 * l;
    const A* sn = (const A*)a.sin + pos * a.table_stride[1] + 8 * l;
    Raw<A> x0, x1, x2, x3;
    x0.template load<WIDE>(cs);
    x1.template load<WIDE>(cs + 64);
    x2.template load<WIDE>(sn);
    x3.template load<WIDE>(sn + 64);
    x0.get(c0);
    x1.get(c1);
    x2.get(s0);
    x3.get(s1);
#pragma unroll
    for (int i = 0; i < 4; ++i) s0[i] ^= 0x8000000080000000ull;  // (its products are taken away)
  }
  uint64_t w0[4], w1[4];
  int normed = -1;  // kind whose weights are in w0, w1
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int h = h0 + j, kind = kind_of(h), head = head_of(h, kind);
    if (h >= heads) break;
    if (kind < 2) {
      uint64_t x[4], y[4];
      lo[j].get(x);
      hi[j].get(y);
      if (const T* norm = (const T*)(kind == 0 ? a.q_norm : a.k_norm)) {
        if (normed != kind) {
          Raw<T> r0, r1;
          r0.template load<WIDE>(norm + 8 * l);
          r1.template load<WIDE>(norm + 64 + 8 * l);
          r0.get(w0);
          r1.get(w1);
          normed = kind;
        }
        uint64_t sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fma2(y[i], y[i], fma2(x[i], x[i], sum));
        const float2 both = unpair(sum);
        float sq = both.x + both.y;
#pragma unroll
        for (int o = 1; o < kRowLanes; o <<= 1) sq += __shfl_xor_sync(lanes, sq, o);
        const float f = rsqrtf(sq * (1.f / kHeadDim) + a.eps);
        const uint64_t scale = pair(f, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = mul2(mul2(x[i], scale), w0[i]);
          y[i] = mul2(mul2(y[i], scale), w1[i]);
        }
      }
      uint64_t z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[i] = fma2(y[i], s0[i], mul2(x[i], c0[i]));
        y[i] = fma2(x[i], s1[i], mul2(y[i], c1[i]));
      }
      lo[j].put(z);
      hi[j].put(y);
    }
    T* dst = 8 * l + (kind == 0 ? (T*)a.out + t * a.out_stride[0] + head * a.out_stride[1]
                    : kind == 1 ? (T*)a.k_cache + pg * a.k_cache_stride[0] + in_page * a.k_cache_stride[1] + head * a.k_cache_stride[2]
                                : (T*)a.v_cache + pg * a.v_cache_stride[0] + in_page * a.v_cache_stride[1] + head * a.v_cache_stride[2]);
    lo[j].template store<WIDE>(dst);
    hi[j].template store<WIDE>(dst + 64);
  }
}

template <typename T, typename A> int launch(const mk_rotate_append_args& a, bool wide, cudaStream_t s) {
  const int heads = a.q_heads + 2 * a.kv_heads;
  const long long per = kRotThreads / kRowLanes;
  // One row to eight lanes, or four that are on their way together where there are rows for all SMs (48 heads a token; 16 tokens 2.3 us
  // against 3.5, 250: 3.1 and 3.8, 500: 5.1 and 4.4, 4000: 31 and 24).
  const bool many = (long long)a.tokens * heads > 8 * per * sm_count();
  const long long grid = ((long long)a.tokens * (many ? (heads + kRows - 1) / kRows : heads) + per - 1) / per;
  if (!wide) rotate_append_kernel<T, A, false, 1><<<(unsigned)(((long long)a.tokens * heads + per - 1) / per), kRotThreads, 0, s>>>(a);
  else if (many) rotate_append_kernel<T, A, true, kRows><<<(unsigned)grid, kRotThreads, 0, s>>>(a);
  else rotate_append_kernel<T, A, true, 1><<<(unsigned)grid, kRotThreads, 0, s>>>(a);
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
  if ((long long)a.tokens * ((long long)a.q_heads + 2ll * a.kv_heads) > 0x7fffffff / kRowLanes) return fail(MK_E_TOO_LARGE, "rotate_append: too many rows");
  if (a.tokens == 0) return 0;
  if (a.k_cache == a.v_cache) return fail(MK_E_INVALID, "rotate_append: k_cache and v_cache share memory");
  bool wide = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos) && aligned16(a.sin) && aligned16(a.k_cache) &&
              aligned16(a.v_cache) && aligned16(a.out) && aligned16(a.q_norm) && aligned16(a.k_norm);
  for (int i = 0; i < 2; ++i) wide = wide && !((a.q_stride[i] | a.k_stride[i] | a.v_stride[i] | a.out_stride[i] | a.table_stride[i]) & 7);
  for (int i = 0; i < 3; ++i) wide = wide && !((a.k_cache_stride[i] | a.v_cache_stride[i]) & 7);
  const bool f32 = a.table_dtype == MK_F32;
  // Rows are written while others are read, so what is written may share memory with nothing else of the call.  (out may be q: the lanes
  // that write a row have read it, and no others do.)
  const bool in_place = a.out == a.q && (a.tokens == 1 || a.out_stride[0] == a.q_stride[0]) && (a.q_heads == 1 || a.out_stride[1] == a.q_stride[1]);
  const long long row = 2 * kHeadDim, entry = f32 ? 4 : 2;
  auto rows = [&](const char* name, const void* at, int heads, const int64_t* stride) -> Memory {
    return {name, at, row, 2, {a.tokens, heads}, {2 * stride[0], 2 * stride[1]}};
  };
  auto cache = [&](const char* name, const void* at, const int64_t* stride) -> Memory {
    return {name, at, row, 3, {a.pages, a.page_size, a.kv_heads}, {2 * stride[0], 2 * stride[1], 2 * stride[2]}};
  };
  auto table = [&](const char* name, const void* at, int64_t stride) -> Memory { return {name, at, entry * kHeadDim, 1, {a.table_rows}, {entry * stride}}; };
  const Memory used[] = {cache("k_cache", a.k_cache, a.k_cache_stride), cache("v_cache", a.v_cache, a.v_cache_stride), rows("out", a.out, a.q_heads, a.out_stride),
                         rows("k", a.k, a.kv_heads, a.k_stride), rows("v", a.v, a.kv_heads, a.v_stride), table("cos", a.cos, a.table_stride[0]),
                         table("sin", a.sin, a.table_stride[1]), list_of("positions", a.positions, a.tokens, 4), list_of("slots", a.slots, a.tokens, 8),
                         list_of("q_norm", a.q_norm, kHeadDim, 2), list_of("k_norm", a.k_norm, kHeadDim, 2), rows("q", in_place ? nullptr : a.q, a.q_heads, a.q_stride)};
  if (int rc = refuse_misaligned("rotate_append", {{"q", a.q, 2}, {"k", a.k, 2}, {"v", a.v, 2}, {"cos", a.cos, (int)entry}, {"sin", a.sin, (int)entry}, {"positions", a.positions, 4},
                                                   {"slots", a.slots, 8}, {"k_cache", a.k_cache, 2}, {"v_cache", a.v_cache, 2}, {"q_norm", a.q_norm, 2}, {"k_norm", a.k_norm, 2},
                                                   {"out", a.out, 2}}))
    return rc;
  if (int rc = refuse_shared("rotate_append", used, 3, sizeof used / sizeof *used)) return rc;
  const cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == MK_BF16) return f32 ? launch<__nv_bfloat16, float>(a, wide, s) : launch<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
  return f32 ? launch<__half, float>(a, wide, s) : launch<__half, __half>(a, wide, s);
}
