// Attention of the new tokens of a batch over a paged K/V cache: what its kernels share.
//
// Request r has the n new rows qo_indptr[r] <= t < qo_indptr[r + 1] and, with its new tokens, `len` positions: its pages are
// kv_indices[kv_indptr[r] .. kv_indptr[r + 1]), the last of them filled up to last_page_len[r].  Row i of the n sits at
// position p = len - n + i and sees position j where
//     0 <= j <= p   and   (no window, or j > p - window, or j < sinks).
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(scale q.k_j); a row that sees nothing is zero, its lse minus infinity.
// What the index arrays say is held against the sizes of the tensors before it is used: a page that does not exist reads as zeros.
#ifndef MK_CHUNK_ATTENTION_CUH
#define MK_CHUNK_ATTENTION_CUH

#include "mk_serving.cuh"

namespace mk_serving {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Weights enter their product with V in 16 bits.  bf16 holds them all with the same relative rounding.  fp16 has fewer and fewer bits below 2^-14
// and nothing below 2^-25, while a row of some ten thousand positions can consist of such weights; so in fp16 they are carried 2^kLift
// times as large, up to 2^15 of the 2^16 that the type holds, and the sums divided by it at the end (both exactly).

// Pieces of a group that are to be joined: the warp, or CTA, with the last one (-1: none), and the group's rows.
struct MergeRecord {
  int last;
  int kv_head, row0, rows, first_token;
};

struct AttnParams {
  mk_chunk_attention_args a;
  int per_kv;           // q heads of a kv head
  bool tile_in_page;    // a page holds whole tiles of the row kernel
  int page_shift;       // log2 of the page size, -1 if it is no power of two
  float scale_log2;     // scale * log2(e): scores and maxima are kept in base 2
  int few_rows;         // requests with at most so many rows (new tokens x q heads of a kv head) are the row kernel's, others the tile kernel's
  int min_tiles;        // a warp's share of the row kernel is no shorter
  int row_ctas;         // of the row kernel
  MergeRecord* merges;  // row kernel -> merge: of the group that a CTA begins and does not end
  float* joined;        // its pieces, two a CTA (of a group from the CTA before, of one that goes on in the next)
  int splits;           // of the tile kernel: pieces of every row's positions
  float* tile_partial;  // [splits][tokens][q heads][130]
};

struct Request {
  int q0, n, len, kv0;  // first row, rows, positions, first entry of the page index
};
__device__ __forceinline__ Request request_of(const mk_chunk_attention_args& a, int r) {
  Request q;
  const int q0 = __ldg(a.qo_indptr + r), q1 = __ldg(a.qo_indptr + r + 1), k0 = __ldg(a.kv_indptr + r), k1 = __ldg(a.kv_indptr + r + 1), last = __ldg(a.last_page_len + r);
  q.q0 = min(max(q0, 0), a.tokens);
  q.n = min(max(q1, q.q0), a.tokens) - q.q0;
  q.kv0 = min(max(k0, 0), a.num_indices);
  const int pages = min(max(k1, q.kv0), a.num_indices) - q.kv0;
  q.len = pages > 0 ? (int)min((long long)(pages - 1) * a.page_size + min(max(last, 0), a.page_size), 0x7fffff00ll) : 0;
  return q;
}
__device__ __forceinline__ bool sees(const mk_chunk_attention_args& a, int j, int p) {
  return j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
}
// Page and row in the page of a position; the page is -1 where it does not exist.
__device__ __forceinline__ void locate(const AttnParams& p, const Request& q, int pos, int* page, int* in_page) {
  const int k = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.a.page_size;
  *in_page = pos - k * p.a.page_size;
  const int pg = pos < q.len ? __ldg(p.a.kv_indices + q.kv0 + k) : -1;
  *page = (unsigned)pg < (unsigned)p.a.pages ? pg : -1;
}

// The tiles of `TILE` positions that rows at positions p0 <= p <= p1 see: `sink` tiles from position 0, the others from `start` on.
template <int TILE> struct Span {
  int sink, start, count;
  __device__ __forceinline__ Span(const mk_chunk_attention_args& a, int p0, int p1) {
    if (p1 < 0) {
      sink = start = count = 0;
      return;
    }
    // (64 bits: the window may be as long as an int)
    const long long w0 = a.window == 0 ? 0 : (long long)max(p0, 0) - a.window + 1;
    start = w0 > 0 ? (int)(w0 / TILE) * TILE : 0;
    sink = min((int)(((long long)a.sinks + TILE - 1) / TILE), start / TILE);
    if (a.window == 0) sink = 0;
    count = sink + (p1 - start) / TILE + 1;
  }
  __device__ __forceinline__ int position(int k) const { return k < sink ? k * TILE : start + (k - sink) * TILE; }
};

// One row over the tiles k0 <= k < k1 of a span, a position at a time and only those that the row sees, by a warp: lane l has dims
// 4 l .. 4 l + 3.  For pieces whose products were not finite: a product with weight 0 is not 0 there, so a value that is not finite
// would reach rows that do not see it.
template <typename T, int TILE>
__device__ __noinline__ void exact_row(const AttnParams& p, const Request& q, const Span<TILE>& span, int k0, int k1, int at, long long tok, int head, int kv_head,
                                       float (&o)[4], float& m, float& l) {
  const mk_chunk_attention_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const T* qr = (const T*)a.q + tok * a.q_stride[0] + head * a.q_stride[1] + 4 * lane;
  float x[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    x[d] = to_float(qr[d]);
    o[d] = 0.f;
  }
  m = -INFINITY;
  l = 0.f;
  for (int i = k0; i < min(k1, span.count); ++i)
    for (int j = span.position(i); j < span.position(i) + TILE; ++j) {
      if (!sees(a, j, at)) continue;
      int page, in;
      locate(p, q, j, &page, &in);
      float s = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      if (page >= 0) {
        const T* kr = (const T*)a.k_cache + (long long)page * a.k_cache_stride[0] + (long long)in * a.k_cache_stride[1] + kv_head * a.k_cache_stride[2] + 4 * lane;
        const T* vr = (const T*)a.v_cache + (long long)page * a.v_cache_stride[0] + (long long)in * a.v_cache_stride[1] + kv_head * a.v_cache_stride[2] + 4 * lane;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          s += x[d] * to_float(kr[d]);
          v[d] = to_float(vr[d]);
        }
      }
#pragma unroll
      for (int e = 16; e > 0; e >>= 1) s += __shfl_xor_sync(kAll, s, e);
      s *= p.scale_log2;
      if (s == -INFINITY) continue;
      const float mn = s > m ? s : m;  // (a NaN score leaves the maximum and enters the weight)
      const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - (mn == -INFINITY ? 0.f : mn));
      l = l * alpha + w;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = o[d] * alpha + w * v[d];
      m = mn;
    }
}

// A word of pinned host memory in which a kernel says that a wait has run out (null: there is none to be had): bit 63, which of the tile
// kernel's barriers in bits 32 on, the CTA below.  One a process, whatever the device.
unsigned long long* lost_word();
// Taken out of it and made an error of: 0, or MK_E_DEVICE with its text.
int report_lost_wait();

// mk_chunk_attention_tiles.cu: whether the tile kernel takes such tensors at all, and its launch
bool tiles_take(const mk_chunk_attention_args& a);
int launch_tile_attention(const AttnParams& p, cudaStream_t s);

}  // namespace mk_serving

#endif
