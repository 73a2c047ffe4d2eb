// mk_plan_step: page allocation, block tables, index pointers and slot map of a serving step, from the requests' lengths.
//
// With held(r) = ceil(length / page) and need(r) = ceil((length + new) / page) - held(r), everything that the step needs is a
// prefix sum over the requests (pages taken from the ring, pages given back, token rows, pages in the index) and a lookup in
// it.  The sums are short (a few hundred to a few thousand requests) and the lookups many (a page each, a token each), so
// every CTA works out all the sums for itself in shared memory and then takes its share of the lookups: one launch, no
// CTA waits for another, no atomics.  What is read and written is about 8 bytes a page and 12 a token; bound by latency:
// 8 requests 5 us, 512 of up to 8000 tokens on pages of 16, with prompt chunks among them, 7 us.
#include "mk_serving.cuh"

namespace mk_serving {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;

struct PlanParams {
  mk_step_plan_args a;
  int shift;  // log2 of the page size, -1 if it is no power of two
};

// Inclusive sums of N values over the block, and the block's totals.  One barrier: `turn` alternates between two places for the warps'
// totals, and whoever writes a place again has passed the barrier of the other one since it was read.
template <int N> struct Scan {
  long long (*carry)[N][kPlanWarps];  // [2]
  int turn = 0;
  __device__ __forceinline__ void operator()(long long (&v)[N], long long (&total)[N], int used) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < used; ++k)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(kAll, v[k], o);
        if (lane >= o) v[k] += u;
      }
    if (lane == 31)
#pragma unroll
      for (int k = 0; k < used; ++k) carry[turn][k][warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < used; ++k) {
      long long c = lane < kPlanWarps ? carry[turn][k][lane] : 0;
#pragma unroll
      for (int o = 1; o < kPlanWarps; o <<= 1) {
        const long long u = __shfl_up_sync(kAll, c, o);
        if (lane >= o) c += u;
      }
      total[k] = __shfl_sync(kAll, c, kPlanWarps - 1);
      const long long before = __shfl_sync(kAll, c, warp > 0 ? warp - 1 : 0);
      if (warp > 0) v[k] += before;
    }
    turn ^= 1;
  }
};

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(const __grid_constant__ PlanParams p) {
  const mk_step_plan_args& a = p.a;
  extern __shared__ int table[];  // three tables of R + 1 first entries: token rows, pages of the index, pages given back
  __shared__ long long carry[2][3][kPlanWarps];
  Scan<3> scan{carry};
  const int R = a.requests, page = a.page_size;
  int* tok0 = table;
  int* kv0 = tok0 + R + 1;
  int* need0 = kv0 + R + 1;
  int* back0 = need0 + R + 1;
  const long long head = a.free_range_in[0], tail = a.free_range_in[1];
  const unsigned longest = (unsigned)min((long long)a.table_width * page, 0x7fffffffll);  // what a row of the block table can hold
  auto length_of = [&](int r) { return (int)min((unsigned)max(0, __ldg(a.lengths + r)), longest); };
  auto divided = [&](unsigned n) { return p.shift >= 0 ? n >> p.shift : n / (unsigned)page; };
  auto pages_of = [&](unsigned n) { return n ? (int)min(divided(n - 1) + 1, 0x7fffffffu) : 0; };  // (a length with more is refused)

  // pages that ended requests give back: they count as free in this step already
  long long back = 0, total[3];
  for (int r0 = 0; r0 < R; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    long long v[3] = {r < R && __ldg(a.new_tokens + r) < 0 ? pages_of(length_of(r)) : 0, 0, 0};
    scan(v, total, 1);
    if (r < R) back0[r + 1] = (int)(back + v[0]);
    back += total[0];
  }
  const long long free_pages = tail - head + back;

  long long wanted = 0, rows = 0, kv = 0, taken = 0, tokens = 0;
  for (int r0 = 0; r0 < R; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    const int len = r < R ? length_of(r) : 0, want = r < R ? __ldg(a.new_tokens + r) : 0;
    const int held = pages_of(len), after = pages_of((unsigned)len + (unsigned)max(0, want));
    const bool valid = want > 0 && after <= a.table_width && (unsigned)len + (unsigned)want <= 0x7fffffffu;  // (positions are ints)
    const int need = valid ? after - held : 0;
    long long v[3] = {need, 0, 0};
    scan(v, total, 1);
    const bool fits = valid && (need == 0 || wanted + v[0] <= free_pages);
    wanted += total[0];
    v[0] = fits ? want : 0;
    scan(v, total, 1);
    const int granted = fits && rows + v[0] <= a.max_tokens ? want : 0;
    rows += total[0];
    const int take = granted > 0 ? need : 0;
    // (want < 0: ended.  A request that gets nothing keeps the pages that it has.)
    const int pages = want < 0 ? 0 : held + take;
    v[0] = granted;
    v[1] = take;
    v[2] = pages;
    scan(v, total, 3);
    if (r < R) {
      tok0[r + 1] = (int)(tokens + v[0]);
      need0[r + 1] = (int)(taken + v[1]);
      kv0[r + 1] = (int)(kv + v[2]);
      if (blockIdx.x == 0) {
        a.granted[r] = granted;
        a.qo_indptr[r + 1] = (int)(tokens + v[0]);
        a.kv_indptr[r + 1] = (int)(kv + v[2]);
        a.last_page_len[r] = pages > 0 ? (int)((long long)len + granted - (long long)(pages - 1) * page) : 0;
      }
    }
    tokens += total[0];
    taken += total[1];
    kv += total[2];
  }
  if (threadIdx.x == 0) {
    tok0[0] = kv0[0] = need0[0] = back0[0] = 0;
    if (blockIdx.x == 0) {
      a.qo_indptr[0] = a.kv_indptr[0] = 0;
      a.free_range_out[0] = head + taken;
      a.free_range_out[1] = tail + back;
    }
  }
  __syncthreads();

  const long long ring = a.ring_size;
  const long long head_at = ring > 0 ? ((head % ring) + ring) % ring : 0, tail_at = ring > 0 ? ((tail % ring) + ring) % ring : 0;
  // page i of those that the step takes, ring first; what ended requests give back in this launch comes from their own rows
  auto taken_page = [&](long long i) -> int {
    const long long in_ring = tail - head;
    if (i < in_ring) {
      const long long at = head_at + i;
      return a.free_pages[at < ring ? at : at % ring];
    }
    const int b = (int)(i - in_ring);
    const int r = find_owner(R, b, [&](int k) { return (long long)back0[k]; });
    return a.block_table[(long long)r * a.table_stride + (b - back0[r])];
  };
  auto page_at = [&](int r, int k) -> int {  // page k of request r, held or taken
    const int held = pages_of(length_of(r));
    return k < held ? a.block_table[(long long)r * a.table_stride + k] : taken_page((long long)need0[r] + k - held);
  };

  const long long n_back = ring > 0 ? back : 0;
  const long long all = kv + a.max_tokens + n_back;
  for (long long e = (long long)blockIdx.x * kPlanThreads + threadIdx.x; e < all; e += (long long)gridDim.x * kPlanThreads) {
    if (e < kv) {  // an entry of the page index; a new page enters its request's table as well
      const int r = find_owner(R, e, [&](int k) { return (long long)kv0[k]; });
      const int k = (int)e - kv0[r], held = pages_of(length_of(r));
      const int pg = page_at(r, k);
      if (e < a.max_indices) a.kv_indices[e] = pg;
      if (k >= held) a.block_table[(long long)r * a.table_stride + k] = pg;
    } else if (e < kv + a.max_tokens) {  // a token row: its position and cache slot
      const int t = (int)(e - kv);
      long long slot = -1;
      int pos = 0;
      if (t < tokens) {
        const int r = find_owner(R, t, [&](int k) { return (long long)tok0[k]; });
        pos = length_of(r) + t - tok0[r];
        const int k = (int)divided((unsigned)pos);
        slot = (long long)page_at(r, k) * page + (pos - k * page);
      }
      a.slots[t] = slot;
      a.positions[t] = pos;
    } else {  // a page given back
      const int b = (int)(e - kv - a.max_tokens);
      const int r = find_owner(R, b, [&](int k) { return (long long)back0[k]; });
      a.free_pages[(tail_at + b) % ring] = a.block_table[(long long)r * a.table_stride + (b - back0[r])];
    }
  }
}

}  // namespace

int sm_count() {
  static std::atomic<int> count[64] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if ((n = count[dev]) == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    count[dev] = n;
  }
  return n;
}
namespace {
using Wide = __int128;  // (sizes and strides of a C caller may be anything)
struct Term {  // count * stride, count between lo and hi
  Wide stride, lo, hi;
};
// Whether offset + sum of the terms k.. can be above -below and below above.  steps: what the search may still take.
bool reaches(const Term* t, int n, int k, Wide offset, Wide below, Wide above, int* steps) {
  Wide least = 0, most = 0;  // of the terms behind k
  for (int i = k + 1; i < n; ++i) least += t[i].lo * t[i].stride, most += t[i].hi * t[i].stride;
  if (k == n) return offset > -below && offset < above;
  if (--*steps < 0) return true;
  // counts with offset + count * stride + most > -below and offset + count * stride + least < above
  auto floor_div = [](Wide x, Wide y) { return x / y - (x % y < 0 ? 1 : 0); };
  Wide lo = floor_div(-below - offset - most, t[k].stride) + 1, hi = floor_div(above - 1 - offset - least, t[k].stride);
  if (lo < t[k].lo) lo = t[k].lo;
  if (hi > t[k].hi) hi = t[k].hi;
  for (Wide c = lo; c <= hi; ++c)
    if (reaches(t, n, k + 1, offset + c * t[k].stride, below, above, steps)) return true;
  return false;
}
}  // namespace
bool share_memory(const Memory& a, const Memory& b) {
  if (!a.at || !b.at || a.reach <= 0 || b.reach <= 0) return false;
  Term t[6];
  int n = 0;
  auto add = [&](long long size, long long stride, bool of_a) {  // entries of b count upwards from those of a
    if (size <= 1 || stride == 0) return;
    Wide lo = of_a ? 1 - (Wide)size : 0, hi = of_a ? 0 : (Wide)size - 1;
    Wide s = stride;
    if (s < 0) {
      s = -s;
      const Wide x = -lo;
      lo = -hi;
      hi = x;
    }
    int k = 0;
    while (k < n && t[k].stride > s) ++k;
    if (k < n && t[k].stride == s) {
      t[k].lo += lo;
      t[k].hi += hi;
      return;
    }
    for (int i = n++; i > k; --i) t[i] = t[i - 1];
    t[k] = {s, lo, hi};
  };
  for (int i = 0; i < a.dims; ++i) {
    if (a.size[i] <= 0) return false;
    add(a.size[i], a.stride[i], true);
  }
  for (int i = 0; i < b.dims; ++i) {
    if (b.size[i] <= 0) return false;
    add(b.size[i], b.stride[i], false);
  }
  int steps = 2000;
  return reaches(t, n, 0, (Wide)(intptr_t)b.at - (Wide)(intptr_t)a.at, b.reach, a.reach, &steps);
}
int refuse_shared(const char* what, const Memory* m, int written, int n) {  // (n <= 16)
  // (most are apart as a whole: a fraction of a microsecond, a microsecond without)
  struct {
    Wide first, last;  // last: behind the last byte
  } at[16];
  for (int i = 0; i < n; ++i) {
    at[i].first = (Wide)(intptr_t)m[i].at;
    at[i].last = at[i].first + m[i].reach;
    for (int k = 0; k < m[i].dims; ++k) {
      const Wide far = m[i].size[k] > 1 ? (Wide)(m[i].size[k] - 1) * m[i].stride[k] : 0;
      (far < 0 ? at[i].first : at[i].last) += far;
    }
  }
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < n; ++j)
      if (at[i].first < at[j].last && at[j].first < at[i].last && share_memory(m[i], m[j])) return fail(MK_E_INVALID, "%s: %s and %s share memory", what, m[i].name, m[j].name);
  return 0;
}
int refuse_misaligned(const char* what, std::initializer_list<Address> all) {
  for (const Address& a : all)
    if ((uintptr_t)a.at % (unsigned)a.bytes) return fail(MK_E_INVALID, "%s: %s must be a multiple of %d bytes", what, a.name, a.bytes);
  return 0;
}
char* error_text() {
  static thread_local char text[kErrorBytes];
  return text;
}

}  // namespace mk_serving

extern "C" int mk_op_error(char* buf, int n) {
  if (!buf || n <= 0) return MK_E_INVALID;
  snprintf(buf, n, "%s", mk_serving::error_text());
  return 0;
}

extern "C" int mk_debug_share_memory(const int64_t* memory, const int64_t* other) {
  using namespace mk_serving;
  Memory m[2] = {};
  for (int k = 0; k < 2; ++k) {
    const int64_t* v = k ? other : memory;
    if (!v || v[2] < 0 || v[2] > 3) return MK_E_INVALID;
    m[k].at = (const void*)(intptr_t)v[0];
    m[k].reach = v[1];
    m[k].dims = (int)v[2];
    for (int i = 0; i < 3; ++i) m[k].size[i] = v[3 + i], m[k].stride[i] = v[6 + i];
  }
  return share_memory(m[0], m[1]) ? 1 : 0;
}

extern "C" int mk_plan_step(const mk_step_plan_args* args, void* stream) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "plan_step: null arguments");
  const mk_step_plan_args& a = *args;
  if (!a.lengths || !a.new_tokens || !a.block_table || !a.free_pages || !a.free_range_in || !a.qo_indptr || !a.kv_indptr || !a.kv_indices ||
      !a.last_page_len || !a.slots || !a.positions || !a.granted || !a.free_range_out)
    return fail(MK_E_INVALID, "plan_step: null pointer");
  if (a.requests < 1 || a.requests > MK_STEP_MAX_REQUESTS)
    return fail(a.requests < 1 ? MK_E_INVALID : MK_E_TOO_LARGE, "plan_step: %d requests (1 to %d)", a.requests, MK_STEP_MAX_REQUESTS);
  if (a.page_size < 1 || a.table_width < 1 || a.table_stride < a.table_width || a.max_tokens < 1 || a.max_indices < 1 || a.ring_size < 1)
    return fail(MK_E_INVALID, "plan_step: sizes must be positive and table rows may not overlap");
  if ((long long)a.requests * a.table_width >= 0x7fffffffll) return fail(MK_E_TOO_LARGE, "plan_step: block table of over 2^31 entries");
  // Every CTA works the sums out for itself, so what one writes no other may read or write.
  const size_t n = (size_t)a.requests;
  const struct {
    const void* at;
    size_t bytes;
    const char* name;
  } arrays[] = {{a.block_table, ((n - 1) * (size_t)a.table_stride + (size_t)a.table_width) * 4, "block_table"},
                {a.free_pages, (size_t)a.ring_size * 4, "free_pages"},
                {a.qo_indptr, (n + 1) * 4, "qo_indptr"},
                {a.kv_indptr, (n + 1) * 4, "kv_indptr"},
                {a.kv_indices, (size_t)a.max_indices * 4, "kv_indices"},
                {a.last_page_len, n * 4, "last_page_len"},
                {a.slots, (size_t)a.max_tokens * 8, "slots"},
                {a.positions, (size_t)a.max_tokens * 4, "positions"},
                {a.granted, n * 4, "granted"},
                {a.free_range_out, 16, "free_range"},
                {a.lengths, n * 4, "lengths"},
                {a.new_tokens, n * 4, "new_tokens"},
                {a.free_range_in, 16, "free_range"}};
  constexpr int kWritten = 10;
  for (int i = 0; i < kWritten; ++i)
    for (int j = i + 1; j < (int)(sizeof arrays / sizeof *arrays); ++j) {
      const uintptr_t x = (uintptr_t)arrays[i].at, y = (uintptr_t)arrays[j].at;
      if (x < y + arrays[j].bytes && y < x + arrays[i].bytes) return fail(MK_E_INVALID, "plan_step: %s and %s share memory", arrays[i].name, arrays[j].name);
    }
  if (int rc = refuse_misaligned("plan_step", {{"lengths", a.lengths, 4}, {"new_tokens", a.new_tokens, 4}, {"block_table", a.block_table, 4}, {"free_pages", a.free_pages, 4},
                                               {"free_range", a.free_range_in, 8}, {"qo_indptr", a.qo_indptr, 4}, {"kv_indptr", a.kv_indptr, 4}, {"kv_indices", a.kv_indices, 4},
                                               {"last_page_len", a.last_page_len, 4}, {"slots", a.slots, 8}, {"positions", a.positions, 4}, {"granted", a.granted, 4},
                                               {"free_range", a.free_range_out, 8}}))
    return rc;
  const size_t smem = 4 * (n + 1) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_shared<step_plan_kernel>(4 * (MK_STEP_MAX_REQUESTS + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return fail(MK_E_CUDA, "plan_step: %s", cudaGetErrorString(e));
  }
  const long long entries = (long long)a.max_indices + a.max_tokens;
  const int ctas = (int)((entries + kPlanThreads - 1) / kPlanThreads);
  PlanParams p{a, -1};
  for (int k = 0; k < 31; ++k)
    if (a.page_size == 1 << k) p.shift = k;
  step_plan_kernel<<<ctas < sm_count() ? ctas : sm_count(), kPlanThreads, smem, (cudaStream_t)stream>>>(p);
  return launched("plan_step");
}
