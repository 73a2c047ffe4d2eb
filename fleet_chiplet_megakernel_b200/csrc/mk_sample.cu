// mk_sample_tokens: a token per request from its row of logits and a given random number.
//
//   w_i = exp((l_i - max l) / temperature)
//   order: larger logits first, equal ones by index.  top_k keeps the first k; of their weights' sum W, top_p keeps a token if the
//   weights before it in the order stay below top_p W; min_p keeps w_i >= min_p.  So each keeps the beginning of the order,
//   and one border in it says what all three keep.
//   The token is the first, by index, at which the running sum of the kept weights exceeds u times their sum.
//
// A token is a whole number: with sums in fp32 one draw in some thousands would fall on the neighbour's side of a border.  Weights
// and their sums are therefore 64-bit, and every sum has one fixed order (no atomics on anything but counts).
//
// A row is taken by a cluster of up to 8 CTAs, as many as leave the SMs busy; each has a contiguous part of the vocabulary and
// reads it a few times, from L2 after the first.  The border is found by counting: a histogram over bins that fall with the logit
// (for top_p with bounds of each bin's weight from its edges) leaves one bin or few that the border can be in, what is
// above is summed, and the few candidates are sorted.  Where they are too many for that (equal logits, flat rows), the histogram is
// repeated over the candidates' range of (logit, index), which a pass divides by 1024.  Bound by the latency of these steps, below
// some tens of rows.
#include <cooperative_groups.h>

#include "mk_serving.cuh"

namespace cg = cooperative_groups;

namespace mk_serving {
namespace {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 1024;          // one a thread
constexpr int kCandidates = 2048;    // sorted at once
constexpr int kMaxCluster = 8;
constexpr int kInner = 1024;         // (2^32 / 1024 elements a CTA)
constexpr double kBinsPerUnit = 32.0;  // linear bins of weights: a factor of exp(1/32) each

// Larger logits are larger keys; -0 and +0 are equal, NaN counts as minus infinity.
__device__ __forceinline__ uint32_t key_of(float l) {
  l = isnan(l) ? -INFINITY : l + 0.f;
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// place in the order: larger is earlier
__device__ __forceinline__ uint64_t place_of(float l, int i) { return ((uint64_t)key_of(l) << 32) | (uint32_t)~i; }

struct SampleShared {
  uint32_t hist[kBins];
  uint32_t inner[kBins];            // of linear bins: how far into the bin its logits lie, summed, in units of 1 / kInner
  uint64_t list[kCandidates];       // rank 0's is used
  double sums[kSampleWarps + 1];
  uint64_t words[kSampleWarps];
  double mass;                      // this CTA's share of a sum over the cluster
  uint64_t best;                    // this CTA's first place
  uint64_t lo, hi;                  // range of this CTA's candidates
  uint32_t listed;                  // rank 0's: candidates in the list
  uint64_t border;                  // written by rank 0 into every CTA
  double border_mass;
  int found;
  int first_bin, last_bin;
};

struct Row {
  const void* logits;
  int dtype, vocab, begin, end;
  float top;
  double inv_t;
};
__device__ __forceinline__ float logit_at(const Row& r, int i) {
  float l;
  if (r.dtype == MK_F32) l = __ldg((const float*)r.logits + i);
  else if (r.dtype == MK_BF16) l = __bfloat162float(((const __nv_bfloat16*)r.logits)[i]);
  else l = __half2float(((const __half*)r.logits)[i]);
  return isnan(l) ? -INFINITY : l + 0.f;
}
__device__ __forceinline__ double weight(const Row& r, float l) {
  if (l == r.top) return 1.0;  // (both may be infinite)
  if (l == -INFINITY) return 0.0;
  return exp(((double)l - (double)r.top) * r.inv_t);
}

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double v, SampleShared& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sums[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = s.sums[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kAll, t, o);
  return t;
}
// Sum of the values before this thread's, in the order of the threads; *total: of all.
template <typename N> __device__ __forceinline__ N block_before(N v, N* scratch, N* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N u = __shfl_up_sync(kAll, in, o);
    if (lane >= o) in += u;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = in;
  __syncthreads();
  N c = scratch[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N u = __shfl_up_sync(kAll, c, o);
    if (lane >= o) c += u;
  }
  *total = __shfl_sync(kAll, c, 31);
  const N warps = __shfl_sync(kAll, c, warp > 0 ? warp - 1 : 0);
  __syncthreads();
  N before = __shfl_up_sync(kAll, in, 1);  // (not in - v: the sum before a thread must be the inclusive one of its neighbour)
  if (lane == 0) before = 0;
  return (warp > 0 ? warps : N(0)) + before;
}

struct Sampler {
  cg::cluster_group cluster;
  SampleShared& s;
  Row r;
  int ranks, rank;

  template <typename N> __device__ __forceinline__ N* peer(N* p, int k) { return cluster.map_shared_rank(p, k); }
  // Sum over the cluster, in the order of the ranks.
  __device__ double cluster_sum(double v) {
    const double mine = block_sum(v, s);
    if (threadIdx.x == 0) s.mass = mine;
    cluster.sync();
    double t = 0.0;
    for (int k = 0; k < ranks; ++k) t += *peer(&s.mass, k);
    cluster.sync();
    return t;
  }

  // First element in the order that the criterion leaves out is not wanted here but the last that it keeps:
  // by count: the k-th; by mass: the last with (weights before it) < limit.  Returns its place; *kept: the weights up to and with it.
  __device__ uint64_t border(bool by_mass, double limit, long long k, double* kept) {
    uint64_t lo = 0, hi = ~0ull;     // places of the candidates
    long long above = 0;             // elements before them
    double above_mass = 0.0;
    long long left = r.vocab;        // candidates
    bool linear = true;              // bins fall linearly with the logit; later: a shift of the place
    const float per_bin = by_mass ? (float)(kBinsPerUnit * r.inv_t) : 64.f;
    for (;;) {
      const int shift = linear ? 0 : max(0, 64 - (int)__clzll(hi - lo) - 10);
      auto depth_of = [&](float l) -> float { return l == -INFINITY ? (float)kBins : r.top == l ? 0.f : fminf((r.top - l) * per_bin, (float)kBins); };
      auto bin_of = [&](float l, uint64_t place) -> int { return linear ? min((int)depth_of(l), kBins - 1) : (int)((hi - place) >> shift); };
      s.hist[threadIdx.x] = s.inner[threadIdx.x] = 0;
      __syncthreads();
      for (int i = r.begin + threadIdx.x; i < r.end; i += kSampleThreads) {
        const float l = logit_at(r, i);
        const uint64_t place = place_of(l, i);
        if (place < lo || place > hi) continue;
        const int b = bin_of(l, place);
        atomicAdd(&s.hist[b], 1u);
        if (by_mass && linear && b < kBins - 1) atomicAdd(&s.inner[b], (uint32_t)((depth_of(l) - (float)b) * (float)kInner));
      }
      cluster.sync();
      uint32_t count = 0;
      for (int q = 0; q < ranks; ++q) count += *peer(&s.hist[threadIdx.x], q);
      // Which bins can the border be in?  By mass: the weights before a bin are known up to those of its edges.
      int first_bin, last_bin;
      if (threadIdx.x == 0) {
        s.first_bin = kBins - 1;
        s.last_bin = 0;
      }
      if (!by_mass) {
        uint64_t total;
        const uint64_t before = block_before((uint64_t)count, s.words, &total);
        // (k is at most the number of elements)
        if (count > 0 && (long long)before + above < k && (long long)(before + count) + above >= k) s.first_bin = s.last_bin = threadIdx.x;
      } else {
        double low_w = 0.0, high_w = 0.0;  // bounds of the mean weight in the bin
        if (linear) {
          // exp is convex: the mean is at least the weight at the mean depth and at most the chord's value there.  The depth is known
          // to 1 / kInner of a bin and to some units of 2^-24.
          uint32_t inner = 0;
          for (int q = 0; q < ranks; ++q) inner += *peer(&s.inner[threadIdx.x], q);
          const double edge = exp(-(double)threadIdx.x / kBinsPerUnit), slope = 1.0 - exp(-1.0 / kBinsPerUnit);
          if (threadIdx.x == kBins - 1) {
            high_w = edge * (1.0 + 1e-4);
          } else if (count > 0) {
            const double f = (double)inner / ((double)count * kInner);
            low_w = edge * exp(-(f + 1.0 / kInner) / kBinsPerUnit) * (1.0 - 1e-5);
            high_w = edge * (1.0 - slope * f) * (1.0 + 1e-5);
          }
        } else {
          const uint64_t top = (uint64_t)threadIdx.x << shift, end = top + ((1ull << shift) - 1);
          const uint64_t a = top <= hi - lo ? hi - top : lo, b = end <= hi - lo ? hi - end : lo;
          high_w = weight(r, logit_of((uint32_t)(a >> 32))) * (1.0 + 1e-9);
          low_w = weight(r, logit_of((uint32_t)(b >> 32))) * (1.0 - 1e-9);
        }
        double total;
        const double low_before = above_mass + block_before(count * low_w, s.sums, &total);
        const double high_before = above_mass + block_before(count * high_w, s.sums, &total);
        // kept for certain: all of a bin whose weights with those before it stay below the limit; left out for certain: low_before >= limit
        if (count > 0 && low_before * (1.0 - 1e-9) < limit) {
          if ((high_before + count * high_w) * (1.0 + 1e-9) >= limit) atomicMin(&s.first_bin, (int)threadIdx.x);
          atomicMax(&s.last_bin, (int)threadIdx.x);
        }
      }
      __syncthreads();
      first_bin = min(s.first_bin, s.last_bin);
      last_bin = s.last_bin;
      uint64_t candidates, all;
      {
        const uint64_t in = (int)threadIdx.x >= first_bin && (int)threadIdx.x <= last_bin ? count : 0;
        const uint64_t ahead = (int)threadIdx.x < first_bin ? count : 0;
        block_before(in, s.words, &candidates);
        block_before(ahead, s.words, &all);
        above += (long long)all;
      }
      // the weights above the candidates, and the candidates themselves or their range
      const bool few = candidates <= kCandidates;
      if (threadIdx.x == 0) {
        s.lo = ~0ull;
        s.hi = 0;
        s.listed = 0;
      }
      cluster.sync();  // (all have read the histograms; rank 0's list is empty)
      uint32_t* listed = peer(&s.listed, 0);
      uint64_t* list = peer(s.list, 0);
      double mass = 0.0;
      uint64_t my_lo = ~0ull, my_hi = 0;
      for (int i = r.begin + threadIdx.x; i < r.end; i += kSampleThreads) {
        const float l = logit_at(r, i);
        const uint64_t place = place_of(l, i);
        if (place < lo || place > hi) continue;
        const int b = bin_of(l, place);
        if (b < first_bin) mass += weight(r, l);
        else if (b <= last_bin) {
          if (few) list[atomicAdd(listed, 1u)] = place;
          my_lo = min(my_lo, place);
          my_hi = max(my_hi, place);
        }
      }
      above_mass += cluster_sum(mass);
      if (few) {
        if (rank == 0) {
          // sorted, earliest first (the list's order was that of arrival, the sorted one is not)
          int n = 32;
          while (n < (int)candidates) n <<= 1;
          for (int i = threadIdx.x; i < n; i += kSampleThreads)
            if (i >= (int)candidates) s.list[i] = 0;
          __syncthreads();
          for (int size = 2; size <= n; size <<= 1)
            for (int step = size >> 1; step > 0; step >>= 1) {
              for (int i = threadIdx.x; i < n / 2; i += kSampleThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const uint64_t x = s.list[a], y = s.list[b];
                if ((x < y) == ((a & size) == 0)) {
                  s.list[a] = y;
                  s.list[b] = x;
                }
              }
              __syncthreads();
            }
          // two of them a thread
          const int at = 2 * threadIdx.x;
          const uint64_t p0 = at < (int)candidates ? s.list[at] : 0, p1 = at + 1 < (int)candidates ? s.list[at + 1] : 0;
          const double w0 = at < (int)candidates ? weight(r, logit_of((uint32_t)(p0 >> 32))) : 0.0;
          const double w1 = at + 1 < (int)candidates ? weight(r, logit_of((uint32_t)(p1 >> 32))) : 0.0;
          double total;
          const double before = above_mass + block_before(w0 + w1, s.sums, &total);
          if (threadIdx.x == 0) s.first_bin = 0;
          __syncthreads();
          bool keep0, keep1;
          if (by_mass) {
            keep0 = at < (int)candidates && (before < limit || above + at == 0);
            keep1 = at + 1 < (int)candidates && before + w0 < limit;
          } else {
            keep0 = at < (int)candidates && above + at < k;
            keep1 = at + 1 < (int)candidates && above + at + 1 < k;
          }
          const int last = keep1 ? at + 1 : keep0 ? at : -1;
          if (last >= 0) atomicMax(&s.first_bin, last);
          __syncthreads();
          if (last == s.first_bin && last >= 0) {
            const uint64_t place = keep1 ? p1 : p0;
            const double up_to = keep1 ? before + w0 + w1 : before + w0;
            for (int q = 0; q < ranks; ++q) {
              *peer(&s.border, q) = place;
              *peer(&s.border_mass, q) = up_to;
            }
          }
        }
        cluster.sync();
        *kept = s.border_mass;
        return s.border;
      }
      // too many: their range, in 1024 parts
      if (my_lo <= my_hi) {
        atomicMin((unsigned long long*)&s.lo, (unsigned long long)my_lo);
        atomicMax((unsigned long long*)&s.hi, (unsigned long long)my_hi);
      }
      cluster.sync();
      lo = ~0ull;
      hi = 0;
      for (int q = 0; q < ranks; ++q) {
        lo = min(lo, *peer(&s.lo, q));
        hi = max(hi, *peer(&s.hi, q));
      }
      cluster.sync();
      if (by_mass && !linear && 4 * (long long)candidates > 3 * left) {
        // bounds from the edges can leave all bins open, where logits of very different weight share one: halve the range
        const uint64_t mid = lo + ((hi - lo) >> 1);
        double w = 0.0, n = 0.0;
        for (int i = r.begin + threadIdx.x; i < r.end; i += kSampleThreads) {
          const float l = logit_at(r, i);
          const uint64_t place = place_of(l, i);
          if (place <= mid || place > hi) continue;
          w += weight(r, l);
          n += 1.0;
        }
        w = cluster_sum(w);
        n = cluster_sum(n);
        if (above_mass + w < limit) {
          above += (long long)n;
          above_mass += w;
          hi = mid;
        } else {
          lo = mid + 1;
        }
      }
      left = (long long)candidates;
      linear = false;
    }
  }
};

__device__ __forceinline__ float setting(const float* per_request, float value, int r) { return per_request ? __ldg(per_request + r) : value; }

__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const __grid_constant__ mk_sample_args a) {
  __shared__ SampleShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int req = blockIdx.x / ranks;
  long long row = req;
  if (a.qo_indptr) {  // the last of the request's rows
    const int q0 = __ldg(a.qo_indptr + req), q1 = __ldg(a.qo_indptr + req + 1);
    row = q1 > q0 && q0 >= 0 ? q1 - 1 : -1;
  }
  if (row < 0 || row >= a.rows) {  // (the whole cluster)
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[req] = -1;
      if (a.logprobs) a.logprobs[req] = -INFINITY;
    }
    return;
  }
  const float temperature = setting(a.temperature, a.temperature_value, req);
  const float top_p = setting(a.top_p, a.top_p_value, req), min_p = setting(a.min_p, a.min_p_value, req);
  const int top_k = a.top_k ? __ldg(a.top_k + req) : a.top_k_value;
  Sampler d{cluster, s, {}, ranks, rank};
  Row& r = d.r;
  r.dtype = a.dtype;
  r.vocab = a.vocab;
  r.logits = (const char*)a.logits + row * a.row_stride * (a.dtype == MK_F32 ? 4 : 2);
  const int per = (a.vocab + ranks - 1) / ranks;
  r.begin = min(a.vocab, rank * per);
  r.end = min(a.vocab, r.begin + per);

  // the first place
  uint64_t best = 0;
  for (int i = r.begin + threadIdx.x; i < r.end; i += kSampleThreads) best = max(best, place_of(logit_at(r, i), i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(kAll, (unsigned long long)best, o));
  if ((threadIdx.x & 31) == 0) s.words[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSampleWarps; ++w) best = max(best, s.words[w]);
    s.best = best;
    s.found = -1;
  }
  cluster.sync();
  best = 0;
  for (int q = 0; q < ranks; ++q) best = max(best, *d.peer(&s.best, q));
  r.top = logit_of((uint32_t)(best >> 32));
  const bool nothing = r.top == -INFINITY;
  if (nothing || !(temperature > 0.f)) {  // no token can be chosen, or the greedy one is
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[req] = nothing ? -1 : (long long)(uint32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[req] = nothing ? -INFINITY : 0.f;
    }
    cluster.sync();  // nobody leaves while another reads its shared memory
    return;
  }
  r.inv_t = 1.0 / (double)temperature;

  uint64_t least = 0;  // the border: places from here on are kept
  double kept_mass = -1.0;
  const bool cut_k = top_k > 0 && top_k < a.vocab, cut_p = top_p < 1.f;
  if (cut_k) least = d.border(false, 0.0, top_k, &kept_mass);
  if (cut_p) {
    if (!cut_k) {
      double w = 0.0;
      for (int i = r.begin + threadIdx.x; i < r.end; i += kSampleThreads) w += weight(r, logit_at(r, i));
      kept_mass = d.cluster_sum(w);
    }
    double unused;
    const uint64_t b = d.border(true, (double)top_p * kept_mass, 0, &unused);
    least = max(least, b);
  }

  // the kept weights in the order of the index: a warp has a contiguous part of the CTA's
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = ((r.end - r.begin + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
  const int b0 = min(r.end, r.begin + warp * part), b1 = min(r.end, b0 + part);
  auto kept = [&](int i) -> double {
    const float l = logit_at(r, i);
    if (place_of(l, i) < least) return 0.0;
    const double w = weight(r, l);
    return w >= (double)min_p ? w : 0.0;
  };
  double mine = 0.0;
  for (int i = b0 + lane; i < b1; i += 32) mine += kept(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(kAll, mine, o);
  __syncthreads();
  if (lane == 0) s.sums[warp] = mine;
  __syncthreads();
  double in_cta = 0.0;
  for (int w = 0; w < kSampleWarps; ++w) in_cta += s.sums[w];
  if (threadIdx.x == 0) s.mass = in_cta;
  cluster.sync();
  // the first CTA whose sum exceeds the goal has the token, and of its warps the first; where rounding leaves none, the last that keeps any
  double total = 0.0;
  for (int q = 0; q < ranks; ++q) total += *d.peer(&s.mass, q);
  const double goal = (double)__ldg(a.u + req) * total;
  double end = 0.0, before = 0.0;
  int owner = -1;
  for (int q = 0; q < ranks; ++q) {
    const double m = *d.peer(&s.mass, q);
    if (m > 0.0 && (owner < 0 || goal >= end)) {
      owner = q;
      before = end;
    }
    end += m;
  }
  if (rank == owner) {
    double from = before;
    end = before;
    owner = -1;
    for (int w = 0; w < kSampleWarps; ++w) {
      const double m = s.sums[w];
      if (m > 0.0 && (owner < 0 || goal >= end)) {
        owner = w;
        from = end;
      }
      end += m;
    }
    if (warp == owner) {
      double run = from;
      int token = -1;
      double w_token = 0.0;
      for (int i0 = b0; i0 < b1; i0 += 32) {
        const int i = i0 + lane;
        const double w = i < b1 ? kept(i) : 0.0;
        double up = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double u = __shfl_up_sync(kAll, up, o);
          if (lane >= o) up += u;
        }
        const unsigned over = __ballot_sync(kAll, w > 0.0 && run + up > goal), any = __ballot_sync(kAll, w > 0.0);
        if (any) {
          const int k = over ? __ffs(over) - 1 : 31 - __clz(any);
          token = i0 + k;
          w_token = __shfl_sync(kAll, w, k);
        }
        if (over) break;
        run += __shfl_sync(kAll, up, 31);
      }
      if (lane == 0) {
        a.tokens[req] = token;
        if (a.logprobs) a.logprobs[req] = (float)log(w_token / total);
      }
    }
  }
  cluster.sync();
}

}  // namespace
}  // namespace mk_serving

extern "C" int mk_sample_tokens(const mk_sample_args* args, void* stream) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "sample_tokens: null arguments");
  const mk_sample_args& a = *args;
  if (!a.logits || !a.u || !a.tokens) return fail(MK_E_INVALID, "sample_tokens: null pointer");
  if (a.dtype != MK_BF16 && a.dtype != MK_F16 && a.dtype != MK_F32) return fail(MK_E_INVALID, "sample_tokens: logits are bf16, fp16 or fp32");
  if (a.requests < 0 || a.rows < 0 || a.vocab < 1 || a.vocab > 0x3fffffff) return fail(MK_E_INVALID, "sample_tokens: bad sizes");
  if (a.requests > 0x7fffffff / kMaxCluster) return fail(MK_E_TOO_LARGE, "sample_tokens: %d requests", a.requests);
  if (!a.qo_indptr && a.rows < a.requests) return fail(MK_E_INVALID, "sample_tokens: %d rows of logits for %d requests", a.rows, a.requests);
  if (a.requests == 0) return 0;
  int ranks = kMaxCluster;
  while (ranks > 1 && ((long long)ranks * a.requests > sm_count() || a.vocab / ranks < 1024)) ranks >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ranks * a.requests));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, a);
  return e == cudaSuccess ? 0 : fail(MK_E_CUDA, "sample_tokens: launch failed: %s", cudaGetErrorString(e));
}
