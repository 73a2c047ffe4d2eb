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
// A row is taken by a cluster of up to 8 CTAs, as many as run at once for all rows; each has a contiguous part of the vocabulary and
// reads it two to four times in 16-byte words, from L2 after the first.  What is kept is mostly a few tokens, so the usual way is to find a
// bound that few logits exceed, to list these, and to do the rest of the work on the sorted list in one CTA:
//   top_k: at least k logits are as large as the k-th largest of any choice of them; of two a thread, its largest and that of another
//          group of 16 bytes, a histogram gives the bound (with one, and 1024 threads a row, top_k = 1000 of 151936 takes 134 us, 41 so);
//   top_p: a histogram of all logits near the largest, in bins of a factor exp(1/64) of the weight, and the sum of all weights in fp32 say
//          to 1e-5 where the border is; the list tells whether a place in it lies that close to the border.
// Where the border is too close to call, all weights are summed in 64 bits and the list is looked at again.  Where the list would be too long, the
// bins that the border can be in are listed in the pass that sums all weights and those above in 64 bits; where these are too many as well, the
// border is found step by step: bins that it can be in, the weights above them, and again over the candidates' range of (logit, index),
// which a step divides by 1024.  The draw then reads the row once more.  CTAs hand each other sums by storing them into their
// neighbours' shared memory ahead of a cluster barrier.  Rows that keep all tokens or thousands are bound by the instructions of the weights in
// 64 bits (some 25 a logit) and of the histograms, the others by the latency of the steps.  151936 fp32 logits, 1 and 64 rows: largest logit 5
// and 8 us, all tokens 13 and 28, top_k = 50 14 and 21, top_p that keeps some thousands 37 and 75; the 64 rows take 6 us of the memory's time.
#include <cooperative_groups.h>

#include "mk_serving.cuh"

namespace cg = cooperative_groups;

namespace mk_serving {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;      // one a thread
constexpr int kCandidates = 2 * kThreads;  // sorted at once, two a thread
constexpr int kMaxCluster = 8;
constexpr int kInner = 1024;         // parts of a bin, at most (inner_parts())
constexpr double kBinsPerUnit = 32.0;
constexpr int kSlots = 4;
constexpr float kNearBins = 64.f;    // bins a unit of (largest logit - logit) / temperature, near the largest
constexpr float kTopBins = 16.f;     // bins a unit of (largest logit - logit) for the bound of the k-th
// In how many parts a bin is divided for the sums of how far into it its logits lie: so many that all logits of the row in one bin, over the
// whole cluster, stay below 2^32.  1024 up to a vocabulary of 2^22, 4 at the largest.
__host__ __device__ constexpr int inner_parts(int vocab) {
  int n = kInner;
  while ((long long)n * vocab > 1ll << 32) n >>= 1;
  return n;
}
static_assert(inner_parts(1 << 22) == kInner && inner_parts(0x3fffffff) == 4, "a largest sum is vocab * (parts - 1)");
constexpr float kSumError = 1e-5f;   // relative, of a sum of weights in fp32: the argument of exp is off by 2^-22 of itself, at most 23 where weights count

// Larger logits are larger keys; -0 and +0 are equal, NaN counts as minus infinity.
__device__ __forceinline__ float clean(float l) { return fmaxf(l, -INFINITY); }
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// place in the order: larger is earlier
__device__ __forceinline__ uint64_t place_of(float l, int i) { return ((uint64_t)key_of(l) << 32) | (uint32_t)~i; }

struct SampleShared {
  uint32_t hist[kBins];
  uint32_t inner[kBins];            // of linear bins: how far into the bin its logits lie, summed, in units of 1 / inner_parts()
  uint64_t list[kCandidates];       // rank 0's is used
  double weights[kCandidates];      // of the list's
  double power[64];                 // 2^(i / 64)
  double sums[kWarps];
  uint64_t words[kWarps];
  double slot[kSlots][kMaxCluster];  // sums of the ranks, in turn; a slot comes round again behind three more barriers
  uint64_t lo[kMaxCluster], hi[kMaxCluster];  // of every rank: first place; the range of its candidates
  uint32_t counts[kMaxCluster];     // of every rank: candidates that it has listed
  uint32_t listed[3];               // rank 0's: candidates in the list, of the rounds in turn; the first list's
  int close;                        // rank 0 -> all: the border is too close to say
  uint64_t border;                  // written by rank 0 into every CTA
  double border_mass;
  int first_bin, last_bin, last_kept;
  uint32_t range[2];                // of the list that is being sorted: largest, smallest upper half
};

// A row, as the groups of 16 bytes (aligned) that it lies in: the first and the last may have elements outside.
template <typename T> struct Row {
  static constexpr int N = 16 / sizeof(T);
  const T* logits;
  int vocab, shift;   // element of a group g: g N - shift + e
  int g0, g1;         // this CTA's groups
  float top;
  double scale;       // 64 log2(e) / temperature
  double largest;     // top
  const double* power;

  __device__ __forceinline__ int index(int g) const { return g * N - shift; }
  __device__ __forceinline__ bool inside(int g) const { return index(g) >= 0 && index(g) + N <= vocab; }
  // The logits of a group that is wholly inside the row.
  __device__ __forceinline__ void load(int g, float (&l)[N]) const {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(logits + index(g)));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        l[e] = clean(__uint_as_float(w[e]));
      } else {
        const float2 f = unpack2<T>(w[e]);
        l[2 * e] = clean(f.x);
        l[2 * e + 1] = clean(f.y);
      }
    }
  }
  // The same of any group; returns a bit for every element that is outside the row.
  __device__ __forceinline__ uint32_t load_edge(int g, float (&l)[N]) const {
    uint32_t outside = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = index(g) + e;
      const bool in = i >= 0 && i < vocab;
      l[e] = in ? clean(to_float(logits[i])) : -INFINITY;
      outside |= in ? 0u : 1u << e;
    }
    return outside;
  }
  float lowest;       // below this logit a weight is 0
  float plain;        // from this logit on a weight needs no care: it is a normal number, and neither infinity nor NaN is in its way
  // exp((l - top) / temperature), exactly 1 for the largest: the argument y in units of ln 2 / 64, its whole part by table (P. T. P. Tang's method, 1989), the rest
  // r (|r| <= 1/2) by the series up to the fourth power; the next term is 4e-14.
  __device__ __forceinline__ double plain_weight(float l) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: a sum with it is rounded to a whole number
    constexpr double c1 = 0.6931471805599453094 / 64.0, c2 = c1 * c1 / 2.0, c3 = c2 * c1 / 3.0, c4 = c3 * c1 / 4.0;
    const double y = ((double)l - largest) * scale, big = y + kRound;
    const int n = __double2loint(big);
    const double r = y - (big - kRound);
    const double t = power[n & 63];
    const double e = fma(t * r, fma(r, fma(r, fma(r, c4, c3), c2), c1), t);
    return __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
  }
  __device__ __forceinline__ double weight(float l) const { return l >= plain ? plain_weight(l) : far_weight(l, top, scale); }
  // next to the smallest numbers, and where infinities meet
  static __device__ __noinline__ double far_weight(float l, float top, double scale) {
    if (l == top) return 1.0;  // (both may be infinite)
    const double y = ((double)l - (double)top) * scale;
    return l == -INFINITY || isnan(y) ? 0.0 : exp(y * (0.6931471805599453094 / 64.0));
  }
  // f(logits, n, index of the first) for all elements of the CTA: n = N at a time, at the row's two ends one.  DEEP: several loads of a
  // thread in flight (code that runs once or twice is better short).
  template <bool DEEP = false, typename F> __device__ __forceinline__ void each_group(const F& f) const {
    constexpr int U = DEEP ? 16 / N : 1;
    const int i0 = g0 < g1 && !inside(g0) ? g0 + 1 : g0, i1 = g1 > i0 && !inside(g1 - 1) ? g1 - 1 : g1;
    int g = i0 + threadIdx.x;
    if constexpr (U > 1) {
#pragma unroll 1
      for (; g + (U - 1) * kThreads < i1; g += U * kThreads) {
        float l[U][N];
#pragma unroll
        for (int k = 0; k < U; ++k) load(g + k * kThreads, l[k]);
#pragma unroll
        for (int k = 0; k < U; ++k) f(l[k], N, index(g + k * kThreads));
      }
    }
#pragma unroll 1
    for (; g < i1; g += kThreads) {
      float l[N];
      load(g, l);
      f(l, N, index(g));
    }
    if (threadIdx.x < 2 * N) {  // a thread an element
      const int edge = threadIdx.x < N ? g0 : g1 - 1, i = index(edge) + (int)threadIdx.x % N;
      const bool mine = threadIdx.x < N ? i0 > g0 : i1 < g1;
      if (mine && i >= 0 && i < vocab) {
        float l[N];
        l[0] = clean(to_float(logits[i]));
        f(l, 1, i);
      }
    }
  }
  // f(logit, index)
  template <bool DEEP = false, typename F> __device__ __forceinline__ void each(const F& f) const {
    each_group<DEEP>([&](const float (&l)[N], int n, int i) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < n) f(l[e], i + e);
    });
  }
};

// f(weight, logit, index) for all elements whose weight is not 0: those that are plain without a branch, so that the weights of a group are
// worked out side by side.
template <typename T, typename F> __device__ __forceinline__ void each_weight(const Row<T>& r, const F& f) {
  constexpr int N = Row<T>::N;
  r.each_group([&](const float (&l)[N], int n, int i) {
    uint32_t unsure = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const double w = r.plain_weight(l[e]);
      if (e < n && l[e] >= r.plain) f(w, l[e], i + e);
      else if (e < n && l[e] >= r.lowest) unsure |= 1u << e;
    }
    while (unsure) {
      const int k = __ffs(unsure) - 1;
      unsure &= unsure - 1;
      const float x = clean(to_float(r.logits[i + k]));
      f(r.weight(x), x, i + k);
    }
  });
}

// Sum over the block in a fixed order; thread 0 to kMaxCluster - 1 get it (and all others).
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
template <typename V> __device__ __forceinline__ V block_before(V v, V* scratch, V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(kAll, in, o);
    if (lane >= o) in += u;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = in;
  __syncthreads();
  V c = scratch[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(kAll, c, o);
    if (lane >= o) c += u;
  }
  *total = __shfl_sync(kAll, c, 31);
  const V warps = __shfl_sync(kAll, c, warp > 0 ? warp - 1 : 0);
  V before = __shfl_up_sync(kAll, in, 1);  // (not in - v: the sum before a thread must be the inclusive one of its neighbour)
  if (lane == 0) before = 0;
  return (warp > 0 ? warps : V(0)) + before;
}

template <typename T> struct Sampler {
  cg::cluster_group cluster;
  SampleShared& s;
  Row<T> r;
  int ranks, rank, turn;  // turn: of the slots and the list's counters

  template <typename V> __device__ __forceinline__ V* peer(V* p, int k) { return cluster.map_shared_rank(p, k); }
  // A sum over the cluster, in the order of the ranks: give() on this side of a barrier, taken() on the other.
  __device__ __forceinline__ void give(double v) {
    const double mine = block_sum(v, s);
    if ((int)threadIdx.x < ranks) *peer(&s.slot[turn & (kSlots - 1)][rank], threadIdx.x) = mine;
  }
  __device__ __forceinline__ double taken() {
    double t = 0.0;
    for (int k = 0; k < ranks; ++k) t += s.slot[turn & (kSlots - 1)][k];
    ++turn;
    return t;
  }
  // Linear bins: the depth below the largest logit in units of a factor exp(1/32) of the weight; the last bin takes all that is deeper.
  __device__ __forceinline__ float depth(float l) const {
    if (l == r.top) return 0.f;
    return fminf((r.top - l) * per_bin, (float)(kBins - 1));  // (infinite differences too)
  }
  float per_bin;
  float parts;            // inner_parts()
  uint32_t count;         // of this thread's bin, over the cluster
  uint32_t inner_count;   // how far into it they lie, summed
  double low_w, high_w;   // bounds of the mean weight in it

  // exp is convex: the mean weight in a bin is at least the weight at the mean depth and at most the chord's value there.  The depth is
  // known to 1 / parts of a bin and to some units of 2^-24 relative.
  __device__ __forceinline__ void mean_bounds(uint32_t inner, float per_unit) {
    low_w = high_w = 0.0;
    const float edge = expf(-(float)threadIdx.x / per_unit);  // (fp32 is off by some 1e-6 here)
    if (threadIdx.x == kBins - 1) {
      high_w = (double)edge * (1.0 + 1e-4);
    } else if (count > 0) {
      const float f = (float)inner / ((float)count * parts);
      low_w = (double)(edge * expf(-(f + 1.f / parts) / per_unit)) * (1.0 - 1e-5);
      high_w = (double)(edge * (1.f - (1.f - expf(-1.f / per_unit)) * f)) * (1.0 + 1e-5);
    }
  }
  // Histogram of the linear bins; with `sum`, *mass: the sum of all weights.
  __device__ void linear_bins(bool sum, double* mass) {
    double w = 0.0;
    r.each([&](float l, int) {
      const float d = depth(l);
      const int b = (int)d;
      atomicAdd(&s.hist[b], 1u);
      if (b < kBins - 1) atomicAdd(&s.inner[b], (uint32_t)((d - (float)b) * parts));
      if (sum) w += r.weight(l);
    });
    if (sum) give(w);
    cluster.sync();
    if (sum) *mass = taken();
    count = 0;
    uint32_t inner = 0;
    for (int q = 0; q < ranks; ++q) {
      count += *peer(&s.hist[threadIdx.x], q);
      inner += *peer(&s.inner[threadIdx.x], q);
    }
    mean_bounds(inner, (float)kBinsPerUnit);
  }

  // The CTAs' lists (s.list, s.listed[2]) end to end at rank 0; returns how long it is (kCandidates + 1: longer than that).
  __device__ int collected() {
    __syncthreads();
    const uint32_t mine = s.listed[2];
    if ((int)threadIdx.x < ranks) *peer(&s.counts[rank], threadIdx.x) = mine;
    cluster.sync();
    uint64_t all = 0, before = 0;
    for (int q = 0; q < ranks; ++q) {
      if (q == rank) before = all;
      all += s.counts[q];
    }
    if (all > kCandidates) return kCandidates + 1;
    if (rank > 0) {
      uint64_t* list = peer(s.list, 0) + before;
      for (int i = threadIdx.x; i < (int)mine; i += kThreads) list[i] = s.list[i];
    }
    cluster.sync();
    return (int)all;
  }
  // List all elements with depth_of(l) < bins (bins <= kBins) at rank 0; returns how many there are, in the whole cluster (kCandidates + 1: more).
  template <typename F> __device__ int list_above(const F& depth_of, float unit, int bins) {
    // most are far below: one comparison with a bound that is safely too low
    float bound = bins < kBins ? r.top - (float)bins / unit * 1.0001f - fabsf(r.top) * 1e-6f : -INFINITY;
    if (isnan(bound)) bound = -INFINITY;  // (the largest is infinite)
    r.template each<true>([&](float l, int i) {
      if (l >= bound && (bins >= kBins || (int)depth_of(l) < bins)) {
        const uint32_t at = atomicAdd(&s.listed[2], 1u);
        if (at < kCandidates) s.list[at] = place_of(l, i);
      }
    });
    return collected();
  }
  // Bins 0 .. of which hold at least k of two logits a thread, its largest and that of another group of 16 bytes: what top_k keeps is in them.
  __device__ int bins_of_top(float mine, float second, bool any, int k) {
    auto depth_of = [&](float l) { return l == r.top ? 0.f : fminf((r.top - l) * kTopBins, (float)(kBins - 1)); };
    if (any) atomicAdd(&s.hist[(int)depth_of(mine)], 1u);
    if (second > -INFINITY) atomicAdd(&s.hist[(int)depth_of(second)], 1u);
    if (threadIdx.x == 0) s.last_bin = kBins;  // (fewer than k: everything)
    cluster.sync();
    uint32_t n = 0;
    for (int q = 0; q < ranks; ++q) n += *peer(&s.hist[threadIdx.x], q);
    uint64_t total;
    const uint64_t before = block_before((uint64_t)n, s.words, &total);
    if (n > 0 && before < (uint64_t)k && before + n >= (uint64_t)k) s.last_bin = threadIdx.x + 1;
    __syncthreads();
    const int bins = s.last_bin;
    return bins;
  }
  // Bins 0 .. that hold what top_p keeps, by sums to kSumError; *mass: the sum of all weights, as exactly; *elements: in these bins.
  __device__ int bins_of_mass(double top_p, float unit, double* mass, long long* elements) {
    const float log2_scale = (float)(r.scale / 64.0);
    auto depth_of = [&](float l) { return l == r.top ? 0.f : fminf((r.top - l) * unit, (float)(kBins - 1)); };
    const float top = r.top == INFINITY ? 3.4028235e38f : r.top;  // (differences without NaN)
    const float near = top - (float)(kBins - 1) / unit * 1.0001f - fabsf(top) * 1e-6f;
    float w = 0.f;
    double sum = 0.0;
    int n_w = 0;
    r.template each_group<true>([&](const float (&l)[Row<T>::N], int n, int) {
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) {
        if (e >= n) break;
        float x;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"((l[e] - top) * log2_scale));
        w += x;
        if (l[e] >= near) {
          const float d = depth_of(l[e]);
          if (d < (float)(kBins - 1)) {
            const int b = (int)d;
            atomicAdd(&s.hist[b], 1u);
            atomicAdd(&s.inner[b], (uint32_t)((d - (float)b) * parts));
          }
        }
      }
      if (++n_w == 8) {  // (no more than 64 terms in fp32)
        sum += (double)w;
        w = 0.f;
        n_w = 0;
      }
    });
    give(sum + (double)w);
    cluster.sync();
    *mass = taken();
    uint32_t n = 0, inner = 0;
    for (int q = 0; q < ranks; ++q) {
      n += *peer(&s.hist[threadIdx.x], q);
      inner += *peer(&s.inner[threadIdx.x], q);
    }
    // at least so much weight is in the bins up to this one
    double total;
    const double low = (double)n * (double)exp2f(-(float)(threadIdx.x + 1) * (1.4427f / kNearBins)) * (1.0 - 1e-4);
    const double before = block_before(threadIdx.x < kBins - 1 ? low : 0.0, s.sums, &total);
    if (threadIdx.x == 0) s.last_bin = kBins;
    __syncthreads();
    const double limit = top_p * *mass * (1.0 + 4.0 * (double)kSumError);
    if (threadIdx.x < kBins - 1 && before + low >= limit) atomicMin(&s.last_bin, (int)threadIdx.x + 1);
    __syncthreads();
    const int bins = s.last_bin;
    uint64_t in;
    block_before((uint64_t)((int)threadIdx.x < bins ? n : 0), s.words, &in);
    *elements = (long long)in;
    count = (int)threadIdx.x < bins ? n : 0;
    inner_count = inner;
    return bins;
  }
  // The border of top_p where the kept are too many for a list: from the bins of bins_of_mass those that it can be in, whose elements are
  // listed, in the pass that sums all weights and those above in 64 bits.  False: too many even so.
  __device__ bool near_border(double top_p, float unit, double mass, uint64_t* place) {
    mean_bounds(inner_count, kNearBins);
    find_bins(true, top_p * mass, 0, 0, 0.0, 4.0 * (double)kSumError);
    const int first_bin = min(s.first_bin, s.last_bin), last_bin = s.last_bin;
    const uint64_t in = (int)threadIdx.x < first_bin ? (uint64_t)count : (int)threadIdx.x <= last_bin ? (uint64_t)count << 32 : 0;
    uint64_t both;
    block_before(in, s.words, &both);
    if ((both >> 32) > kCandidates) return false;
    const float above = (float)first_bin, below = (float)(last_bin + 1);
    double sum = 0.0, ahead = 0.0;
    each_weight(r, [&](double w, float l, int i) {
      sum += w;
      const float d = fminf((r.top - l) * unit, (float)(kBins - 1));  // (NaN: both are infinite)
      if (!(d >= above)) {
        ahead += w;
      } else if (d < below) {
        const uint32_t at = atomicAdd(&s.listed[2], 1u);
        if (at < kCandidates) s.list[at] = place_of(l, i);
      }
    });
    give(sum);
    const int from_sum = turn++;
    give(ahead);
    const int n_list = collected();  // (its barriers stand between giving and taking)
    ahead = taken();
    sum = 0.0;
    for (int k = 0; k < ranks; ++k) sum += s.slot[from_sum & (kSlots - 1)][k];
    if (n_list > kCandidates) return false;
    if (rank == 0) cut(n_list, false, 0, true, top_p * sum, (long long)(both & 0xffffffffu), ahead);
    cluster.sync();
    *place = s.border;
    return true;
  }
  // Histograms anew, for the way in steps.
  __device__ void clear_bins() {
    cluster.sync();  // (nobody reads them any more)
    s.hist[threadIdx.x] = s.inner[threadIdx.x] = 0;
    __syncthreads();
  }

  // Which bins can the border be in?  -> s.first_bin, s.last_bin (of the places behind `above` elements with the weights above_mass)
  __device__ void find_bins(bool by_mass, double limit, long long k, long long above, double above_mass, double slack = 1e-9) {
    if (threadIdx.x == 0) {
      s.first_bin = kBins - 1;
      s.last_bin = 0;
    }
    if (!by_mass) {
      uint64_t total;
      const uint64_t before = block_before((uint64_t)count, s.words, &total);  // (its barriers stand behind the two stores)
      if (count > 0 && (long long)before + above < k && (long long)(before + count) + above >= k) s.first_bin = s.last_bin = threadIdx.x;
    } else {
      double total;
      const double low_before = above_mass + block_before(count * low_w, s.sums, &total);
      const double high_before = above_mass + block_before(count * high_w, s.sums, &total);
      // kept for certain: all of a bin whose weights with those before it stay below the limit; left out for certain: low_before >= limit
      if (count > 0 && low_before * (1.0 - slack) < limit) {
        if ((high_before + count * high_w) * (1.0 + slack) >= limit) atomicMin(&s.first_bin, (int)threadIdx.x);
        atomicMax(&s.last_bin, (int)threadIdx.x);
      }
    }
    __syncthreads();
  }

  // Sorts s.list[0 .. n), the largest first, zeros behind them.  The upper half of an entry: LOGITS: the key of a logit, else ~index.
  template <bool LOGITS> static __device__ __noinline__ void sort_list(SampleShared& s, int n_list, int vocab) {
    const int t = threadIdx.x;
    __syncthreads();
    if (n_list <= kThreads / 8) {
      // Few: eight threads count how many of the others are larger than one of them (no two are equal but zeros).  (top_k = 50: 14.7 us,
      // 16.7 through the bins below.)
      const uint64_t mine = (t >> 3) < n_list ? s.list[t >> 3] : 0;
      int larger = 0;
      for (int j = t & 7; j < n_list; j += 8) larger += s.list[j] > mine;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) larger += __shfl_xor_sync(kAll, larger, o);
      __syncthreads();
      if (t < kThreads / 8) s.list[t] = 0;
      __syncthreads();
      if ((t & 7) == 0 && mine) s.list[larger] = mine;
      __syncthreads();
      return;
    }
    // More: into bins that are even between the smallest and the largest, and counted within them as long as they hold few.
    // (top_k = 1000 of 151936 fp32 logits, both sorts in it: 24 us like this, 46 by sort_by_steps.)
    const uint64_t x[2] = {t < n_list ? s.list[t] : 0, t + kThreads < n_list ? s.list[t + kThreads] : 0};
    const uint32_t a = x[0] >> 32, b = x[1] >> 32;
    const uint32_t most = __reduce_max_sync(kAll, max(a, b)), least = __reduce_min_sync(kAll, min(x[0] ? a : ~0u, x[1] ? b : ~0u));
    if (t == 0) s.range[0] = 0, s.range[1] = ~0u;
    s.hist[t] = 0;
    __syncthreads();
    if ((t & 31) == 0) {
      atomicMax(&s.range[0], most);
      atomicMin(&s.range[1], least);
    }
    __syncthreads();
    const uint32_t hi = s.range[0], lo = s.range[1];
    auto below = [&](uint32_t v) -> float { return LOGITS ? logit_of(hi) - logit_of(v) : (float)(hi - v); };
    const float per = (float)(kBins - 1) / below(lo);
    // 16-bit logits that are next to each other: a bin is one value, or part of the indices of one.
    constexpr int kZeros = sizeof(T) == 4 ? 0 : __is_same(T, __half) ? 13 : 16;  // low bits that all keys have in common
    const uint32_t values = ((hi - lo) >> kZeros) + 1, parts = kBins / values;
    const bool by_value = LOGITS && kZeros && values <= kBins / 2;
    const float per_index = (float)parts / (float)vocab;
    int bin[2], at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (does not fall from one place to the next; 0 where the range is not finite)
      bin[h] = by_value ? (int)(((hi - (uint32_t)(x[h] >> 32)) >> kZeros) * parts + min(parts - 1, (uint32_t)((float)(uint32_t)~(uint32_t)x[h] * per_index)))
                        : min(kBins - 1, (int)(below(x[h] >> 32) * per));
      if (x[h]) at[h] = (int)atomicAdd(&s.hist[bin[h]], 1u);
    }
    __syncthreads();
    const uint32_t mine = s.hist[t];
    uint64_t total;
    const uint64_t before = block_before((uint64_t)mine, s.words, &total);
    if (__syncthreads_or(mine > 64)) {
      sort_by_steps(s, n_list);
      return;
    }
    s.inner[t] = (uint32_t)before;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (x[h]) s.list[s.inner[bin[h]] + at[h]] = x[h];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at[h] = 0;
      if (!x[h]) continue;
      const int i0 = (int)s.inner[bin[h]], n = (int)s.hist[bin[h]];
      at[h] = i0;
      for (int j = i0; j < i0 + n; ++j) at[h] += s.list[j] > x[h];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (x[h]) s.list[at[h]] = x[h];
      if (t + h * kThreads >= n_list) s.list[t + h * kThreads] = 0;
    }
    __syncthreads();
  }
  static __device__ __noinline__ void sort_by_steps(SampleShared& s, int n_list) {
    const int t = threadIdx.x;
    int n = kThreads / 4;
    while (n < n_list) n <<= 1;
    uint64_t x0 = t < n_list ? s.list[t] : 0, x1 = t + kThreads < n_list ? s.list[t + kThreads] : 0;
    if (n <= kThreads) {
      sort_steps<false>(s, x0, x1, n);
    } else {
      sort_steps<true>(s, x0, x1, n);
    }
    __syncthreads();
    s.list[t] = x0;
    s.list[t + kThreads] = x1;
    __syncthreads();
  }
  template <bool BOTH> static __device__ __forceinline__ void sort_steps(SampleShared& s, uint64_t& x0, uint64_t& x1, int n) {
    const int t = threadIdx.x;
    // the earlier of two places takes the larger where the run falls, else the smaller
    auto pick = [](uint64_t x, uint64_t y, bool larger) { return larger == (x > y) ? x : y; };
#pragma unroll 1
    for (int size = 2; size <= n; size <<= 1) {
      const bool down0 = (t & size) == 0, down1 = ((t + kThreads) & size) == 0;
#pragma unroll 1
      for (int step = size >> 1; step > 0; step >>= 1) {
        const bool first = (t & step) == 0;
        uint64_t y0, y1 = 0;
        if (step == kThreads) {  // (both are this thread's)
          const uint64_t a = max(x0, x1);
          x1 = min(x0, x1);
          x0 = a;
          continue;
        }
        if (step >= 32) {
          __syncthreads();
          s.list[t] = x0;
          if (BOTH) s.list[t + kThreads] = x1;
          __syncthreads();
          y0 = s.list[t ^ step];
          if (BOTH) y1 = s.list[(t ^ step) + kThreads];
        } else {
          y0 = __shfl_xor_sync(kAll, (unsigned long long)x0, step);
          if (BOTH) y1 = __shfl_xor_sync(kAll, (unsigned long long)x1, step);
        }
        x0 = pick(x0, y0, first == down0);
        if (BOTH) x1 = pick(x1, y1, first == down1);
      }
    }
  }
  // Sum of the values ahead of each of a thread's two, in the order of the sorted numbers.
  __device__ __forceinline__ void before_both(const double (&w)[2], int n, double (&before)[2], double* total) {
    double first, second = 0.0;
    before[0] = block_before(w[0], s.sums, &first);
    if (n > kThreads) {
      before[1] = first + block_before(w[1], s.sums, &second);
    } else {
      before[1] = first;
    }
    *total = first + second;
  }

  // The draw from the sorted list alone (rank 0): it holds all that can be kept.  Without top_k, `mass` is the sum of all weights to
  // `error`, relative; false where that leaves the border open.
  __device__ bool draw(int n_list, bool by_k, int k, bool by_mass, double top_p, double mass, double error, float min_p, double u, int64_t* token, float* logprob) {
    const int t = threadIdx.x;
    sort_list<true>(s, n_list, r.vocab);
    const uint64_t place[2] = {t < n_list ? s.list[t] : 0, t + kThreads < n_list ? s.list[t + kThreads] : 0};
    bool keep[2], open = false;
    double w[2], before[2], total;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = t + h * kThreads;
      keep[h] = at < n_list && (!by_k || at < k);
      w[h] = keep[h] ? r.weight(logit_of((uint32_t)(place[h] >> 32))) : 0.0;
    }
    before_both(w, n_list, before, &total);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = t + h * kThreads;
      if (by_mass) {
        const double limit = top_p * (by_k ? total : mass), slack = error * limit;
        open = open || (keep[h] && at > 0 && before[h] > limit - slack && before[h] < limit + slack);
        // (a list that ends below the limit does not hold the border)
        open = open || (!by_k && at == 0 && total < limit + slack && n_list < r.vocab);
        keep[h] = keep[h] && (before[h] < limit || at == 0);
      }
      keep[h] = keep[h] && w[h] > 0.0 && w[h] >= (double)min_p;
      s.weights[at] = w[h];
    }
    if (__syncthreads_or(open)) return false;
    // the kept ones in the order of the index
#pragma unroll
    for (int h = 0; h < 2; ++h) s.list[t + h * kThreads] = keep[h] ? (place[h] & 0xffffffffu) << 32 | (uint32_t)(t + h * kThreads + 1) : 0;
    // (what is kept is the beginning of the sorted list)
    const int kept = __syncthreads_count(keep[0]) + (n_list > kThreads ? __syncthreads_count(keep[1]) : 0);
    sort_list<false>(s, kept, r.vocab);
    const uint64_t by_index[2] = {t < kept ? s.list[t] : 0, t + kThreads < kept ? s.list[t + kThreads] : 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = t + h * kThreads < kept ? s.weights[(uint32_t)by_index[h] - 1] : 0.0;
    before_both(w, n_list, before, &total);
    const double goal = u * total;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (t + h * kThreads < kept && before[h] + w[h] > goal) atomicMin(&s.first_bin, t + h * kThreads);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (t + h * kThreads == min(s.first_bin, kept - 1)) {
        *token = (int64_t)(uint32_t)~(uint32_t)(by_index[h] >> 32);
        if (logprob) *logprob = (float)log(w[h] / total);
      }
    return true;
  }

  // The border among `n_list` sorted candidates, by rank 0; `above` elements with the weights `mass` stand before them.  by_k: the first k
  // of the order are kept; by_mass: those before which less than `limit` lies, with by_k less than limit times the first k's weights.
  __device__ void cut(int n_list, bool by_k, long long k, bool by_mass, double limit, long long above, double mass) {
    const int t = threadIdx.x;
    sort_list<true>(s, n_list, r.vocab);
    const uint64_t place[2] = {t < n_list ? s.list[t] : 0, t + kThreads < n_list ? s.list[t + kThreads] : 0};
    if (t == 0) s.last_kept = 0;
    bool keep[2];
    double w[2], before[2], total;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = t + h * kThreads;
      keep[h] = at < n_list && (!by_k || above + at < k);
      w[h] = keep[h] ? r.weight(logit_of((uint32_t)(place[h] >> 32))) : 0.0;
    }
    before_both(w, n_list, before, &total);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = t + h * kThreads;
      before[h] += mass;
      if (by_mass) keep[h] = keep[h] && (before[h] < (by_k ? limit * (mass + total) : limit) || above + at == 0);
      if (keep[h]) atomicMax(&s.last_kept, at);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (t + h * kThreads == s.last_kept)
        for (int q = 0; q < ranks; ++q) {
          *peer(&s.border, q) = place[h];
          *peer(&s.border_mass, q) = before[h] + w[h];
        }
  }

  // The last place that is kept.  Linear bins first; by_k: the k-th, and with by_mass that of top_p = `limit` among them where one list
  // holds them all (*both says so); by_mass alone: weights before it < limit.  *kept: the weights up to and with it.
  __device__ uint64_t border(bool by_k, long long k, bool by_mass, double limit, double* kept, bool* both) {
    uint64_t lo = 0, hi = ~0ull;     // places of the candidates
    long long above = 0;             // elements before them
    double above_mass = 0.0;
    long long left = r.vocab;        // candidates
    bool linear = true;
    int shift = 0;
    *both = false;
    for (;;) {
      find_bins(!by_k, limit, k, above, above_mass);
      int first_bin = min(s.first_bin, s.last_bin);
      const int last_bin = s.last_bin;
      uint64_t candidates, ahead;
      {
        // both counts in one sum: 2^32 a half
        const uint64_t mine = (int)threadIdx.x < first_bin ? (uint64_t)count : (int)threadIdx.x <= last_bin ? (uint64_t)count << 32 : 0;
        uint64_t total;
        block_before(mine, s.words, &total);
        candidates = total >> 32;
        ahead = total & 0xffffffffu;
      }
      if (linear && by_k && candidates + ahead <= kCandidates) {  // all of the first k in one list
        candidates += ahead;
        ahead = 0;
        first_bin = 0;
        *both = true;
      }
      above += (long long)ahead;
      // the weights above the candidates, and the candidates themselves or their range
      const bool few = candidates <= kCandidates;
      uint32_t* listed = peer(&s.listed[turn & 1], 0);
      uint64_t* list = peer(s.list, 0);
      double mass = 0.0;
      uint64_t my_lo = ~0ull, my_hi = 0;
      r.each([&](float l, int i) {
        const uint64_t place = place_of(l, i);
        if (place < lo || place > hi) return;
        const int b = linear ? (int)depth(l) : (int)((hi - place) >> shift);
        if (b < first_bin) {
          mass += r.weight(l);
        } else if (b <= last_bin) {
          if (few) list[atomicAdd(listed, 1u)] = place;
          my_lo = min(my_lo, place);
          my_hi = max(my_hi, place);
        }
      });
      give(mass);
      if (!few) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          my_lo = min(my_lo, (uint64_t)__shfl_xor_sync(kAll, (unsigned long long)my_lo, o));
          my_hi = max(my_hi, (uint64_t)__shfl_xor_sync(kAll, (unsigned long long)my_hi, o));
        }
        if (threadIdx.x < 2) s.words[threadIdx.x] = threadIdx.x ? 0 : ~0ull;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
          atomicMin((unsigned long long*)&s.words[0], (unsigned long long)my_lo);
          atomicMax((unsigned long long*)&s.words[1], (unsigned long long)my_hi);
        }
        __syncthreads();
        if ((int)threadIdx.x < ranks) {
          *peer(&s.lo[rank], threadIdx.x) = s.words[0];
          *peer(&s.hi[rank], threadIdx.x) = s.words[1];
        }
      }
      cluster.sync();
      above_mass += taken();
      if (few) {
        if (rank == 0) {
          if (threadIdx.x == 0) s.listed[(turn - 1) & 1] = 0;  // (for the round after the next; a barrier stands between)
          cut((int)candidates, by_k, k, *both ? by_mass : !by_k, limit, above, above_mass);
        }
        cluster.sync();
        *kept = s.border_mass;
        return s.border;
      }
      // too many: their range, in 1024 parts
      lo = ~0ull;
      hi = 0;
      for (int q = 0; q < ranks; ++q) {
        lo = min(lo, s.lo[q]);
        hi = max(hi, s.hi[q]);
      }
      if (!by_k && !linear && 4 * (long long)candidates > 3 * left) {
        // bounds from the edges can leave all bins open, where logits of very different weight share one: halve the range
        const uint64_t mid = lo + ((hi - lo) >> 1);
        double w = 0.0, n = 0.0;
        r.each([&](float l, int i) {
          const uint64_t place = place_of(l, i);
          if (place <= mid || place > hi) return;
          w += r.weight(l);
          n += 1.0;
        });
        give(w);
        cluster.sync();
        w = taken();
        give(n);
        cluster.sync();
        n = taken();
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
      shift = max(0, 64 - (int)__clzll(hi - lo) - 10);
      s.hist[threadIdx.x] = 0;  // (all have read the last one: a barrier stands between)
      __syncthreads();
      r.each([&](float l, int i) {
        const uint64_t place = place_of(l, i);
        if (place >= lo && place <= hi) atomicAdd(&s.hist[(int)((hi - place) >> shift)], 1u);
      });
      cluster.sync();
      count = 0;
      for (int q = 0; q < ranks; ++q) count += *peer(&s.hist[threadIdx.x], q);
      const uint64_t first = (uint64_t)threadIdx.x << shift, last = first + ((1ull << shift) - 1);
      high_w = r.weight(logit_of((uint32_t)((first <= hi - lo ? hi - first : lo) >> 32))) * (1.0 + 1e-9);
      low_w = r.weight(logit_of((uint32_t)((last <= hi - lo ? hi - last : lo) >> 32))) * (1.0 - 1e-9);
    }
  }
};

__device__ __forceinline__ float setting(const float* per_request, float value, int r) { return per_request ? __ldg(per_request + r) : value; }

template <typename T> __global__ void __launch_bounds__(kThreads, 1) sample_kernel(const __grid_constant__ mk_sample_args a) {
  __shared__ SampleShared s;
  constexpr int N = Row<T>::N;
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int req = blockIdx.x / ranks;
  long long row = req;
  if (a.qo_indptr) {  // the last of the request's rows
    const int q0 = __ldg(a.qo_indptr + req), q1 = __ldg(a.qo_indptr + req + 1);
    row = q1 > q0 && q0 >= 0 ? q1 - 1 : -1;
  }
  if (row < 0 || row >= a.rows) {  // (the whole cluster)
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[req] = -1;
      if (a.logprobs) a.logprobs[req] = -INFINITY;
    }
    return;
  }
  const float temperature = setting(a.temperature, a.temperature_value, req);
  const float top_p = setting(a.top_p, a.top_p_value, req), min_p = fminf(setting(a.min_p, a.min_p_value, req), 1.f);  // (the largest always stays)
  const int top_k = a.top_k ? __ldg(a.top_k + req) : a.top_k_value;
  const double u = (double)__ldg(a.u + req);
  Sampler<T> d{cluster, s, {}, ranks, rank, 0};
  Row<T>& r = d.r;
  r.vocab = a.vocab;
  r.logits = (const T*)a.logits + row * a.row_stride;
  r.shift = (int)((reinterpret_cast<uintptr_t>(r.logits) & 15) / sizeof(T));
  r.power = s.power;
  const int groups = (a.vocab + r.shift + N - 1) / N, per = (groups + ranks - 1) / ranks;
  r.g0 = min(groups, rank * per);
  r.g1 = min(groups, r.g0 + per);

  // the first place
  s.hist[threadIdx.x] = s.inner[threadIdx.x] = 0;
  if (threadIdx.x < 64) s.power[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
  if (threadIdx.x < 3) s.listed[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.first_bin = 0x7fffffff;
  float top = -INFINITY, second = -INFINITY;
  int top_at = 0x7fffffff;
  r.template each_group<true>([&](const float (&l)[N], int n, int i) {
    float most = l[0];
#pragma unroll
    for (int e = 1; e < N; ++e)
      if (e < n) most = fmaxf(most, l[e]);
    second = fmaxf(second, fminf(most, top));
    if (most > top || (most == top && i < top_at)) {  // (rarely)
      top = most;
      int k = 0;
#pragma unroll
      for (int e = N - 1; e > 0; --e)
        if (e < n && l[e] == most) k = e;
      top_at = i + (l[0] == most ? 0 : k);
    }
  });
  uint64_t best = top_at == 0x7fffffff ? 0 : place_of(top, top_at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(kAll, (unsigned long long)best, o));
  if ((threadIdx.x & 31) == 0) s.words[threadIdx.x >> 5] = best;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA has begun before its shared memory is written
  best = s.words[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(kAll, (unsigned long long)best, o));
  if ((int)threadIdx.x < ranks) *d.peer(&s.hi[rank], threadIdx.x) = best;
  cluster.sync();
  best = 0;
  for (int q = 0; q < ranks; ++q) best = max(best, s.hi[q]);
  r.top = logit_of((uint32_t)(best >> 32));
  const bool nothing = r.top == -INFINITY;
  if (nothing || !(temperature > 0.f)) {  // no token can be chosen, or the greedy one is (no CTA looks into another any more)
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[req] = nothing ? -1 : (long long)(uint32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[req] = nothing ? -INFINITY : 0.f;
    }
    return;
  }
  const double inv_t = 1.0 / (double)temperature;
  r.scale = inv_t * (64.0 / 0.6931471805599453094);
  r.largest = (double)r.top;
  // (rounded up; exp(-700) is 1e-304.  With an infinite largest logit or temperature no logit, or every finite one, is plain.)
  r.plain = r.top == INFINITY ? __uint_as_float(0x7fc00000u) : fmaxf(__double2float_ru((double)r.top - 700.0 * (double)temperature), -3.4028235e38f);
  r.lowest = fmaxf(__double2float_rd((double)r.top - 760.0 * (double)temperature), -INFINITY);  // (exp(-746) is 0 in 64 bits)
  d.per_bin = (float)(kBinsPerUnit * inv_t);
  d.parts = (float)inner_parts(a.vocab);

  uint64_t least = 0;  // the border: places from here on are kept
  const bool cut_k = top_k > 0 && top_k < a.vocab, cut_p = top_p < 1.f;
  if (cut_k || cut_p) {
    double mass = 0.0;
    // the short way: a list of all that can be kept
    int listed;
    bool near = false, done = false;
    const float near_unit = (float)((double)kNearBins * inv_t);
    if (cut_k) {
      const int bins = d.bins_of_top(top, second, top_at != 0x7fffffff, top_k);
      listed = d.list_above([&](float l) { return l == r.top ? 0.f : fminf((r.top - l) * kTopBins, (float)(kBins - 1)); }, kTopBins, bins);
    } else {
      const float unit = near_unit;
      long long elements;
      const int bins = d.bins_of_mass((double)top_p, unit, &mass, &elements);
      near = bins < kBins;
      listed = near && elements <= kCandidates ? d.list_above([&](float l) { return l == r.top ? 0.f : fminf((r.top - l) * unit, (float)(kBins - 1)); }, unit, bins) : kCandidates + 1;
    }
    if (listed <= kCandidates) {
#pragma unroll 1
      for (bool exact = cut_k;; exact = true) {
        bool open = false;
        if (rank == 0) open = !d.draw(listed, cut_k, top_k, cut_p, (double)top_p, mass, exact ? 0.0 : (double)kSumError, min_p, u, a.tokens + req, a.logprobs ? a.logprobs + req : nullptr);
        if (cut_k) return;  // (no sum in fp32 is in it: the border is never open, and nobody looks into another CTA any more)
        if (rank == 0 && (int)threadIdx.x < ranks) *d.peer(&s.close, threadIdx.x) = open;
        cluster.sync();
        if (!s.close) return;
        if (exact) break;
        // too close to call (a row in a few hundred): the sum of all weights in 64 bits
        mass = 0.0;
        each_weight(r, [&](double w, float, int) { mass += w; });
        d.give(mass);
        cluster.sync();
        mass = d.taken();
      }
    }
    // the border by itself
    if (near && listed > kCandidates) done = d.near_border((double)top_p, near_unit, mass, &least);
    if (!done) {
    // the way in steps
    d.clear_bins();
    d.linear_bins(!cut_k, &mass);
    bool both = false;
    if (cut_k) {
      const uint32_t count = d.count;
      const double low = d.low_w, high = d.high_w;
      least = d.border(true, top_k, cut_p, (double)top_p, &mass, &both);
      d.count = count;
      d.low_w = low;
      d.high_w = high;
    }
    if (cut_p && !both) {
      double unused;
      least = max(least, d.border(false, 0, true, (double)top_p * mass, &unused, &both));
    }
    }
  }

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // (min_p: bounds that are safely too low and too high; between them the weight itself decides)
  const float min_at = r.top + temperature * logf(fmaxf(min_p, 1e-45f)), min_off = (fabsf(r.top) + fabsf(min_at)) * 1e-6f + temperature * 1e-3f;
  const uint32_t border_key = (uint32_t)(least >> 32);
  const float border_logit = least ? logit_of(border_key) : -INFINITY;
  const float least_logit = fmaxf(fmaxf(border_logit, r.lowest), min_p > 0.f ? min_at - min_off : -INFINITY);
  const bool never = isnan(r.plain) || (min_p > 0.f && !(min_at + min_off < INFINITY));
  // kept for certain from here on: above the border's logit
  const float sure = never || border_logit == INFINITY ? __uint_as_float(0x7fc00000u)
                                                       : fmaxf(least ? logit_of(border_key + 1) : -INFINITY, fmaxf(r.plain, min_p > 0.f ? min_at + min_off : -INFINITY));
  auto perhaps = [&](float l, int i) -> double {
    if (l < least_logit || (least != 0 && place_of(l, i) < least)) return 0.0;
    const double w = r.weight(l);
    return min_p > 0.f && w < (double)min_p ? 0.0 : w;
  };
  auto kept_sum = [&](int g) -> double {  // of a group
    float l[N];
    uint32_t outside = 0, unsure = 0;
    if (r.inside(g)) r.load(g, l);
    else outside = r.load_edge(g, l);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const double w = r.plain_weight(l[e]);
      if (l[e] >= sure) sum += w;
      else if (l[e] >= least_logit) unsure |= 1u << e;
    }
    unsure &= ~outside;
    while (unsure) {  // (at a border, or next to the smallest numbers)
      const int i = r.index(g) + __ffs(unsure) - 1;
      unsure &= unsure - 1;
      sum += perhaps(clean(to_float(r.logits[i])), i);
    }
    return sum;
  };
  // The kept weights in the order of the index: a warp has a contiguous part of the CTA's.  The CTA in which the running sum exceeds the
  // goal deals that part out to its warps again, until a lane has one group.  (One loop, so that its instructions are fetched once.)
  double goal = 0.0, total = 0.0, from = 0.0, mine, up;
  int lo = r.g0, hi = r.g1, owner;
  // the first of 32 values whose running sum exceeds the goal; where rounding leaves none, the last that is not 0; -1: all are
  auto find = [&](double v) -> int {
    up = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(kAll, up, o);
      if (lane >= o) up += x;
    }
    const unsigned over = __ballot_sync(kAll, v > 0.0 && from + up > goal), any = __ballot_sync(kAll, v > 0.0);
    const int k = over ? __ffs(over) - 1 : 31 - __clz(any);
    const double ahead = __shfl_sync(kAll, up, max(k - 1, 0));
    if (k > 0) from += ahead;
    return k;
  };
#pragma unroll 1
  for (bool first = true;; first = false) {
    const int part = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int b0 = min(hi, lo + warp * part), b1 = min(hi, b0 + part);
    mine = 0.0;
#pragma unroll 2
    for (int g = b0 + lane; g < b1; g += 32) mine += kept_sum(g);
    double sum = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    __syncthreads();
    if (lane == 0) s.sums[warp] = sum;
    __syncthreads();
    if (first) {
      const double* in_rank = s.slot[d.turn & (kSlots - 1)];
      double in_cta = s.sums[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) in_cta += __shfl_xor_sync(kAll, in_cta, o);
      if ((int)threadIdx.x < ranks) *d.peer(&s.slot[d.turn & (kSlots - 1)][rank], threadIdx.x) = in_cta;
      cluster.sync();  // the last time that a CTA touches another
      for (int q = 0; q < ranks; ++q) total += in_rank[q];
      goal = u * total;
      if (rank != find(lane < ranks ? in_rank[lane] : 0.0)) return;
    }
    owner = find(s.sums[lane]);
    if (part <= 32) break;
    lo = min(hi, lo + owner * part);
    hi = min(hi, lo + part);
  }
  if (warp != owner) return;
  const int part = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32, k = find(mine);
  if (lane != k) return;
  const int i0 = r.index(min(hi, lo + warp * part) + lane);
  int token = -1;
  double w_token = 0.0;
#pragma unroll 1
  for (int i = max(i0, 0); i < min(i0 + N, r.vocab); ++i) {
    const double w = perhaps(clean(to_float(r.logits[i])), i);
    if (!(w > 0.0)) continue;
    token = i;
    w_token = w;
    from += w;
    if (from > goal) break;
  }
  a.tokens[req] = token;
  if (a.logprobs) a.logprobs[req] = (float)log(w_token / total);
}

template <typename T> cudaError_t launch(const mk_sample_args& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // The widest cluster of which the device runs as many at once as there are rows.  (A cluster lies within a group of SMs: 16 rows on
  // clusters of 8, which take 128 of 148 SMs, need two turns: top_k = 50 of 151936 fp32 logits 30 us, 20 on clusters of 4.)
  static std::atomic<int> at_once[64][4] = {};
  int dev = 0, ranks = kMaxCluster;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) ranks = 1;
  for (int k = 3; ranks > 1; ranks >>= 1, --k) {
    if (a.vocab / ranks < 1024 || (long long)ranks * a.requests > sm_count()) continue;
    cfg.gridDim = dim3((unsigned)ranks);
    attr[0].val.clusterDim.x = (unsigned)ranks;
    if (at_once[dev][k] == 0) {
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<T>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        continue;
      }
      at_once[dev][k] = n > 0 ? n : -1;
    }
    if (a.requests <= at_once[dev][k]) break;
  }
  cfg.gridDim = dim3((unsigned)(ranks * a.requests));
  attr[0].val.clusterDim.x = (unsigned)ranks;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

}  // namespace
}  // namespace mk_serving

extern "C" int mk_sample_tokens(const mk_sample_args* args, void* stream) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "sample_tokens: null arguments");
  const mk_sample_args& a = *args;
  if ((!a.logits && a.rows != 0) || !a.u || !a.tokens) return fail(MK_E_INVALID, "sample_tokens: null pointer");  // (an empty tensor has no address)
  if (a.dtype != MK_BF16 && a.dtype != MK_F16 && a.dtype != MK_F32) return fail(MK_E_INVALID, "sample_tokens: logits are bf16, fp16 or fp32");
  if (a.requests < 0 || a.rows < 0 || a.vocab < 1) return fail(MK_E_INVALID, "sample_tokens: bad sizes");
  if (a.vocab > 0x3fffffff) return fail(MK_E_TOO_LARGE, "sample_tokens: a vocabulary of %d (up to 2^30 - 1)", a.vocab);
  if (a.requests > 0x7fffffff / kMaxCluster) return fail(MK_E_TOO_LARGE, "sample_tokens: %d requests", a.requests);
  if (!a.qo_indptr && a.rows < a.requests) return fail(MK_E_INVALID, "sample_tokens: %d rows of logits for %d requests", a.rows, a.requests);
  if (a.requests == 0) return 0;
  // A request's token is written while others are drawn, so it may share memory with nothing that they read.
  const int size = a.dtype == MK_F32 ? 4 : 2;
  const Memory used[] = {list_of("out", a.tokens, a.requests, 8), list_of("logprobs", a.logprobs, a.requests, 4),
                         {"logits", a.logits, (long long)a.vocab * size, 1, {a.rows}, {a.row_stride * size}}, list_of("u", a.u, a.requests, 4),
                         list_of("temperature", a.temperature, a.requests, 4), list_of("top_k", a.top_k, a.requests, 4), list_of("top_p", a.top_p, a.requests, 4),
                         list_of("min_p", a.min_p, a.requests, 4), list_of("qo_indptr", a.qo_indptr, a.requests + 1ll, 4)};
  if (int rc = refuse_misaligned("sample_tokens", {{"out", a.tokens, 8}, {"logprobs", a.logprobs, 4}, {"logits", a.logits, size}, {"u", a.u, 4}, {"temperature", a.temperature, 4},
                                                   {"top_k", a.top_k, 4}, {"top_p", a.top_p, 4}, {"min_p", a.min_p, 4}, {"qo_indptr", a.qo_indptr, 4}}))
    return rc;
  if (int rc = refuse_shared("sample_tokens", used, 2, sizeof used / sizeof *used)) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = a.dtype == MK_F32 ? launch<float>(a, st) : a.dtype == MK_BF16 ? launch<__nv_bfloat16>(a, st) : launch<__half>(a, st);
  return e == cudaSuccess ? 0 : fail(MK_E_CUDA, "sample_tokens: launch failed: %s", cudaGetErrorString(e));
}
