// mk_chunk_attention, many rows: chunks of a prompt.
//
// The rows of a kv head (new tokens x its q heads) are cut into tiles of 128 rows, two to a CTA, which walk together over the
// positions that they see in tiles of 128: K and V are read once per 256 rows, 4 x 128 x 128 x 128 multiplications a tile.  Bound by the
// tensor cores and, as much, by the exponentials (16 a cycle and SM: as many cycles as the products of their tile take), so both have to
// run all the time:
//   warps 0-3, 4-7   softmax of the first and the second row tile: a thread has a row, so no value crosses threads
//   warp 8           loads: Q once, then K and V tiles through a ring of five 32 KB stages; a box is as much of a page as a tile holds
//   warp 9           tcgen05.mma: S = Q K^T (both from shared memory), O += P V (P from tensor memory, V with the dims on the N side as
//                    it lies in the cache); while one row tile is in its softmax the other one's products run
// Tensor memory: S and O of both row tiles, 4 x 128 columns; P overwrites the S that it comes from, and
// its product with V begins with the first 64 positions.  O is scaled only when a
// row's maximum has grown by more than 2^8 (fp16: 2^4) over the one in use: until then weights above 1 are as good as any, the sum has them too.
// P is rounded to the type of V, which adds as much error as the rounding of the output (fp16: weights of less than 2^-25 of the
// largest are off by 2^-36 of it); everything else is fp32.
// V rows behind a request's last position are cleared in shared memory (weight 0 times NaN is NaN); pieces whose sums are not
// finite all the same are done again by exact_row.
// Few CTAs (short chunks of long requests): every row tile's positions are cut into pieces, and a second kernel merges them.
// 2048 tokens behind 6111, 32 q and 8 kv heads: 230 us in bf16 (1040 TFLOP/s), 250 in fp16, the products alone 172 (256 items take two turns of
// 148 CTAs).  A pair of tiles takes 2.0 us, the products 1.1 of it, the exponentials as much; a CTA 10 us to begin and to end, which bounds
// short walks (windows of 1024 over 7100 rows: 172 us, 196 in fp16).
// Every wait has a limit; what gives up is reported (lost_word), and nothing is under way when the CTA ends.
#include <cuda.h>

#include "mk_chunk_attention.cuh"

namespace mk_serving {
namespace {

constexpr int kTile = 128;                       // rows, and positions
constexpr int kHalfBytes = kTile * 128;          // 128 rows of 64 elements, 128-byte swizzle
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kStages = 5;
constexpr int kTileThreads = 320, kLoadWarp = 8, kMmaWarp = 9;
constexpr int kSmemBytes = 2 * kStageBytes + kStages * kStageBytes + 256;
constexpr int kTries = 16;
constexpr unsigned long long kWaitNs = 2000000000ull;  // a wait that takes longer has lost its partner (where the caller sets no limit)
template <typename T> constexpr float kGrow = __is_same(T, __half) ? 4.f : 8.f;    // log2 of the weights that a stale maximum may lead to
template <typename T> constexpr float kLift = __is_same(T, __half) ? 11.f : 0.f;   // log2 of what they are carried larger by

struct TileParams {
  AttnParams p;
  CUtensorMap q, k, v;
  int tokens_per_tile;  // 128 / q heads of a kv head
  int box;              // positions of a box of K or V
  bool tries;           // whether a wait tries kTries times before it looks at the clock
  unsigned long long wait_ns;
  unsigned long long* lost;  // host memory: where a wait has run out
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// (returns at once; bar_try may sleep for a while)
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// dead: null, or the CTA's word that says which wait has run out (the address of its barrier)
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* dead, unsigned long long limit) {
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  for (;;) {
    if (bar_test(bar, parity)) return true;
    if (dead && *dead) return false;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    if (t - t0 >= limit) {
      if (dead) *dead = (int)bar;
      return false;
    }
    __nanosleep(20);
  }
}
// False once a wait of this CTA has run out: every role then leaves its loop.
__device__ __forceinline__ bool bar_wait(const TileParams& tp, uint32_t bar, uint32_t parity, volatile int* dead) {
  if (tp.tries) {
#pragma unroll 1
    for (int i = 0; i < kTries; ++i)
      if (bar_try(bar, parity)) return true;
  }
  return bar_wait_slow(bar, parity, dead, tp.wait_ns);
}
// The same by a warp: all of its lanes go on, or none.
__device__ __forceinline__ bool warp_wait(const TileParams& tp, uint32_t bar, uint32_t parity, volatile int* dead) {
  return __all_sync(kAll, bar_wait(tp, bar, parity, dead));
}
// What is under way already is waited for whatever the caller's limit is, and whether or not another wait has run out.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  if (!bar_try(bar, parity)) bar_wait_slow(bar, parity, nullptr, kWaitNs);
  __syncwarp();
}
__device__ __forceinline__ bool elect() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0u;
}
__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
               "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void load_box4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
               "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
// Descriptors of shared memory operands, 128-byte swizzle.  k contiguous: groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) { return (uint64_t)((saddr >> 4) & 0x3fffu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61); }
// The other dimension contiguous (V): 64 of its elements are a row, the next 64 are kHalfBytes further on, 8 k rows 1024 bytes.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(kHalfBytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
               "r"(add ? 1u : 0u)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "r"(add ? 1u : 0u)
               : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
#define MK_R8(b) "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), "=r"(r[b + 6]), "=r"(r[b + 7])
#define MK_I8(b) "r"(r[b]), "r"(r[b + 1]), "r"(r[b + 2]), "r"(r[b + 3]), "r"(r[b + 4]), "r"(r[b + 5]), "r"(r[b + 6]), "r"(r[b + 7])
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tm_load(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : MK_R8(0), MK_R8(8), MK_R8(16), MK_R8(24)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_load16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : MK_R8(0), MK_R8(8) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MK_I8(0), MK_I8(8), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tm_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x[j] of lane k of four <-> x[k] of lane j
__device__ __forceinline__ void transpose(uint32_t (&x)[4][4], int lane) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & o) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the lane below gives its upper one and gets the other's lower one
        const bool upper = lane & o;
        const uint32_t y = __shfl_xor_sync(kAll, upper ? x[j][e] : x[j | o][e], o);
        if (upper) x[j][e] = y; else x[j | o][e] = y;
      }
    }
}

// Bit e: position first + e is seen by a row at position at, 0 <= e < 32.
__device__ __forceinline__ uint32_t seen_bits(const mk_chunk_attention_args& a, int first, int at) {
  auto below = [](long long n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << (int)n) - 1u; };  // bits 0 .. n - 1
  uint32_t bits = below((long long)at - first + 1);
  if (a.window) bits &= ~below((long long)at - a.window + 1 - first) | below((long long)a.sinks - first);
  return bits;
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads, 1) chunk_attention_tiles(const __grid_constant__ TileParams tp) {
  const AttnParams& p = tp.p;
  const mk_chunk_attention_args& a = p.a;
  extern __shared__ __align__(1024) unsigned char raw[];  // (the swizzle's groups of 8 rows)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the row kernel takes the SMs as they become free
  // The CTA's rows.  CTAs that begin late should have little to do: of up to 32 requests the one with most positions comes first, else the last
  // of the batch (a warp's lanes hold the requests), and of its rows the last (6 chunks of 90 to 333 tokens behind 330 to 1900 cached: 59 us, 63 in the
  // order of the batch; more than 32 requests have not been tried).
  const int pieces = a.kv_heads * p.splits, tokens = 2 * tp.tokens_per_tile;
  const int slot = (int)(blockIdx.x / pieces), piece = blockIdx.x % pieces;
  const int kv_head = piece % a.kv_heads, split = piece / a.kv_heads;
  Request q;
  long long first;  // of the request's rows
  if (a.requests <= 32) {
    q = request_of(a, min(lane, a.requests - 1));
    const int slots = lane < a.requests && (long long)q.n * p.per_kv > p.few_rows ? (q.n + tokens - 1) / tokens : 0;
    int ahead = 0;
    for (int j = 0; j < a.requests; ++j) {
      const int len = __shfl_sync(kAll, q.len, j), many = __shfl_sync(kAll, slots, j);
      if (len > q.len || (len == q.len && j < lane)) ahead += many;
    }
    const unsigned owner = __ballot_sync(kAll, slot >= ahead && slot < ahead + slots);
    if (!owner) return;
    const int r = __ffs(owner) - 1;
    first = (long long)__shfl_sync(kAll, ahead + slots - 1 - slot, r) * tokens;
    q.q0 = __shfl_sync(kAll, q.q0, r);
    q.n = __shfl_sync(kAll, q.n, r);
    q.len = __shfl_sync(kAll, q.len, r);
    q.kv0 = __shfl_sync(kAll, q.kv0, r);
  } else {
    const int last = (int)(gridDim.x / pieces) - 1 - slot;
    auto base = [&](int r) { return (long long)(min(max(__ldg(a.qo_indptr + r), 0), a.tokens) / tokens + r); };
    const int r = find_owner_warp(a.requests, last, base);
    q = request_of(a, r);
    first = (last - base(r)) * tokens;
    if (first < 0 || first >= q.n || (long long)q.n * p.per_kv <= p.few_rows) return;
  }
  const int t0 = (int)first, live = min(tokens, q.n - t0);  // new tokens of this CTA
  const bool two = live > tp.tokens_per_tile;
  const Span<kTile> span(a, q.len - q.n + t0, q.len - q.n + t0 + live - 1);
  const int k0 = (int)((long long)span.count * split / p.splits), k1 = (int)((long long)span.count * (split + 1) / p.splits);
  const int n = k1 - k0;

  const uint32_t smem = smem_addr(raw);
  const uint32_t sq = smem, skv = smem + 2 * kStageBytes, bars = skv + kStages * kStageBytes;
  const uint32_t q_full = bars, tail_full = bars + 8, s_full = bars + 16, p_full = bars + 32, o_full = bars + 64, kv_full = bars + 80, kv_empty = kv_full + 8 * kStages;
  const uint32_t tm_slot = kv_empty + 8 * kStages, done = tm_slot + 16;
  volatile int* dead = reinterpret_cast<volatile int*>(raw + (tm_slot + 8 - smem));
  if (tid == 32 * kLoadWarp) {
    bar_init(q_full, 1);
    bar_init(tail_full, 1);
    bar_init(done, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(s_full + 8 * i, 1);
      bar_init(p_full + 16 * i, kTile);      // the first half of the positions, the second
      bar_init(p_full + 16 * i + 8, kTile);
      bar_init(o_full + 8 * i, 1);
    }
    for (int i = 0; i < kStages; ++i) {
      bar_init(kv_full + 8 * i, 1);
      bar_init(kv_empty + 8 * i, 1);
    }
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tm_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp) {  // (Q needs nothing of the others)
    __syncwarp();
    if (n > 0 && elect()) {
      const uint32_t bytes = (uint32_t)(p.per_kv * tp.tokens_per_tile * 256);
      bar_expect(q_full, two ? 2 * bytes : bytes);
      for (int i = 0; i < (two ? 2 : 1); ++i)
        for (int h = 0; h < 2; ++h)
          load_box3(sq + i * kStageBytes + h * kHalfBytes, &tp.q, q_full, 64 * h, kv_head * p.per_kv, q.q0 + t0 + i * tp.tokens_per_tile);
    }
  }
  // The loads wait for nobody: their warp has set the barriers up, and tensor memory they do not use.
  uint32_t tm = 0;
  if (warp == kLoadWarp) {
    asm volatile("barrier.cta.arrive 1, %0;" ::"n"(kTileThreads) : "memory");
  } else {
    fence_before();
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(kTileThreads) : "memory");
    fence_after();
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tm) : "r"(tm_slot));
  }
  const uint32_t tm_o = tm + 256;

  if (n > 0 && warp == kLoadWarp) {
    // ---- loads
    const int boxes = kTile / tp.box;           // of a half tile: at most 16
    const int rg = lane % boxes, half = lane / boxes;
    int stage = 0, parity = 1, sent = 0;  // (the first round of empty waits passes)
    bool ok = true, cut = false;          // cut: the last tile, whose rows behind the last position are cleared, is under way or there
    for (int i = 0; i < n && ok; ++i) {
      const int start = span.position(k0 + i);
      // a page that does not exist, or a box behind the last position, has coordinate -1: zeros
      int page, in;
      locate(p, q, start + rg * tp.box, &page, &in);
      for (int v = 0; v < 2; ++v) {
        ok = warp_wait(tp, kv_empty + 8 * stage, parity, dead);
        if (!ok) break;
        // V rows behind the last position but in its box are cleared before anyone sees the tile
        const int rest = q.len - start;
        const bool tail = v == 1 && rest < kTile && rest % tp.box != 0;
        const uint32_t bar = tail ? tail_full : kv_full + 8 * stage, dst = skv + stage * kStageBytes;
        if (elect()) bar_expect(bar, kStageBytes);
        __syncwarp();
        if (half < 2) load_box4(dst + half * kHalfBytes + rg * tp.box * 128, v ? &tp.v : &tp.k, bar, 64 * half, kv_head, in, page);
        __syncwarp();
        if (tail) {  // (of the last tile alone)
          cut = true;
          ok = warp_wait(tp, tail_full, 0, dead);
          if (!ok) break;
          const int end = (rest / tp.box + 1) * tp.box;
          for (int e = lane; e < (end - rest) * 16; e += 32) {
            const uint32_t at = dst + (uint32_t)((e & 1) * kHalfBytes + (rest + (e >> 4)) * 128 + ((e >> 1) & 7) * 16);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (elect()) bar_arrive(kv_full + 8 * stage);
          __syncwarp();
        }
        ++sent;
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1;
        }
      }
    }
    // No copy may be in flight when the CTA's shared memory goes to another one.  (Those that nobody has waited for, where a wait has run out; a
    // stage that was filled again had been read, and a tile that was cut short is behind all others.)
    bar_drain(q_full, 0);
    for (int k = max(0, sent - kStages); k < sent; ++k) bar_drain(kv_full + 8 * (k % kStages), (k / kStages) & 1);
    if (cut) bar_drain(tail_full, 0);
  } else if (n > 0 && warp == kMmaWarp) {
    // ---- products
    constexpr uint32_t type = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
    constexpr uint32_t qk = (1u << 4) | (type << 7) | (type << 10) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);
    constexpr uint32_t pv = qk | (1u << 16);  // B with its other dimension contiguous
    int stage = 0, parity = 0;
    // A lane whose wait has run out goes on beside the others to the end of the round, where all of them agree to leave: agreeing on every wait
    // takes 3 % of the whole kernel's time.  What the elected lane does not have it does not multiply.
    bool ok = bar_wait(tp, q_full, 0, dead);
    auto advance = [&]() {
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    };
    auto scores = [&](int w, uint32_t k) {  // S_w = Q_w K^T
      if (elect() && ok) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = (ks >> 2) * kHalfBytes + (ks & 3) * 32;
          mma_ss(tm + 128 * w, desc_k(sq + w * kStageBytes + off), desc_k(k + off), qk, ks > 0);
        }
        commit(s_full + 8 * w);
      }
      __syncwarp();
    };
    auto sums = [&](int w, uint32_t v, bool add, int half) {  // O_w += P_w V over half of the positions
      if (elect() && ok) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const int k = 4 * half + ks;
          mma_ts(tm_o + 128 * w, tm + 128 * w + 8 * k, desc_mn(v + k * 2048), pv, add || k > 0);
        }
      }
      __syncwarp();
    };
    auto release = [&](uint32_t bar) {
      if (elect() && ok) commit(bar);
      __syncwarp();
    };
    ok = bar_wait(tp, kv_full, 0, dead) && ok;
    fence_after();
    scores(0, skv);
    if (two) scores(1, skv);
    release(kv_empty);
    advance();
    ok = __all_sync(kAll, ok);
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t v = skv + stage * kStageBytes, v_empty = kv_empty + 8 * stage;
      ok = bar_wait(tp, kv_full + 8 * stage, parity, dead);
      advance();
      const uint32_t k = skv + stage * kStageBytes, k_empty = kv_empty + 8 * stage;
      const bool more = i + 1 < n;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (w && !two) break;
        for (int half = 0; half < 2; ++half) {
          ok = bar_wait(tp, p_full + 16 * w + 8 * half, i & 1, dead) && ok;
          fence_after();
          sums(w, v, i > 0, half);
        }
        if (!more) release(o_full + 8 * w);
        if (more && w == 0) ok = bar_wait(tp, kv_full + 8 * stage, parity, dead) && ok;
        if (w == (two ? 1 : 0)) release(v_empty);
        if (more) scores(w, k);
      }
      if (more) {
        release(k_empty);
        advance();
      }
      ok = __all_sync(kAll, ok);
    }
  } else if (warp < 8 && (warp < 4 || two)) {
    // ---- softmax: a thread has a row
    const int w = warp >> 2, row = tid & 127;
    const int in_tile = row / p.per_kv, tok = w * tp.tokens_per_tile + in_tile;
    const bool mine = in_tile < tp.tokens_per_tile && tok < live;
    const int at = mine ? q.len - q.n + t0 + tok : -1;
    const int head = kv_head * p.per_kv + row - in_tile * p.per_kv;
    // positions of the tile's rows: what all of them see needs no mask
    const int at0 = q.len - q.n + t0 + w * tp.tokens_per_tile, at1 = min(at0 + tp.tokens_per_tile, q.len - q.n + t0 + live) - 1;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tm + 128 * w + lanes, to = tm_o + 128 * w + lanes;
    // Weights are exp2(score - base).  The base is a maximum of the row's scores that may lag behind: it moves when a score is more
    // than 2^kGrow above it, and no weight is lost meanwhile as long as the type holds it.  bf16 has the range of fp32, so there the
    // scores of a tile are weighed with the base that the tiles before have left, as they come out of tensor memory, and
    // their maximum moves the base for the next tile; fp16 has no such range, and its tiles are looked through first.
    // (A weight that is too large even so makes the row's sums infinite, and exact_row does it again.)
    constexpr bool kLag = __is_same(T, __nv_bfloat16);
    bool unset = mine;
    float base = 0.f, l = 0.f, top = -INFINITY;
    bool ok = true;
    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
    uint64_t sum[2] = {0, 0};
    auto hide = [&](uint32_t (&s)[32], int first) {
      const uint32_t bits = seen_bits(a, first, at);
#pragma unroll
      for (int e = 0; e < 32; ++e) s[e] = bits >> e & 1 ? s[e] : 0xff800000u;
    };
    auto largest = [&](const uint32_t (&s)[32]) -> float {
      float x = __uint_as_float(s[0]), y = __uint_as_float(s[1]);
#pragma unroll
      for (int e = 2; e < 32; e += 4) {
        x = fmaxf(fmaxf(x, __uint_as_float(s[e])), __uint_as_float(s[e + 1]));
        if (e + 2 < 32) y = fmaxf(fmaxf(y, __uint_as_float(s[e + 2])), __uint_as_float(s[e + 3]));
      }
      return fmaxf(x, y);
    };
    auto weigh = [&](const uint32_t (&s)[32], int c) {  // the weights of quarter c of a tile
      const uint64_t base2 = pair(kLift<T> - base, kLift<T> - base);
      uint32_t w16[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float2 y = unpair(fma2(pair(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale2, base2));
        const float2 x = make_float2(ex2(y.x), ex2(y.y));
        sum[e & 1] = add2(sum[e & 1], pair(x.x, x.y));
        w16[e] = pack2<T>(x.x, x.y);
      }
      tm_store16(ts + 16 * c, w16);
      if (c & 1) {  // half of the positions: their product with V can begin
        tm_wait_store();
        fence_before();
        bar_arrive(p_full + 16 * w + 4 * (c - 1));
      }
    };
    // the base of a row that has moved; what there is of the row's sums follows
    auto move_base = [&](bool sums) {
      const bool grow = top > base + kGrow<T> || (unset && top > -INFINITY);
      if (!__any_sync(kAll, grow)) return;
      const float to_base = kLift<T> != 0.f ? ceilf(top) : top;  // (a whole number, so that the lift can be taken from it without rounding)
      // (no weight yet: whatever there is, is zero.  exp2f and not ex2, which has no numbers below 2^-126: a weight of 2^127 is what the row may
      // consist of.)
      const float alpha = !grow ? 1.f : unset ? 0.f : exp2f(base - to_base);
      if (grow) {
        base = to_base;
        unset = false;
      }
      l *= alpha;
      __syncwarp();  // (loads and stores of tensor memory are a warp's together, here and behind the call)
      if (!sums) return;
      // The next columns come while these are scaled.  (fp16 rows move their base more often than bf16 ones, within a window after its first tile
      // above all, which has few positions: windows of 1024 over 7100 rows 202 us without, 196 so; 183 if it moved after 2^8, which leaves 2^7 for the lift.)
      uint32_t o[2][16];
      tm_load16(to, o[0]);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        tm_wait_load();
        if (c < 7) tm_load16(to + 16 * (c + 1), o[(c + 1) & 1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c & 1][e] = __float_as_uint(__uint_as_float(o[c & 1][e]) * alpha);
        tm_store16(to + 16 * c, o[c & 1]);
      }
    };
    for (int i = 0; i < n; ++i) {
      ok = warp_wait(tp, s_full + 8 * w, i & 1, dead);
      if (!ok) break;
      fence_after();
      const int start = span.position(k0 + i);
      const bool masked = !(start + kTile - 1 <= at0 && (a.window == 0 || start > (long long)at1 - a.window || start + kTile <= a.sinks));
      uint32_t s[2][32];
      if constexpr (kLag) move_base(i > 0);
      if (!kLag || __any_sync(kAll, unset)) {  // (kLag: the first tile; rows whose first tiles are all hidden)
        tm_load(ts, s[0]);
        tm_wait_load();
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < 3) tm_load(ts + 32 * (c + 1), s[(c + 1) & 1]);
          if (masked) hide(s[c & 1], start + 32 * c);
          mx = fmaxf(mx, largest(s[c & 1]));
          if (c < 3) tm_wait_load();
        }
        top = mx * p.scale_log2;
        tm_load(ts, s[0]);  // (for the weights)
        move_base(i > 0);
      } else {
        tm_load(ts, s[0]);
      }
      float mx = -INFINITY;
      tm_wait_load();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c < 3) tm_load(ts + 32 * (c + 1), s[(c + 1) & 1]);
        if (masked) hide(s[c & 1], start + 32 * c);
        if constexpr (kLag) mx = fmaxf(mx, largest(s[c & 1]));
        weigh(s[c & 1], c);
        if (c < 3) tm_wait_load();
      }
      if constexpr (kLag) top = mx * p.scale_log2;
      const float2 both = unpair(add2(sum[0], sum[1]));
      l += both.x + both.y;
      sum[0] = sum[1] = 0;
    }
    constexpr float kDrop = __is_same(T, __half) ? 0x1p-11f : 1.f;  // 2^-kLift
    l *= kDrop;
    const float m = l == 0.f ? -INFINITY : base;
    // ---- the rows' outputs
    if (ok && n > 0) ok = warp_wait(tp, o_full + 8 * w, 0, dead);
    fence_after();
    const long long token = (long long)q.q0 + t0 + tok;
    const size_t part = ((size_t)split * a.tokens + token) * a.q_heads + head;
    float* part_o = p.tile_partial + part * kHeadDim;
    float* part_ml = p.tile_partial + (size_t)p.splits * a.tokens * a.q_heads * kHeadDim + 2 * part;
    T* dst = mine ? (T*)a.out + token * a.out_stride[0] + (long long)head * a.out_stride[1] : nullptr;
    // Four lanes write 64 bytes of a row together, their own four rows in turn: a store of 16 bytes to 32 rows takes the
    // SM 32 cycles (windows of 1024, 7100 rows: 179 us like that, 174 like this).
    T* rows[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) rows[k] = reinterpret_cast<T*>(__shfl_sync(kAll, reinterpret_cast<unsigned long long>(dst), (lane & ~3) + k));
    bool bad = mine && !(l < 0x1p100f);  // (sums that are not finite, or with those of other pieces might not be)
    const float inv = !ok ? __uint_as_float(0x7fc00000u) : p.splits > 1 ? kDrop : l == 0.f ? 0.f : kDrop / l;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t o[32];
      __syncwarp();  // (lanes without a row, and those whose sums are not finite, have left the others below)
      if (n > 0 && ok) {
        tm_load(to + 32 * c, o);
        tm_wait_load();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0u;
      }
      float f[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        f[e] = __uint_as_float(o[e]);
        bad = bad || (mine && !isfinite(f[e]));
        f[e] *= inv;
      }
      if (p.splits > 1) {
        if (mine) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(part_o + 32 * c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        }
      } else {
        uint32_t x[4][4];  // 16 bytes of 8 dims each; then of the four rows
#pragma unroll
        for (int e = 0; e < 32; e += 2) x[e >> 3][(e >> 1) & 3] = pack2<T>(f[e], f[e + 1]);
        transpose(x, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (rows[k]) *reinterpret_cast<uint4*>(rows[k] + 32 * c + 8 * (lane & 3)) = make_uint4(x[k][0], x[k][1], x[k][2], x[k][3]);
      }
    }
    if (mine) {
      if (p.splits > 1) {
        part_ml[0] = m;
        part_ml[1] = ok ? l : __uint_as_float(0x7fc00000u);
      } else if (a.lse) {
        a.lse[token * a.lse_stride[0] + head * a.lse_stride[1]] = !ok ? __uint_as_float(0x7fc00000u) : l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      }
    }
    unsigned again = __ballot_sync(kAll, bad && ok);
    while (again) {
      const int src = __ffs(again) - 1;
      again &= again - 1;
      const int at_ = __shfl_sync(kAll, at, src), head_ = __shfl_sync(kAll, head, src);
      const long long token_ = __shfl_sync(kAll, token, src);
      float o[4], m_, l_;
      exact_row<T, kTile>(p, q, span, k0, k1, at_, token_, head_, kv_head, o, m_, l_);
      const size_t part_ = ((size_t)split * a.tokens + token_) * a.q_heads + head_;
      if (p.splits > 1) {
#pragma unroll
        for (int d = 0; d < 4; ++d) p.tile_partial[part_ * kHeadDim + 4 * lane + d] = o[d];
        if (lane == 0) {
          float* ml = p.tile_partial + (size_t)p.splits * a.tokens * a.q_heads * kHeadDim + 2 * part_;
          ml[0] = m_;
          ml[1] = l_;
        }
      } else {
        T* d_ = (T*)a.out + token_ * a.out_stride[0] + (long long)head_ * a.out_stride[1] + 4 * lane;
#pragma unroll
        for (int d = 0; d < 4; ++d) d_[d] = from_float<T>(l_ == 0.f ? 0.f : o[d] / l_);
        if (a.lse && lane == 0) a.lse[token_ * a.lse_stride[0] + head_ * a.lse_stride[1]] = l_ == 0.f ? -INFINITY : (m_ + log2f(l_)) * kLn2;
      }
    }
  }
  fence_before();
  __syncthreads();
  if (*dead) {  // a wait has run out: no product may be under way when tensor memory goes to another CTA
    if (warp == kMmaWarp) {
      fence_after();
      if (elect()) commit(done);
      __syncwarp();
      bar_drain(done, 0);
    }
    if (tid == 0) {
      *(volatile unsigned long long*)tp.lost = 1ull << 63 | (unsigned long long)((uint32_t)(*dead - (int)bars) / 8) << 32 | blockIdx.x;
      __threadfence_system();
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
  }
}

// A warp per row: its pieces in the order of the positions.
template <typename T> __global__ void __launch_bounds__(256) chunk_attention_join(const __grid_constant__ AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const mk_chunk_attention_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)a.tokens * a.q_heads;
  if (row >= rows) return;
  const int tok = (int)(row / a.q_heads), head = (int)(row - (long long)tok * a.q_heads);
  const int r = find_owner_warp(a.requests, tok, [&](int i) { return (long long)__ldg(a.qo_indptr + i); });
  const Request q = request_of(a, r);
  if (tok < q.q0 || tok >= q.q0 + q.n || (long long)q.n * p.per_kv <= p.few_rows) return;
  const float* ml = p.tile_partial + (size_t)p.splits * rows * kHeadDim;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * (s * rows + row)]);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float ms = ml[2 * (s * rows + row)], ls = ml[2 * (s * rows + row) + 1];
    const float4 x = reinterpret_cast<const float4*>(p.tile_partial + (s * rows + row) * kHeadDim)[lane];
    const float f = ms == -INFINITY ? 0.f : exp2f(ms - m);
    l += f * ls;
    o.x += f * x.x; o.y += f * x.y;
    o.z += f * x.z; o.w += f * x.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint2 v = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  *reinterpret_cast<uint2*>((T*)a.out + (long long)tok * a.out_stride[0] + (long long)head * a.out_stride[1] + 4 * lane) = v;
  if (a.lse && lane == 0) a.lse[(long long)tok * a.lse_stride[0] + (long long)head * a.lse_stride[1]] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encode_fn() {
  static Encode fn = []() -> Encode {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return (Encode)f;
  }();
  return fn;
}
bool encode(CUtensorMap* map, int dtype, int dims, const void* ptr, const cuuint64_t* size, const long long* stride, const cuuint32_t* box) {
  cuuint64_t bytes[3];
  cuuint32_t one[4] = {1, 1, 1, 1};
  for (int i = 0; i + 1 < dims; ++i) bytes[i] = (cuuint64_t)stride[i] * 2;
  return encode_fn()(map, dtype == MK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)dims, const_cast<void*>(ptr), size, bytes, box,
                     one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T> int launch(const TileParams& tp, cudaStream_t s) {
  const AttnParams& p = tp.p;
  cudaError_t e = allow_shared<chunk_attention_tiles<T>>(kSmemBytes);
  if (e != cudaSuccess) return fail(MK_E_CUDA, "chunk_attention: %s", cudaGetErrorString(e));
  const long long slots = p.a.tokens / (2 * tp.tokens_per_tile) + p.a.requests;
  chunk_attention_tiles<T><<<(unsigned)(slots * p.a.kv_heads * p.splits), kTileThreads, kSmemBytes, s>>>(tp);
  if (int rc = launched("chunk_attention")) return rc;
  if (p.splits == 1) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((long long)p.a.tokens * p.a.q_heads + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, chunk_attention_join<T>, p);
  return e == cudaSuccess ? 0 : fail(MK_E_CUDA, "chunk_attention: launch failed: %s", cudaGetErrorString(e));
}

}  // namespace

// Boxes of K and V are whole groups of 8 positions of one page; the maximum is taken ahead of the scale.  A stride of 0 or beyond 2^40
// bytes has no tensor map.
bool tiles_take(const mk_chunk_attention_args& a) {
  const int per_kv = a.q_heads / a.kv_heads;
  if (a.page_size % 8 || per_kv > kTile || !(a.scale > 0.f) || !(a.scale < INFINITY)) return false;
  auto fits = [](long long s) { return s > 0 && s < (1ll << 39); };
  for (int i = 0; i < 3; ++i)
    if (!fits(a.k_cache_stride[i]) || !fits(a.v_cache_stride[i])) return false;
  return fits(a.q_stride[0]) && fits(a.q_stride[1]);
}

int launch_tile_attention(const AttnParams& p, cudaStream_t s) {
  const mk_chunk_attention_args& a = p.a;
  TileParams tp = {};
  tp.p = p;
  tp.tokens_per_tile = kTile / p.per_kv;
  tp.wait_ns = a.wait_ns ? (unsigned long long)a.wait_ns : kWaitNs;
  tp.tries = tp.wait_ns >= 100000;  // (so many take some microseconds)
  if (!(tp.lost = lost_word())) return fail(MK_E_CUDA, "chunk_attention: no pinned host memory for the kernel's status");
  tp.box = a.page_size & -a.page_size;
  if (tp.box > kTile) tp.box = kTile;
  if (!encode_fn()) return fail(MK_E_CUDA, "chunk_attention: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t q_size[3] = {kHeadDim, (cuuint64_t)a.q_heads, (cuuint64_t)a.tokens};
  const long long q_stride[2] = {a.q_stride[1], a.q_stride[0]};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)p.per_kv, (cuuint32_t)tp.tokens_per_tile};
  const cuuint64_t kv_size[4] = {kHeadDim, (cuuint64_t)a.kv_heads, (cuuint64_t)a.page_size, (cuuint64_t)a.pages};
  const long long k_stride[3] = {a.k_cache_stride[2], a.k_cache_stride[1], a.k_cache_stride[0]}, v_stride[3] = {a.v_cache_stride[2], a.v_cache_stride[1], a.v_cache_stride[0]};
  const cuuint32_t kv_box[4] = {64, 1, (cuuint32_t)tp.box, 1};
  if (!encode(&tp.q, a.dtype, 3, a.q, q_size, q_stride, q_box) || !encode(&tp.k, a.dtype, 4, a.k_cache, kv_size, k_stride, kv_box) ||
      !encode(&tp.v, a.dtype, 4, a.v_cache, kv_size, v_stride, kv_box))
    return fail(MK_E_CUDA, "chunk_attention: no tensor map for these shapes and strides");
  return a.dtype == MK_BF16 ? launch<__nv_bfloat16>(tp, s) : launch<__half>(tp, s);
}

}  // namespace mk_serving
