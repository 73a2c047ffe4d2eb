// mk_chunk_attention: entry point, the kernel for few rows and the merge of its pieces.  (The kernel for many rows: mk_chunk_attention_tiles.cu.)
//
// Few rows (one new token per request up to short chunks).  The rows of a kv head (new tokens x its q heads) are cut into groups
// of 8 or 16; a group has to walk over all K and V rows that it sees, 512 bytes and 4 x 128 x 8 multiplications a position:
// bound by HBM as long as all SMs stream evenly.  So the unit of work is a tile of 16 positions of a group, and all units of
// the batch are dealt out as contiguous ranges of equal length to warps, whatever the requests' lengths are: no synchronisation while
// the data streams, and one long request among short ones takes no longer than the sum says.  A warp that holds a group's whole
// range writes its outputs; pieces of a group are joined in shared memory by the CTA when its warps are done, and what is left of groups
// that several CTAs have worked on by a second kernel, both in the order of the positions.  K and V tiles come by 16-byte
// cp.async into a ring of the warp's own, two tiles ahead of the sums and across the border between two groups.
// 64 requests of 90 to 2200 positions, 8 kv heads: 57 us, 5.3 TB/s of 6.5 that a copy reaches; 4 of 20000 to 32700, 4 kv heads: 44 us, 4.9
// TB/s.  A bare cp.async stream of this shape reaches 6.0 to 6.2; the rest is the ring's filling, the last CTA and the merge.
// (CTAs taking a group's tiles with all warps in turn, joined after every group: 46 us like this for long contexts, but twice the
// time for short ones, 123 and 62 us, where what begins and ends a group is longer than the ring covers.)
//
// S = Q K^T with the rows on the M side of mma.m16n8k16, then O^T += V^T P^T with 16 dims on M, for which the scores are the B
// operand as they are.  P enters as the sum of two 16-bit values (their product with V is cheap here, and the rounding of P would
// otherwise be as large as that of the output).  A product with P = 0 is not 0 where V is not finite, so a piece whose sums are not
// finite is done again one row and position at a time, with the positions alone that the row sees.
#include "mk_chunk_attention.cuh"

namespace mk_serving {
namespace {

constexpr int kRowWarps = 8, kRowThreads = 32 * kRowWarps;
constexpr int kPos = 16;                          // positions of a tile
constexpr int kTileBytes = kPos * kHeadDim * 2;   // of K, and of V behind it
constexpr int kBegin = 4;                         // units that a group counts more than its tiles: what beginning and ending one takes
constexpr int kMaxRequests = MK_STEP_MAX_REQUESTS / 2;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void mma(float4& c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float4& c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c.x), "+f"(c.y), "+f"(c.z), "+f"(c.w) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float4& c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c.x), "+f"(c.y), "+f"(c.z), "+f"(c.w) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The groups of ROWS rows of a request and how many tiles each is counted as (the longest one's).
template <int ROWS> struct Groups {
  int groups, tiles;
  __device__ __forceinline__ Groups(const AttnParams& p, const Request& q) {
    const long long rows = (long long)q.n * p.per_kv;
    const bool mine = q.n > 0 && rows <= p.few_rows;
    groups = mine ? (int)((rows + ROWS - 1) / ROWS) : 0;
    tiles = 0;
    if (!mine) return;
    // A group without a window sees up to len positions; with one, its tokens span at most `span` positions more than the window.
    const long long span = (ROWS + p.per_kv - 1) / p.per_kv + 1;
    long long t = ((long long)q.len + kPos - 1) / kPos;
    if (p.a.window) {
      const long long w = ((long long)p.a.window + span + kPos - 1) / kPos + 2 + ((long long)p.a.sinks + kPos - 1) / kPos;
      t = t < w ? t : w;
    }
    tiles = (int)(t < 1 ? 1 : t);
  }
};

// sums of one group's rows over some positions, as the fragments that the mma leave: lane (g, t) = (lane / 4, lane % 4) holds, for the
// 16 dims of m-tile i, dims g and g + 8 of rows 2 t and 2 t + 1 (and of the rows 8 further on)
__host__ __device__ constexpr int part_floats(int rows) { return rows * kHeadDim + 2 * rows; }

// Pieces of a group being joined by a warp, for the 16 dims of one m-tile: maximum and sum of rows g (and g + 8), weighted sums as the
// fragments.  U: pieces whose loads are in flight together.
template <int NT, int U> struct Joined {
  static constexpr int ROWS = 8 * NT;
  float m[NT], l[NT];
  float4 o[NT];
  // part(q): piece q of n
  template <typename F> __device__ __forceinline__ void add(const F& part, int n_parts, int tile, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.f;
      o[n] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 1
    for (int w = 0; w < n_parts; w += U) {
      float4 x[U][NT];
      float mw[U][NT], lw[U][NT];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const float* pt = part(min(w + k, n_parts - 1));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          x[k][n] = reinterpret_cast<const float4*>(pt)[(n * 8 + tile) * 32 + lane];
          mw[k][n] = pt[ROWS * kHeadDim + 8 * n + g];
          lw[k][n] = pt[ROWS * kHeadDim + ROWS + 8 * n + g];
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top = m[n];
#pragma unroll
        for (int k = 0; k < U; ++k) top = fmaxf(top, mw[k][n]);
        const float base = top == -INFINITY ? 0.f : top;
        float f = exp2f(m[n] - base);
        m[n] = top;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (w + k >= n_parts) break;
          // (a piece that saw nothing of a row has weight 0 and finite sums; a NaN score has left its mark in l)
          const float fx = exp2f(mw[k][n] - base);
          l[n] = l[n] * f + lw[k][n] * fx;
          const float a0 = __shfl_sync(kAll, f, 8 * t), a1 = __shfl_sync(kAll, f, 8 * t + 4), b0 = __shfl_sync(kAll, fx, 8 * t), b1 = __shfl_sync(kAll, fx, 8 * t + 4);
          const float4& y = x[k][n];
          o[n].x = o[n].x * a0 + b0 * y.x; o[n].y = o[n].y * a1 + b1 * y.y;
          o[n].z = o[n].z * a0 + b0 * y.z; o[n].w = o[n].w * a1 + b1 * y.w;
          f = 1.f;
        }
      }
    }
  }
  __device__ __forceinline__ void store(float* pt, int tile, int lane) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      reinterpret_cast<float4*>(pt)[(n * 8 + tile) * 32 + lane] = o[n];
      if (tile == 0 && (lane & 3) == 0) {
        pt[ROWS * kHeadDim + 8 * n + (lane >> 2)] = m[n];
        pt[ROWS * kHeadDim + ROWS + 8 * n + (lane >> 2)] = l[n];
      }
    }
  }
  // The rows of `rec`: outputs and logarithms of the sums.
  template <typename T> __device__ __forceinline__ void write(const AttnParams& p, const MergeRecord& rec, int tile, int lane) const {
    const mk_chunk_attention_args& a = p.a;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
      const float i0 = __shfl_sync(kAll, inv, 8 * t), i1 = __shfl_sync(kAll, inv, 8 * t + 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * n + 2 * t + e;
        if (row >= rec.rows) continue;
        const int x = rec.row0 + row, tok = x / p.per_kv, head = rec.kv_head * p.per_kv + (x - tok * p.per_kv);
        T* dst = (T*)a.out + (long long)(rec.first_token + tok) * a.out_stride[0] + head * a.out_stride[1] + 16 * tile + g;
        dst[0] = from_float<T>((e ? o[n].y : o[n].x) * (e ? i1 : i0));
        dst[8] = from_float<T>((e ? o[n].w : o[n].z) * (e ? i1 : i0));
      }
      const int row = 8 * n + g;
      if (a.lse && tile == 0 && t == 0 && row < rec.rows) {
        const int x = rec.row0 + row, tok = x / p.per_kv, head = rec.kv_head * p.per_kv + (x - tok * p.per_kv);
        a.lse[(long long)(rec.first_token + tok) * a.lse_stride[0] + head * a.lse_stride[1]] = l[n] == 0.f ? -INFINITY : (m[n] + log2f(l[n])) * kLn2;
      }
    }
  }
};

// RING: stages of a warp, three where shared memory has the room.
template <typename T, int NT, int RING> struct RowWarp {
  static constexpr int ROWS = 8 * NT;
  static constexpr int kRing = RING;
  static constexpr float kLift = __is_same(T, __half) ? 32768.f : 1.f;  // (weights are at most 1 here; hi + lo then reach down to 2^-40)
  static constexpr int kWarpRing = kRing * 2 * kTileBytes;
  static constexpr int kPartsBytes = kRowWarps * part_floats(ROWS) * (int)sizeof(float);
  static int smem_bytes(int requests) { return kRowWarps * kWarpRing + kPartsBytes + (requests + 1) * 8; }
  // Where a warp leaves its pieces for the CTA: the first, if its group has begun in another's range, in a place of its own, the last, if
  // its group goes on, in the ring, which is done with by then.
  static __device__ __forceinline__ float* piece(unsigned char* smem, int warp, bool from_start) {
    return reinterpret_cast<float*>(from_start ? smem + warp * kWarpRing : smem + kRowWarps * kWarpRing + warp * part_floats(ROWS) * sizeof(float));
  }
  const AttnParams& p;
  const long long* first;  // first unit of every request (shared memory)
  unsigned char* smem;
  int lane, warp;

  // A piece: tiles k .. k_end of one group of one kv head; u units are behind this warp, it goes on to u_end.
  struct Cursor {
    long long u, u_end;
    Request q;
    int r, kv_head, group, k, k_end, tiles, row0, rows, p0, p1, sink, start, count;
    bool from_start, to_end;  // the piece has the group's first tile, its last
    __device__ __forceinline__ int position(int i) const { return i < sink ? i * kPos : start + (i - sink) * kPos; }
  };
  // the piece that begins at unit c.u, or behind the units of a group's beginning there: c.u is moved to its first tile
  __device__ __forceinline__ void open(Cursor& c) const {
    c.r = find_owner(p.a.requests, c.u, [&](int i) { return first[i]; });
    c.q = request_of(p.a, c.r);
    const Groups<ROWS> g(p, c.q);
    const long long in = c.u - first[c.r];
    const int item = (int)(in / (g.tiles + kBegin)), x = (int)(in - (long long)item * (g.tiles + kBegin));
    c.tiles = g.tiles;
    c.k = max(0, x - kBegin);
    c.from_start = c.k == 0;
    c.k_end = (int)min((long long)g.tiles, max(0ll, x - kBegin + (c.u_end - c.u)));
    c.to_end = c.k_end == g.tiles;
    // (a range that ends within the units of a group's beginning has none of its tiles)
    c.u = c.k_end > c.k ? c.u + max(0, kBegin - x) : c.u_end;
    c.kv_head = item / g.groups;
    c.group = item - c.kv_head * g.groups;
    c.row0 = c.group * ROWS;
    c.rows = (int)min((long long)ROWS, (long long)c.q.n * p.per_kv - c.row0);
    c.p0 = c.q.len - c.q.n + c.row0 / p.per_kv;
    c.p1 = c.q.len - c.q.n + (c.row0 + c.rows - 1) / p.per_kv;
    const Span<kPos> s(p.a, c.p0, c.p1);
    c.sink = s.sink;
    c.start = s.start;
    c.count = s.count;
  }

  // What a lane has to know of the tile that is loaded next: where a page holds whole tiles its page, else the page of position
  // lane & 15.  Looked up a tile ahead: the address waits for it.
  __device__ __forceinline__ int page_ahead(const Cursor& c) const {
    if (c.k >= c.count) return -1;
    const int pos = c.position(c.k) + (p.tile_in_page ? 0 : lane & 15);
    if (pos >= c.q.len) return -1;
    return __ldg(p.a.kv_indices + c.q.kv0 + (p.page_shift >= 0 ? pos >> p.page_shift : pos / p.a.page_size));
  }
  // K and V rows of the cursor's tile -> stage; rows that are not there become zeros
  __device__ __forceinline__ void load(const Cursor& c, int page, uint32_t stage) const {
    const mk_chunk_attention_args& a = p.a;
    const int start = c.position(c.k), live = c.k < c.count ? c.q.len - start : 0;  // rows of the tile that the request has
    const bool known = (unsigned)page < (unsigned)a.pages;
    const T* kc = (const T*)a.k_cache + c.kv_head * a.k_cache_stride[2] + (lane & 7) * 8;
    const T* vc = (const T*)a.v_cache + c.kv_head * a.v_cache_stride[2] + (lane & 7) * 8;
    auto in_page = [&](int pos) { return p.page_shift >= 0 ? pos & (a.page_size - 1) : pos % a.page_size; };
    // a lane copies 16 bytes of the rows lane / 8 + 4 j, of either half of the dims
    auto copy = [&](int j, const T* kr, const T* vr, bool there) {
      const int row = (lane >> 3) + 4 * j;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t dst = stage + (uint32_t)(row * 256 + ((((lane & 7) + 8 * half) ^ (row & 7)) << 4));
        cp_async16(dst, kr + 64 * half, there);
        cp_async16(dst + kTileBytes, vr + 64 * half, there);
      }
    };
    if (p.tile_in_page) {
      const long long pg = known ? page : 0, in = in_page(start) + (lane >> 3);
      const T *kr = kc + pg * a.k_cache_stride[0] + in * a.k_cache_stride[1], *vr = vc + pg * a.v_cache_stride[0] + in * a.v_cache_stride[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) copy(j, kr + 4 * j * a.k_cache_stride[1], vr + 4 * j * a.v_cache_stride[1], known && (lane >> 3) + 4 * j < live);
    } else {
      const bool mine = known && (lane & 15) < live;
      const long long pg = mine ? page : 0, in = mine ? in_page(start + (lane & 15)) : 0;
      const long long ko = pg * a.k_cache_stride[0] + in * a.k_cache_stride[1], vo = pg * a.v_cache_stride[0] + in * a.v_cache_stride[1];
      const unsigned there = __ballot_sync(kAll, mine);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (lane >> 3) + 4 * j;
        copy(j, kc + __shfl_sync(kAll, ko, row), vc + __shfl_sync(kAll, vo, row), there >> row & 1);
      }
    }
  }

  __device__ __forceinline__ float* slot_of(const Cursor& c) const { return piece(smem, warp, c.from_start); }
  // A group that begins here and goes on in other warps' ranges, or that has come into this CTA's from the one before: what joining
  // its pieces takes.
  __device__ __forceinline__ void leave(const Cursor& c, long long per, MergeRecord* rec) const {
    if (lane != 0) return;
    rec->last = (int)((c.u - 1 + c.tiles - c.k_end) / per);  // warp with the group's last piece (c.u: behind this one)
    rec->kv_head = c.kv_head;
    rec->row0 = c.row0;
    rec->rows = c.rows;
    rec->first_token = c.q.q0;
  }
  __device__ __forceinline__ long long row_token(const Cursor& c, int row, int* head) const {
    const int x = c.row0 + row, tok = x / p.per_kv;
    *head = c.kv_head * p.per_kv + (x - tok * p.per_kv);
    return c.q.q0 + tok;
  }

  // The piece again, a row and a position at a time.
  __device__ __noinline__ void exactly(const Cursor& c, int k0) const {
    const mk_chunk_attention_args& a = p.a;
    Span<kPos> span(a, c.p0, c.p1);
    for (int row = 0; row < c.rows; ++row) {
      int head;
      const long long tok = row_token(c, row, &head);
      float o[4], m, l;
      exact_row<T, kPos>(p, c.q, span, k0, c.k_end, c.q.len - c.q.n + (c.row0 + row) / p.per_kv, tok, head, c.kv_head, o, m, l);
      if (c.from_start && c.to_end) {
        T* dst = (T*)a.out + tok * a.out_stride[0] + head * a.out_stride[1] + 4 * lane;
#pragma unroll
        for (int d = 0; d < 4; ++d) dst[d] = from_float<T>(l == 0.f ? 0.f : o[d] / l);
        if (a.lse && lane == 0) a.lse[tok * a.lse_stride[0] + head * a.lse_stride[1]] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      } else {
        float* part = slot_of(c);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int dim = 4 * lane + d, i = dim >> 4, half = (dim >> 3) & 1, g = dim & 7, nt = row >> 3, t = (row & 7) >> 1;
          part[(((nt * 8 + i) * 32) + g * 4 + t) * 4 + half * 2 + (row & 1)] = o[d];
        }
        if (lane == 0) {
          part[ROWS * kHeadDim + row] = m;
          part[ROWS * kHeadDim + ROWS + row] = l;
        }
      }
    }
  }

  // came_in: record of the CTA's first piece, where its group has begun before; begun: of the group that this warp begins and does not end
  __device__ void run(long long u0, long long u1, long long per, MergeRecord* came_in, MergeRecord* begun) {
    const mk_chunk_attention_args& a = p.a;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * kWarpRing);
    Cursor ld, c;
    ld.u = c.u = u0;
    ld.u_end = c.u_end = u1;
    open(ld);
    c = ld;
    // The loader is kRing - 1 tiles ahead of the sums, across the border between two pieces.
    int page = page_ahead(ld);
    auto load_next = [&](int stage) {
      if (ld.u < ld.u_end) {
        load(ld, page, ring + (uint32_t)(stage * 2 * kTileBytes));
        ++ld.u;
        if (++ld.k == ld.k_end && ld.u < ld.u_end) open(ld);
        if (ld.u < ld.u_end) page = page_ahead(ld);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) load_next(i);
    int stage = 0;
    while (c.u < c.u_end) {
      // q rows as the A operand: rows g and g + 8
      uint32_t qf[8][4];
      int pos[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = g + 8 * h;
        pos[h] = -1;
        const T* qr = nullptr;
        if (h < NT && row < c.rows) {
          int head;
          const long long tok = row_token(c, row, &head);
          qr = (const T*)a.q + tok * a.q_stride[0] + head * a.q_stride[1];
          pos[h] = c.q.len - c.q.n + (c.row0 + row) / p.per_kv;
        }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qf[ks][h] = qr ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 2 * t) : 0u;
          qf[ks][h + 2] = qr ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8 + 2 * t) : 0u;
        }
      }
      float4 o[NT][8];
      float m[NT], l[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[n][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      const int k0 = c.k;
      for (; c.k < c.k_end; ++c.k, ++c.u) {
        cp_async_wait<kRing - 2>();
        __syncwarp();
        const uint32_t ks_ = ring + (uint32_t)(stage * 2 * kTileBytes), vs = ks_ + kTileBytes;
        const int fill = stage == 0 ? kRing - 1 : stage - 1;
        stage = stage == kRing - 1 ? 0 : stage + 1;
        load_next(fill);  // (the stage that the last tile left: every lane is past its reads)
        __syncwarp();     // (lanes whose position is behind the end have looked no page up; ldmatrix and mma are the warp's together)
        if (c.k >= c.count) continue;
        const int start = c.position(c.k);
        const uint32_t lrow = (uint32_t)((lane & 7) + ((lane >> 4) << 3)), lchunk = (uint32_t)((lane >> 3) & 1);
        float4 s[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t kf[4];
          ldmatrix4(ks_ + lrow * 256 + (((2 * ks + lchunk) ^ (lrow & 7)) << 4), kf);
          mma<T>(s[0], qf[ks], kf[0], kf[1]);
          mma<T>(s[1], qf[ks], kf[2], kf[3]);
        }
        float sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sc[n][0] = (n ? s[0].z : s[0].x) * p.scale_log2;
          sc[n][1] = (n ? s[0].w : s[0].y) * p.scale_log2;
          sc[n][2] = (n ? s[1].z : s[1].x) * p.scale_log2;
          sc[n][3] = (n ? s[1].w : s[1].y) * p.scale_log2;
        }
        // every live row sees the whole tile, or each its own part
        if (!(start + kPos - 1 <= c.p0 && (a.window == 0 || start > (long long)c.p1 - a.window || start + kPos <= a.sinks))) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = start + (e >> 1) * 8 + 2 * t + (e & 1);
              if (!sees(a, j, pos[n])) sc[n][e] = -INFINITY;
            }
        }
        uint32_t hi[NT][2], lo[NT][2];
        float alpha[NT];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float mx = fmaxf(fmaxf(sc[n][0], sc[n][1]), fmaxf(sc[n][2], sc[n][3]));
          mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
          const float mn = fmaxf(m[n], mx), base = mn == -INFINITY ? 0.f : mn;
          alpha[n] = m[n] == mn ? 1.f : exp2f(m[n] - base);
          moved = moved || m[n] != mn;
          m[n] = mn;
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = exp2f(sc[n][e] - base) * kLift;
          l[n] = l[n] * alpha[n] + ((w[0] + w[1]) + (w[2] + w[3]));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            hi[n][e] = pack2<T>(w[2 * e], w[2 * e + 1]);
            const float2 back = unpack2<T>(hi[n][e]);
            lo[n][e] = pack2<T>(w[2 * e] - back.x, w[2 * e + 1] - back.y);
          }
        }
        if (__any_sync(kAll, moved)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float a0 = __shfl_sync(kAll, alpha[n], 8 * t), a1 = __shfl_sync(kAll, alpha[n], 8 * t + 4);  // rows 2 t and 2 t + 1
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[n][i].x *= a0; o[n][i].y *= a1;
              o[n][i].z *= a0; o[n][i].w *= a1;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t vf[4];
          ldmatrix4t(vs + lrow * 256 + (((2 * i + lchunk) ^ (lrow & 7)) << 4), vf);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma<T>(o[n][i], vf, hi[n][0], hi[n][1]);
            mma<T>(o[n][i], vf, lo[n][0], lo[n][1]);
          }
        }
        __syncwarp();
      }
      // the piece is done
      bool bad = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor_sync(kAll, l[n], 1);
        l[n] += __shfl_xor_sync(kAll, l[n], 2);
        if constexpr (kLift != 1.f) {
          l[n] *= 1.f / kLift;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[n][i].x *= 1.f / kLift; o[n][i].y *= 1.f / kLift;
            o[n][i].z *= 1.f / kLift; o[n][i].w *= 1.f / kLift;
          }
        }
        bad = bad || !isfinite(l[n]);
#pragma unroll
        for (int i = 0; i < 8; ++i) bad = bad || !isfinite((o[n][i].x + o[n][i].y) + (o[n][i].z + o[n][i].w));
      }
      if (__any_sync(kAll, bad)) {
        const Cursor copy = c;  // (so that the cursor itself can stay in registers)
        exactly(copy, k0);
      } else if (c.from_start && c.to_end) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
          const float i0 = __shfl_sync(kAll, inv, 8 * t), i1 = __shfl_sync(kAll, inv, 8 * t + 4);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 8 * n + 2 * t + e;
            if (row >= c.rows) continue;
            int head;
            const long long tok = row_token(c, row, &head);
            T* dst = (T*)a.out + tok * a.out_stride[0] + head * a.out_stride[1] + g;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              dst[16 * i] = from_float<T>((e ? o[n][i].y : o[n][i].x) * (e ? i1 : i0));
              dst[16 * i + 8] = from_float<T>((e ? o[n][i].w : o[n][i].z) * (e ? i1 : i0));
            }
          }
          const int row = 8 * n + g;
          if (a.lse && t == 0 && row < c.rows) {
            int head;
            const long long tok = row_token(c, row, &head);
            a.lse[tok * a.lse_stride[0] + head * a.lse_stride[1]] = l[n] == 0.f ? -INFINITY : (m[n] + log2f(l[n])) * kLn2;
          }
        }
      } else {
        float* part = slot_of(c);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 8; ++i) reinterpret_cast<float4*>(part)[(n * 8 + i) * 32 + lane] = o[n][i];
          if (t == 0) {
            part[ROWS * kHeadDim + 8 * n + g] = m[n];
            part[ROWS * kHeadDim + ROWS + 8 * n + g] = l[n];
          }
        }
      }
      if (c.from_start ? !c.to_end : came_in != nullptr) leave(c, per, c.from_start ? begun : came_in);
      came_in = nullptr;
      if (c.u < c.u_end) open(c);
    }
    cp_async_wait<0>();
  }
};

template <typename T, int NT, int RING>
__global__ void __launch_bounds__(kRowThreads, 1) chunk_attention_rows(const __grid_constant__ AttnParams p) {
  using Warp = RowWarp<T, NT, RING>;
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ MergeRecord chains[kRowWarps + 1];
  long long* first = reinterpret_cast<long long*>(smem + kRowWarps * Warp::kWarpRing + Warp::kPartsBytes);
  __shared__ long long carry[kRowWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = p.a.requests;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the merge waits for this grid's end before it reads)
  long long total = 0;
  for (int r0 = 0; r0 < R; r0 += kRowThreads) {
    const int r = r0 + threadIdx.x;
    long long v = 0;
    if (r < R) {
      const Groups<8 * NT> g(p, request_of(p.a, r));
      v = (long long)g.groups * (g.tiles + kBegin) * p.a.kv_heads;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(kAll, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) carry[warp] = v;
    __syncthreads();
    long long before = total;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      if (w < warp) before += carry[w];
      total += carry[w];
    }
    if (r < R) first[r + 1] = before + v;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[0] = 0;
  __syncthreads();
  // Ranges that follow each other go to the warps of a CTA, whose pieces of a group are joined there.
  const long long shares = (long long)gridDim.x * kRowWarps;
  long long per = (total + shares - 1) / shares;
  per = per > p.min_tiles ? per : p.min_tiles;
  const int w = blockIdx.x * kRowWarps + warp, w_end = blockIdx.x * kRowWarps + kRowWarps - 1;
  const long long u0 = w * per, u1 = min(total, u0 + per);
  if (lane == 0) chains[warp].last = -1;
  if (threadIdx.x == 0) {
    chains[kRowWarps].last = -1;
    p.merges[blockIdx.x].last = -1;
  }
  __syncthreads();
  if (u0 < u1) Warp{p, first, smem, lane, warp}.run(u0, u1, per, warp == 0 ? chains + kRowWarps : nullptr, chains + warp);
  __syncthreads();
  // The CTA's chains of pieces, the one that has come in first; a warp has 16 of the dims of each.
#pragma unroll 1
  for (int k = kRowWarps; k >= 0; --k) {
    const MergeRecord rec = chains[k];
    if (rec.last < 0) continue;
    const bool came_in = k == kRowWarps;
    const int k0 = came_in ? 0 : k, k1 = min(rec.last, w_end) - blockIdx.x * kRowWarps;
    Joined<NT, 4> j;
    j.add([&](int q) { return Warp::piece(smem, k0 + q, q == 0 && !came_in); }, k1 - k0 + 1, warp, lane);
    if (!came_in && rec.last <= w_end) {
      j.template write<T>(p, rec, warp, lane);
    } else {
      j.store(p.joined + (size_t)(2 * blockIdx.x + (came_in ? 0 : 1)) * part_floats(ROWS), warp, lane);
      if (!came_in && threadIdx.x == 0) {
        MergeRecord r = rec;
        r.last = rec.last / kRowWarps;  // CTA with the last piece
        p.merges[blockIdx.x] = r;
      }
    }
  }
  // (launched while the tile kernel may still run: the stream goes on when both are done)
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Joins what the CTAs of the row kernel have left of the groups that several of them have worked on, in the order of the positions.
template <typename T, int NT>
__global__ void __launch_bounds__(256) chunk_attention_merge(const __grid_constant__ AttnParams p) {
  const int lane = threadIdx.x & 31, tile = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const MergeRecord rec = p.merges[blockIdx.x];
  if (rec.last < 0) return;
  auto part = [&](int q) { return p.joined + (size_t)(2 * (blockIdx.x + q) + (q == 0 ? 1 : 0)) * part_floats(8 * NT); };
  Joined<NT, 8 / NT> j;
  j.add(part, rec.last - (int)blockIdx.x + 1, tile, lane);
  j.template write<T>(p, rec, tile, lane);
}

cudaError_t launch_after(const void* kernel, dim3 grid, int threads, size_t smem, const AttnParams& p, cudaStream_t s) {
  // may be set up, and begin, while the kernel before it still runs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AttnParams copy = p;
  void* args[1] = {&copy};
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

constexpr int kMostSmem = 232448 - 1024;  // of a CTA, without what the kernel declares
template <typename T, int NT, int RING> int launch_rows(const AttnParams& p, bool behind_tiles, cudaStream_t s) {
  const int smem = RowWarp<T, NT, RING>::smem_bytes(p.a.requests);
  if constexpr (RING > 2) {
    if (smem > kMostSmem) return launch_rows<T, NT, RING - 1>(p, behind_tiles, s);  // (some hundreds of requests)
  }
  cudaError_t e = allow_shared<chunk_attention_rows<T, NT, RING>>(kMostSmem);
  if (e != cudaSuccess) return fail(MK_E_CUDA, "chunk_attention: %s", cudaGetErrorString(e));
  if (behind_tiles) {  // (the two write different rows; the kernel ahead of the tile kernel is done when that one begins)
    e = launch_after((const void*)chunk_attention_rows<T, NT, RING>, dim3(p.row_ctas), kRowThreads, smem, p, s);
  } else {
    chunk_attention_rows<T, NT, RING><<<p.row_ctas, kRowThreads, smem, s>>>(p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(MK_E_CUDA, "chunk_attention: launch failed: %s", cudaGetErrorString(e));
  e = launch_after((const void*)chunk_attention_merge<T, NT>, dim3(p.row_ctas), 256, 0, p, s);
  return e == cudaSuccess ? 0 : fail(MK_E_CUDA, "chunk_attention: launch failed: %s", cudaGetErrorString(e));
}

// Which kernels a call takes and what it needs of the workspace.
// Requests of up to 32 rows a kv head (new tokens x its q heads) are the row kernel's.  (24 requests of 6 tokens and a chunk of 200, 4 q heads a
// kv head: 79 us, with 16 as the limit 69; but 8 x 6 tokens alone 36 and 57, 64 x 6 84 and 90.  With 64 as the limit: 8 x 12 tokens 50
// instead of 59, 64 x 12 143 instead of 90.)
// A caller that gives no max_new has a grid of the tile kernel's launched ahead, whose CTAs find nothing to do in a batch of single tokens: 64 of 90 to
// 2200 positions, 32 q and 8 kv heads: 66 us, 57 with max_new; 4 of 20000 to 32700: 48 and 44.
constexpr int kFewRows = 32;
struct Layout {
  bool rows, tiles;
  int nt, few_rows, row_ctas, splits;
  size_t joined, tile_partial, bytes;
};
Layout layout_of(const mk_chunk_attention_args& a) {
  Layout l = {};
  const int per_kv = a.q_heads / a.kv_heads;
  const long long most = a.max_new > 0 && a.max_new < a.tokens ? a.max_new : a.tokens;
  l.tiles = most * per_kv > kFewRows && tiles_take(a);
  l.rows = !l.tiles || a.requests > 1;
  l.few_rows = !l.tiles ? 0x7fffffff : l.rows ? kFewRows : 0;
  // Groups of 8 rows, or of 16.  Beside chunks the row kernel mostly has single tokens, and 16 rows take twice the work of 8 whether
  // they are there or not (a chunk of 500 and 64 single tokens of 4 q heads a kv head: 64 us with 8, 70 with 16; a chunk of 200 and 24
  // requests of 6 tokens, whose K and V 8 rows read three times: 80 and 73).
  l.nt = (l.tiles ? per_kv : most * per_kv) <= 8 ? 1 : 2;
  l.row_ctas = sm_count();
  l.splits = 1;
  if (l.tiles) {
    const long long tokens = 2 * (128 / per_kv), ctas = (a.tokens + tokens - 1) / tokens * a.kv_heads;
    // As many CTAs as SMs; but every request may have a slot that turns out empty, and a thousand CTAs with nothing to do take longer
    // than a long chunk in few pieces (18 single tokens that the caller has not said to be such: 43 us for 2300, 28 for 580).
    const long long grid = (a.tokens / tokens + a.requests) * a.kv_heads;
    while (l.splits < 16 && 2 * l.splits * ctas <= sm_count() && 2 * l.splits * grid <= 4 * sm_count()) l.splits *= 2;
  }
  l.joined = l.rows ? (l.row_ctas * sizeof(MergeRecord) + 255) / 256 * 256 : 0;
  l.tile_partial = l.joined + (l.rows ? 2 * l.row_ctas * part_floats(8 * l.nt) * sizeof(float) : 0);
  l.bytes = l.tile_partial + (l.splits > 1 ? (size_t)l.splits * a.tokens * a.q_heads * (kHeadDim + 2) * sizeof(float) : 0);
  if (l.bytes == 0) l.bytes = 16;
  return l;
}

int check_pointers(const mk_chunk_attention_args& a) {
  if (!a.q || !a.k_cache || !a.v_cache || !a.qo_indptr || !a.kv_indptr || (!a.kv_indices && a.num_indices != 0) || !a.last_page_len || !a.out)
    return fail(MK_E_INVALID, "chunk_attention: null pointer");  // (an empty tensor has no address)
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.out)) return fail(MK_E_INVALID, "chunk_attention: pointers must be 16-byte aligned");
  return refuse_misaligned("chunk_attention", {{"lse", a.lse, 4}, {"qo_indptr", a.qo_indptr, 4}, {"kv_indptr", a.kv_indptr, 4}, {"kv_indices", a.kv_indices, 4},
                                               {"last_page_len", a.last_page_len, 4}});
}
int check_sizes(const mk_chunk_attention_args& a) {
  if (a.dtype != MK_BF16 && a.dtype != MK_F16) return fail(MK_E_INVALID, "chunk_attention: rows and caches are bf16 or fp16");
  if (a.tokens < 0 || a.q_heads < 1 || a.kv_heads < 1 || a.page_size < 1 || a.pages < 1 || a.num_indices < 0 || a.window < 0 || a.sinks < 0 || a.max_new < 0 || a.wait_ns < 0)
    return fail(MK_E_INVALID, "chunk_attention: negative or zero size");
  if (a.q_heads % a.kv_heads) return fail(MK_E_INVALID, "chunk_attention: %d q heads on %d kv heads", a.q_heads, a.kv_heads);
  if (a.requests < 1 || a.requests > kMaxRequests)
    return fail(a.requests < 1 ? MK_E_INVALID : MK_E_TOO_LARGE, "chunk_attention: %d requests (1 to %d)", a.requests, kMaxRequests);
  if ((long long)a.tokens * a.q_heads > 0x3fffffffll || (long long)a.requests * a.kv_heads > 0x3fffffffll || a.kv_heads > 65535) return fail(MK_E_TOO_LARGE, "chunk_attention: too many rows");
  for (int i = 0; i < 3; ++i)
    if ((a.k_cache_stride[i] | a.v_cache_stride[i]) & 7) return fail(MK_E_INVALID, "chunk_attention: rows of the caches must start at multiples of 16 bytes");
  for (int i = 0; i < 2; ++i)
    if ((a.q_stride[i] | a.out_stride[i]) & 7) return fail(MK_E_INVALID, "chunk_attention: rows of q and out must start at multiples of 16 bytes");
  return 0;
}

std::atomic<unsigned long long*> g_lost{nullptr};

}  // namespace

unsigned long long* lost_word() {
  unsigned long long* word = g_lost.load();
  if (word) return word;
  // (allowed while a stream is captured: the allocation has no part in the graph)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* fresh = nullptr;
  const cudaError_t e = cudaHostAlloc(&fresh, sizeof *word, cudaHostAllocPortable | cudaHostAllocMapped);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return cudaGetLastError(), nullptr;
  unsigned long long* const made = static_cast<unsigned long long*>(fresh);
  *made = 0;
  if (g_lost.compare_exchange_strong(word, made)) return made;
  cudaFreeHost(fresh);  // (another thread was faster)
  return word;
}
int report_lost_wait() {
  unsigned long long* word = g_lost.load();
  if (!word || __atomic_load_n(word, __ATOMIC_RELAXED) == 0) return 0;
  const unsigned long long said = __atomic_exchange_n(word, 0ull, __ATOMIC_ACQ_REL);
  if (!said) return 0;
  static const char* const kNames[] = {"the rows of q", "the last rows of V", "scores", "scores", "weights", "weights", "weights", "weights", "sums", "sums"};
  const unsigned bar = (unsigned)(said >> 32) & 0xffff;
  const char* name = bar < sizeof kNames / sizeof *kNames ? kNames[bar] : bar < 15 ? "a tile of K or V" : "a stage to become free";
  return fail(MK_E_DEVICE, "chunk_attention: in an earlier call the wait for %s ran out (CTA %u): rows of its output may be NaN", name, (unsigned)said);
}

}  // namespace mk_serving

extern "C" int mk_op_check(void) { return mk_serving::report_lost_wait(); }

extern "C" int64_t mk_chunk_attention_workspace(const mk_chunk_attention_args* args) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "chunk_attention: null arguments");
  if (int rc = check_sizes(*args)) return rc;
  return (int64_t)layout_of(*args).bytes;
}

extern "C" int mk_chunk_attention(const mk_chunk_attention_args* args, void* stream) {
  using namespace mk_serving;
  if (!args) return fail(MK_E_INVALID, "chunk_attention: null arguments");
  const mk_chunk_attention_args& a = *args;
  if (int rc = report_lost_wait()) return rc;
  if (int rc = check_pointers(a)) return rc;
  if (int rc = check_sizes(a)) return rc;
  if (a.tokens == 0) return 0;
  const Layout l = layout_of(a);
  if (!a.workspace || a.workspace_bytes < (int64_t)l.bytes || (((uintptr_t)a.workspace) & 15))
    return fail(MK_E_INVALID, "chunk_attention: a workspace of %lld bytes, 16-byte aligned, is needed", (long long)l.bytes);
  // Outputs are written while others are worked out, so they may share memory with nothing else of the call.
  auto rows = [&](const char* name, const void* at, const int64_t* stride, int bytes, int n) -> Memory {
    return {name, at, (long long)n * bytes, 2, {a.tokens, a.q_heads}, {bytes * stride[0], bytes * stride[1]}};
  };
  auto cache = [&](const char* name, const void* at, const int64_t* stride) -> Memory {
    return {name, at, 2 * kHeadDim, 3, {a.pages, a.page_size, a.kv_heads}, {2 * stride[0], 2 * stride[1], 2 * stride[2]}};
  };
  const Memory used[] = {rows("out", a.out, a.out_stride, 2, kHeadDim), rows("lse", a.lse, a.lse_stride, 4, 1), list_of("workspace", a.workspace, (long long)l.bytes, 1),
                         rows("q", a.q, a.q_stride, 2, kHeadDim), cache("k_cache", a.k_cache, a.k_cache_stride), cache("v_cache", a.v_cache, a.v_cache_stride),
                         list_of("qo_indptr", a.qo_indptr, a.requests + 1ll, 4), list_of("kv_indptr", a.kv_indptr, a.requests + 1ll, 4),
                         list_of("kv_indices", a.kv_indices, a.num_indices, 4), list_of("last_page_len", a.last_page_len, a.requests, 4)};
  if (int rc = refuse_shared("chunk_attention", used, 3, sizeof used / sizeof *used)) return rc;
  AttnParams p = {};
  p.a = a;
  p.per_kv = a.q_heads / a.kv_heads;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a.page_size == 1 << s) p.page_shift = s;
  p.scale_log2 = a.scale * kLog2e;
  p.row_ctas = l.row_ctas;
  p.tile_in_page = a.page_size % kPos == 0;
  p.min_tiles = 2;
  p.merges = reinterpret_cast<MergeRecord*>(a.workspace);
  p.joined = reinterpret_cast<float*>((char*)a.workspace + l.joined);
  p.few_rows = l.few_rows;
  p.splits = l.splits;
  p.tile_partial = reinterpret_cast<float*>((char*)a.workspace + l.tile_partial);
  const cudaStream_t s = (cudaStream_t)stream;
  if (l.tiles)
    if (int rc = launch_tile_attention(p, s)) return rc;
  if (!l.rows) return 0;
  const bool behind = l.tiles && l.splits == 1;
  // (two stages beside the parts of 16 rows)
  if (a.dtype == MK_BF16) return l.nt == 1 ? launch_rows<__nv_bfloat16, 1, 3>(p, behind, s) : launch_rows<__nv_bfloat16, 2, 2>(p, behind, s);
  return l.nt == 1 ? launch_rows<__half, 1, 3>(p, behind, s) : launch_rows<__half, 2, 2>(p, behind, s);
}
