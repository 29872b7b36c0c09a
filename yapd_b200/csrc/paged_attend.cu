// Attention of new tokens over a paged key-value cache.
//
// For a row of scores t_j = scale * log2(e) * q.k_j the softmax-weighted sum of
// the values is carried in one pass over the tokens: with m the largest t so
// far, z = sum 2^(t_j - m) and o = sum 2^(t_j - m) v_j, and two such triples
// over disjoint tokens join by scaling both to the larger m.  So the tokens of
// a request can be cut anywhere.
//
// The work is flattened into units of one tile of keys for one group of key
// heads of one request, and every CTA takes the same number of consecutive
// units, whatever the requests' lengths.  A (request, head group) that one CTA
// holds whole is written by it; one that is cut leaves a triple per CTA in the
// workspace, which a second kernel joins in their order.  No CTA waits for
// another one.
#include <cuda.h>  // CUtensorMap and the encode signature (the driver is reached at run time)

#include <atomic>
#include <cmath>
#include <mutex>

#include "select_common.cuh"
#include "serve_common.cuh"

namespace serve {
namespace {

constexpr int kWarps = 4;                     // that multiply; one more fetches
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kMaxRows = 64;  // query rows times key heads of a unit at most
constexpr int64_t kWaitNs = 500000000;

// A (request, head group, row block) that several CTAs hold parts of.
struct Piece {
  int b, head0, rb;
  int parts;   // 0: none
  int second;  // whether the first CTA's share begins with another piece
};

struct Attend {
  yapd_attend_args a;
  Div page;
  Div groups;        // query heads per key head
  int group;
  int rows;          // new_tokens * group: query rows that share a key head
  int wr;            // warps along the rows: 1, 2, 4 (1 unless M = 16)
  int hg;            // key heads of a unit: 1, 2, 4
  int head_groups, row_blocks;
  bool boxes;        // pages are whole groups of 16 tokens
  uint32_t keep;     // bits of the queries that count: none where the scale is 0
  uint32_t negate;   // sign bits of the queries to turn
  float scale_log2;  // positive
  int64_t wait_ns;   // limit of each wait
  Piece* pieces;     // (gridDim): the cut piece that begins in the CTA's share
  float* partials;   // (gridDim, 2) of (kMaxRows, D) sums and (kMaxRows, 2) maxima and sums of weights
};

// ------------------------------------------------------------ shapes by type

// M: query rows of a warp, 4, 8 or 16.
//
// A stage holds the keys, then the values, of a tile: groups of 16 tokens, in a
// group a slab for each 128 (64) bytes of the head dimension of each head, in a
// slab a row for each token. The 16-byte chunks of a row are permuted by the
// token (swizzle), so that the same chunk of eight tokens lies in eight
// different banks; it is the layout that a tensor copy of a group writes.
template <class T, int D, int M>
struct Shape {
  static constexpr int kRows = sizeof(T) == 2 ? (D == 32 ? 128 : 64) : (D == 32 ? 64 : 32);  // tokens x heads of a stage
  static constexpr int kStep = kRows / kWarps < 32 ? kRows / kWarps : 32;  // keys of one softmax step
  static constexpr int kBytes = D * (int)sizeof(T);
  static constexpr int kInner = kBytes % 128 == 0 ? 128 : 64;  // bytes of a row
  static constexpr int kSlabs = kBytes / kInner;               // of a head
  static constexpr int kSlab = 16 * kInner;
  static constexpr int kHalf = kRows * kBytes;
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kStages = 3;
  static constexpr int kMaxHeads = kRows / 16 < kWarps ? kRows / 16 : kWarps;  // key heads of a tile
  static constexpr int kWords = kRows / 32;          // of a mask of a tile's keys
  static constexpr int kQuery = sizeof(T) == 4 ? M * (D + 4) : 0;  // floats of a warp's queries in shared memory
  static constexpr int kSmem = kStages * kStage + kWarps * kQuery * 4;
  // CTAs of an SM: as many as its 228 KB hold, and no more than leave a thread
  // the registers of its sums (16 rows, 128 rows of blocks: 109 us with three
  // CTAs, 127 with two, 133 with four; in 32 bits 247 us with two, 296 with three)
  static constexpr int kRoom = 228 * 1024 / (kSmem + 1024 + 1024), kMost = sizeof(T) == 4 ? (M == 16 ? 2 : 3) : M == 16 ? 3 : 4;
  static constexpr int kFit = kRoom < kMost ? kRoom : kMost;
  static_assert(kWarps * M * D * 4 <= kStage, "the warps' triples meet in a stage");

  // Where 16-byte chunk `ch` of a row lies: token `tok` (of 16).
  __device__ static __forceinline__ int turn(int tok) { return (kInner == 128 ? tok & 7 : tok >> 1 & 3) << 4; }
};

// ----------------------------------------------------------------- the cache

// Tokens of a request; none where its length does not fit its table.
__device__ __forceinline__ int slot_len(const Attend& p, int b, int& slot) {
  const yapd_cache& c = p.a.cache;
  slot = p.a.slots ? p.a.slots[b] : b;
  if (slot < 0 || slot >= c.slots) {
    slot = -1;
    return 0;
  }
  const int64_t n = c.kv_len[slot];
  return fits(c, n) ? (int)n : 0;
}

// What the queries of a request of `len` tokens see: tokens below `sinks`, and
// from `low` on (the first query's window; later ones' start later).
__device__ __forceinline__ int first_low(const Attend& p, int len) {
  if (p.a.window <= 0) return 0;
  const int64_t low = (int64_t)len - p.a.new_tokens - p.a.window + 1;
  return low > 0 ? (int)low : 0;
}
__device__ __forceinline__ int sinks_of(const Attend& p) { return (int)(p.a.sinks < INT32_MAX ? p.a.sinks : INT32_MAX); }

// Tiles of `keys` tokens: those of the sinks, then those of the window.
struct Span {
  int sink_tiles, skip, tiles;
};
__device__ __forceinline__ Span span_of(const Attend& p, int len, int shift) {
  const int low = first_low(p, len), sinks = min(sinks_of(p), len);
  Span s;
  const int all = (len + (1 << shift) - 1) >> shift;
  s.sink_tiles = (sinks + (1 << shift) - 1) >> shift;
  const int start = low >> shift;
  s.skip = start > s.sink_tiles ? start - s.sink_tiles : 0;
  s.tiles = all - s.skip;
  return s;
}

// A position in the flattened work: request, (head group, row block), tile.
struct Cursor {
  int b, slot, len, hr, tile;
  Span span;
};

__device__ __forceinline__ void enter(const Attend& p, Cursor& c, int shift) {
  c.len = slot_len(p, c.b, c.slot);
  c.span = span_of(p, c.len, shift);
}
__device__ __forceinline__ void advance(const Attend& p, Cursor& c, int shift) {
  if (++c.tile < c.span.tiles) return;
  c.tile = 0;
  if (++c.hr < p.head_groups * p.row_blocks) return;
  c.hr = 0;
  do {
    if (++c.b >= p.a.B) return;
    enter(p, c, shift);
  } while (c.span.tiles == 0);
}
__device__ __forceinline__ int tile_start(const Cursor& c, int shift) {
  return (c.tile < c.span.sink_tiles ? c.tile : c.tile + c.span.skip) << shift;
}

__device__ __forceinline__ uint32_t smem_addr(const void* x) { return (uint32_t)__cvta_generic_to_shared(x); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// A box of 16 tokens of one page, all slabs of the unit's heads.
__device__ __forceinline__ void copy_group(uint32_t to, const CUtensorMap* map, uint64_t* bar, int token, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %3, %6}], [%2];" ::"r"(to),
      "l"(map), "r"(smem_addr(bar)), "r"(0), "r"(token), "r"(head), "r"(page)
      : "memory");
}
// A warp's bounded wait: its lanes go on or give up together, since every lane
// has a clock of its own and the products and shuffles that follow need them all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int64_t limit_ns) {
  return __all_sync(~0u, yapd::mbar_wait_bounded(bar, parity, limit_ns));
}
// Arrives at `bar` when all earlier copies of this thread have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ------------------------------------------------------------ matrix products

__device__ __forceinline__ void load_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_x4_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

// c (16 x 8, 32 bits) += a (16 x 16) b (16 x 8)
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ float2 unpack2(uint32_t x, __nv_bfloat16) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t x, __half) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
// What a weight is multiplied with where it enters a product, and a sum of values
// by the inverse of at its end. The smallest number in half precision is 2^-24:
// weights below 2^-25 of the largest one, which thousands of tokens may have, would
// leave the sums of the values while the sum of weights counts them. From 2^14 down
// their halves reach 2^-38. The other types have the exponents of 32 bits.
template <class T>
constexpr float kUp = 1.0f;
template <>
constexpr float kUp<__half> = 16384.0f;

// x and y, times kUp, as the sums of two T each
template <class T>
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
  x *= kUp<T>;
  y *= kUp<T>;
  high = pack2<T>(x, y);
  const float2 h = unpack2(high, T());
  low = pack2<T>(x - h.x, y - h.y);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ the rows

// One thread's share of a warp's M query rows (g = lane / 4, t = lane % 4).
//
// Scores are accumulators of (rows x keys): the thread holds rows g and, with
// M = 16, g + 8, and of each eight keys 2t and 2t + 1.  With M <= 8 the second
// half of the rows is zeros.
//
// Sums: with M = 16, or in 32 bits, (rows x dims) the same way: the thread's
// rows, dims 8n + 2t and + 1.  With M <= 8 in 16 bits (dims x rows): dims 16n +
// g and + 8, rows 2t and 2t + 1, so that no row of the product is empty; the
// scores, turned over, are the second operand as they lie in the registers.
// With M = 4 rows 4 to 7 repeat rows 0 to 3, and where the weights enter the
// product as two 16-bit halves the repeated rows carry the low halves.
template <class T, int D, int M>
struct Rows {
  static constexpr int kOwn = M == 16 ? 2 : 1;                       // rows whose scores the thread holds
  static constexpr bool kTurned = sizeof(T) == 2 && M <= 8;
  static constexpr int kSums = kTurned ? D / 16 : D / 8, kEach = kTurned ? 4 : 2 * kOwn;
  uint32_t q[sizeof(T) == 2 ? D / 16 : 1][2 * kOwn];
  float o[kSums][kEach];
  float m[kOwn], z[kOwn];
  int end[kOwn], low[kOwn];  // visible: [low, end) and [0, sinks)
};

__device__ __forceinline__ int row_of(int lane, int M, int r) { return ((lane >> 2) & (M - 1)) + 8 * r; }

template <class T>
__device__ __forceinline__ const T* query_at(const Attend& p, int b, int head, int row) {
  const int i = (int)div_floor(row, p.groups), h = head * p.group + row - i * p.group;
  return (const T*)p.a.q + b * p.a.q_stride_req + i * p.a.q_stride_pos + h * p.a.q_stride_head;
}

// The queries of M rows from `row0` on (rows past the last one: zeros).
template <class T, int D, int M>
__device__ __forceinline__ void begin_rows(const Attend& p, Rows<T, D, M>& w, const Cursor& c, int head, int row0,
                                           float* qs) {
  using R = Rows<T, D, M>;
  const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
  for (int n = 0; n < R::kSums; ++n)
#pragma unroll
    for (int e = 0; e < R::kEach; ++e) w.o[n][e] = 0.0f;
#pragma unroll
  for (int r = 0; r < R::kOwn; ++r) {
    const int row = row0 + row_of(lane, M, r), i = (int)div_floor(row, p.groups);
    const int place = c.len - p.a.new_tokens + i;
    w.m[r] = -INFINITY;
    w.z[r] = 0.0f;
    w.end[r] = p.a.causal ? min(c.len, place + 1) : c.len;
    const int64_t low = p.a.window > 0 ? place - p.a.window + 1 : 0;
    w.low[r] = low > 0 ? (int)low : 0;
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int r = 0; r < R::kOwn; ++r) {
      const int row = row0 + row_of(lane, M, r);
      const T* q = query_at<T>(p, c.b, head, row);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w.q[k][r + R::kOwn * e] =
              row < p.rows ? (*(const uint32_t*)(q + 16 * k + 8 * e + 2 * t) & p.keep) ^ p.negate : 0u;
    }
  } else {
    __syncwarp();
    for (int x = lane; x < M * (D / 4); x += 32) {
      const int r = x / (D / 4), d = x % (D / 4) * 4, row = row0 + r;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row < p.rows) v = *(const float4*)(query_at<T>(p, c.b, head, row) + d);
      if (!p.keep) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p.negate) v = make_float4(-v.x, -v.y, -v.z, -v.w);
      *(float4*)(qs + r * (D + 4) + d) = v;
    }
    __syncwarp();
  }
}

// Where a warp's keys lie in a stage, and how the layout goes on.
struct Place {
  const char* keys;  // the group's first slab of the warp's head
  int first;         // token of the group that a step begins with
  int slab;          // bytes between the slabs of a head
  int group;         // bytes between groups
};

// Scores of N keys: s[n][2 r + e] is row r's, key 8n + 2t + e.
template <class T, int D, int M, int N>
__device__ __forceinline__ void scores(const Rows<T, D, M>& w, float (&s)[N / 8][4], const Place& at, const float* qs) {
  using S = Shape<T, D, M>;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
  if constexpr (sizeof(T) == 2) {
    const int tok = (lane >> 4) * 8 + (lane & 7);
    const uint32_t row = smem_addr(at.keys) + tok * S::kInner + ((lane >> 3 & 1) << 4 ^ S::turn(tok));
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t a[4];
      if constexpr (M == 16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = w.q[k][e];
      } else {
        a[0] = w.q[k][0];
        a[2] = w.q[k][1];
        a[1] = a[3] = 0u;
      }
      constexpr int kIn = S::kInner / 32;  // products of a slab
#pragma unroll
      for (int n = 0; n < N / 16; ++n) {
        uint32_t f[4];
        load_x4(f, ((row + k / kIn * at.slab) ^ (k % kIn << 5)) + n * at.group);
        mma<T>(s[2 * n], a, f[0], f[1]);
        mma<T>(s[2 * n + 1], a, f[2], f[3]);
      }
    }
  } else {
    const int t = lane & 3, row = row_of(lane, M, 0);
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      const float4 q0 = *(const float4*)(qs + row * (D + 4) + d);
      float4 q1 = q0;
      if constexpr (M == 16) q1 = *(const float4*)(qs + (row + 8) * (D + 4) + d);
      const char* const slab = at.keys + d / 32 * at.slab;
#pragma unroll
      for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = at.first + 8 * n + 2 * t + e;
          const float4 k = *(const float4*)(slab + tok * S::kInner + (d % 32 * 4 ^ S::turn(tok)));
          s[n][e] = fmaf(q0.w, k.w, fmaf(q0.z, k.z, fmaf(q0.y, k.y, fmaf(q0.x, k.x, s[n][e]))));
          if constexpr (M == 16)
            s[n][2 + e] = fmaf(q1.w, k.w, fmaf(q1.z, k.z, fmaf(q1.y, k.y, fmaf(q1.x, k.x, s[n][2 + e]))));
        }
    }
  }
}

template <class T>
__device__ __forceinline__ bool finite_half(uint32_t x);
template <>
__device__ __forceinline__ bool finite_half<__nv_bfloat16>(uint32_t x) { return (x & 0x7f80u) != 0x7f80u; }
template <>
__device__ __forceinline__ bool finite_half<__half>(uint32_t x) { return (x & 0x7c00u) != 0x7c00u; }
template <class T>
__device__ __forceinline__ bool finite_word(uint32_t x) {
  if constexpr (sizeof(T) == 4)
    return (x & 0x7f800000u) != 0x7f800000u;
  else
    return finite_half<T>(x & 0xffffu) && finite_half<T>(x >> 16);
}

// Where element `d` of key `x` of a step lies, in the keys' or the values' half.
template <class T, int D, int M>
__device__ __forceinline__ const T* element_at(const Place& at, const char* half, int x, int d) {
  using S = Shape<T, D, M>;
  const int y = at.first + x, tok = y & 15, byte = d * (int)sizeof(T);
  return (const T*)(half + (y >> 4) * at.group + byte / S::kInner * at.slab + tok * S::kInner +
                    (byte % S::kInner ^ S::turn(tok)));
}

template <int S, int E>
struct Sums {
  float o[S][E];
};
template <int N>
struct Weights {
  float s[N / 8][4];
  uint32_t see;  // bit 4n + e: s[n][e] is of a visible token
};

// Zeros in the place of what is not finite.
template <class T>
__device__ __forceinline__ void clean(uint32_t (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (!finite_half<T>(f[e] & 0xffffu)) f[e] &= 0xffff0000u;
    if (!finite_half<T>(f[e] >> 16)) f[e] &= 0xffffu;
  }
}

// o += s v, with kClean only the finite values.  In 16 bits the weights enter as sums of two halves: one rounding
// of 2^-9 to each weight would cost as much precision as the output's own.
template <class T, int D, int M, int N, bool kClean>
__device__ __forceinline__ void values(float (&o)[Rows<T, D, M>::kSums][Rows<T, D, M>::kEach], const float (&s)[N / 8][4],
                                       const Place& at) {
  using S = Shape<T, D, M>;
  const int lane = threadIdx.x & 31;
  const char* const vals = at.keys + S::kHalf;
  constexpr int kIn = S::kInner / 32;  // 16 dims of a slab
  if constexpr (sizeof(T) == 2 && M <= 8) {
    // values (dims x keys) times weights (keys x rows)
    const int tok = (lane >> 4) * 8 + (lane & 7);
    const uint32_t row = smem_addr(vals) + tok * S::kInner + ((lane >> 3 & 1) << 4 ^ S::turn(tok));
#pragma unroll
    for (int n = 0; n < N / 16; ++n) {
      uint32_t h0, h1, l0, l1;
      split<T>(s[2 * n][0], s[2 * n][1], h0, l0);
      split<T>(s[2 * n + 1][0], s[2 * n + 1][1], h1, l1);
      if (M == 4 && lane >= 16) {
        h0 = l0;
        h1 = l1;
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t f[4];
        load_x4_turned(f, ((row + d / kIn * at.slab) ^ (d % kIn << 5)) + n * at.group);
        if (kClean) clean<T>(f);
        mma<T>(o[d], f, h0, h1);
        if (M != 4) mma<T>(o[d], f, l0, l1);
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    const int tok = lane & 15;
    const uint32_t row = smem_addr(vals) + tok * S::kInner + ((lane >> 4) << 4 ^ S::turn(tok));
#pragma unroll
    for (int n = 0; n < N / 16; ++n) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        split<T>(s[2 * n + (e >> 1)][2 * (e & 1)], s[2 * n + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t f[4];
        load_x4_turned(f, ((row + d / kIn * at.slab) ^ (d % kIn << 5)) + n * at.group);
        if (kClean) clean<T>(f);
        mma<T>(o[2 * d], hi, f[0], f[1]);
        mma<T>(o[2 * d + 1], hi, f[2], f[3]);
        mma<T>(o[2 * d], lo, f[0], f[1]);
        mma<T>(o[2 * d + 1], lo, f[2], f[3]);
      }
    }
  } else {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int from = (lane & ~3) + x;
          const float p0 = __shfl_sync(~0u, s[n][e], from);
          float p1 = 0.0f;
          if constexpr (M == 16) p1 = __shfl_sync(~0u, s[n][2 + e], from);
          const int tok = at.first + 8 * n + 2 * x + e;
          const char* const v = vals + tok * S::kInner;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            float2 f = *(const float2*)(v + d / 4 * at.slab + ((d % 4 * 32 + t * 8) ^ S::turn(tok)));
            if (kClean) {
              if (!isfinite(f.x)) f.x = 0.0f;
              if (!isfinite(f.y)) f.y = 0.0f;
            }
            o[d][0] = fmaf(p0, f.x, o[d][0]);
            o[d][1] = fmaf(p0, f.y, o[d][1]);
            if constexpr (M == 16) {
              o[d][2] = fmaf(p1, f.x, o[d][2]);
              o[d][3] = fmaf(p1, f.y, o[d][3]);
            }
          }
        }
  }
}

// o += s v where a value is not finite: the weight 0 of a token that a row does
// not see must not meet it. The finite ones as ever, then the others one by one,
// for the rows that see them.
template <class T, int D, int M, int N>
__device__ __noinline__ Sums<Rows<T, D, M>::kSums, Rows<T, D, M>::kEach> values_with_care(
    Sums<Rows<T, D, M>::kSums, Rows<T, D, M>::kEach> sums, Weights<N> w, Place at) {
  using R = Rows<T, D, M>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  values<T, D, M, N, true>(sums.o, w.s, at);
  const char* const vals = at.keys + Shape<T, D, M>::kHalf;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = 8 * n + 2 * x + e;
        // the weights of the two rows that the thread's sums are of
        float p[2];
        bool see[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int from = R::kTurned ? ((2 * t + r) & (M - 1)) * 4 + x : (lane & ~3) + x;
          const int slot = R::kTurned || M != 16 ? e : 2 * r + e;
          p[r] = __shfl_sync(~0u, w.s[n][slot], from);
          see[r] = __shfl_sync(~0u, w.see, from) >> (4 * n + slot) & 1;
        }
#pragma unroll
        for (int d = 0; d < R::kSums; ++d)
#pragma unroll
          for (int k = 0; k < R::kEach; ++k) {
            const int r = R::kTurned ? k & 1 : k >> 1, dim = R::kTurned ? 16 * d + g + 8 * (k >> 1) : 8 * d + 2 * t + (k & 1);
            const float f = to_f32(*element_at<T, D, M>(at, vals, key, dim));
            if (!isfinite(f) && see[r]) sums.o[d][k] = fmaf(p[r], f, sums.o[d][k]);
          }
      }
  return sums;
}

// One softmax step: N keys, the first of them token `j0`.  `mixed`: some row
// may not see some of them (`known`, from bit `bit0` on: the keys that are tokens).
template <class T, int D, int M, int N>
__device__ __forceinline__ void step(const Attend& p, Rows<T, D, M>& w, const Place& at, const float* qs, int j0,
                                     bool mixed, const uint32_t* known, int bit0) {
  using R = Rows<T, D, M>;
  const int lane = threadIdx.x & 31, t = lane & 3;
  float s[N / 8][4];
  scores<T, D, M, N>(w, s, at, qs);
  uint32_t see = 0;
  if (mixed) {
    const int sinks = sinks_of(p);
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2 * R::kOwn; ++e) {
        const int x = 8 * n + 2 * t + (e & 1), j = j0 + x, r = e >> 1, bit = bit0 + x;
        const bool v = (known[bit >> 5] >> (bit & 31) & 1) && j < w.end[r] && (j >= w.low[r] || j < sinks);
        see |= (uint32_t)v << (4 * n + e);
        if (!v) s[n][e] = -INFINITY;
      }
  }
  float fix[R::kOwn], base[R::kOwn];
  bool moved = false;
#pragma unroll
  for (int r = 0; r < R::kOwn; ++r) {
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < N / 8; ++n) top = fmaxf(top, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
    const float m = fmaxf(w.m[r], top * p.scale_log2);  // the scale is positive (see `keep`, `negate`)
    base[r] = m == -INFINITY ? 0.0f : m;
    fix[r] = ex2(w.m[r] - base[r]);
    moved |= fix[r] != 1.0f;
    w.m[r] = m;
  }
  if (__any_sync(~0u, moved)) {
#pragma unroll
    for (int r = 0; r < R::kOwn; ++r) w.z[r] *= fix[r];
    float f[2];  // of the rows that the thread's sums are of
    if constexpr (R::kTurned) {
#pragma unroll
      for (int r = 0; r < 2; ++r) f[r] = __shfl_sync(~0u, fix[0], ((2 * t + r) & (M - 1)) * 4);
    } else {
      f[0] = fix[0];
      f[1] = fix[R::kOwn - 1];
    }
#pragma unroll
    for (int d = 0; d < R::kSums; ++d)
#pragma unroll
      for (int e = 0; e < R::kEach; ++e) w.o[d][e] *= f[R::kTurned ? e & 1 : e >> 1];
  }
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2 * R::kOwn; ++e) {
      s[n][e] = ex2(fmaf(s[n][e], p.scale_log2, -base[e >> 1]));
      w.z[e >> 1] += s[n][e];
    }
  if (mixed) {
    // a value that is not finite reaches only the rows that see its token
    constexpr int kPer = D * (int)sizeof(T) / 4, kEl = 4 / (int)sizeof(T);
    const char* const vals = at.keys + Shape<T, D, M>::kHalf;
    bool careful = false;
    for (int x = lane; x < N * kPer; x += 32)
      careful |= !finite_word<T>(*(const uint32_t*)element_at<T, D, M>(at, vals, x / kPer, x % kPer * kEl));
    if (__any_sync(~0u, careful)) {
      // by value: nothing of the common path has an address
      Sums<R::kSums, R::kEach> sums;
      Weights<N> weights;
#pragma unroll
      for (int d = 0; d < R::kSums; ++d)
#pragma unroll
        for (int e = 0; e < R::kEach; ++e) sums.o[d][e] = w.o[d][e];
#pragma unroll
      for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) weights.s[n][e] = s[n][e];
      weights.see = see;
      sums = values_with_care<T, D, M, N>(sums, weights, at);
#pragma unroll
      for (int d = 0; d < R::kSums; ++d)
#pragma unroll
        for (int e = 0; e < R::kEach; ++e) w.o[d][e] = sums.o[d][e];
      return;
    }
  }
  values<T, D, M, N, false>(w.o, s, at);
}

// The keys that a warp has added to its sums.
struct Added {
  int b, len, shift;      // request, its tokens, tiles of 2^shift
  int tile0, tile1;       // of these tiles ...
  int first, span;        // ... `span` keys from `first` on
};

// The sum of the values of dim `dim` that are not finite, of the keys that a row
// with the bounds `end` and `low` sees: infinite, NaN, or 0 where all are finite.
template <class T>
__device__ __noinline__ float not_finite(const Attend& p, Added a, int head, int dim, int end, int low) {
  const yapd_cache& c = p.a.cache;
  const Span span = span_of(p, a.len, a.shift);
  const int slot = p.a.slots ? p.a.slots[a.b] : a.b, sinks = sinks_of(p);
  const int32_t* const row = c.page_table + (int64_t)slot * c.max_pages;
  const T* const vals = (const T*)c.kv + p.a.layer * c.stride_layer +
                        ((int64_t)c.page_size * c.kv_heads + head) * c.head_dim + dim;
  float odd = 0.0f;
  for (int tile = a.tile0; tile <= a.tile1; ++tile) {
    const int j0 = ((tile < span.sink_tiles ? tile : tile + span.skip) << a.shift) + a.first, j1 = min(j0 + a.span, end);
#pragma unroll 4
    for (int j = j0; j < j1; ++j) {
      if (j < low && j >= sinks) continue;
      const int q = (int)div_floor(j, p.page), g = row[q];
      if (g < 0 || g >= c.pages) continue;
      const float f = to_f32(vals[g * c.stride_page + (int64_t)(j - q * c.page_size) * c.kv_heads * c.head_dim]);
      if (!isfinite(f)) odd += f;
    }
    if (isnan(odd)) break;
  }
  return odd;
}

// The largest size of three numbers, NaN if one is.
__device__ __forceinline__ float larger_size(float x, float y, float z) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}

// An infinite value makes a sum infinite, but its products with the two halves of a
// weight may be NaN: the second half may be 0 or negative. Where a sum is not
// finite, the values that made it so are read once more. Once to a piece: the steps
// would have to wait for their products to look at them (128 rows of 16 positions:
// 113 us instead of 107).
template <class T, int D, int M>
__device__ __forceinline__ void make_good(const Attend& p, Rows<T, D, M>& w, const Added& a, int head) {
  using R = Rows<T, D, M>;
  if constexpr (sizeof(T) == 2) {
    float most = 0.0f;
#pragma unroll
    for (int d = 0; d < R::kSums; ++d)
#pragma unroll
      for (int e = 0; e < R::kEach; e += 2) most = larger_size(most, w.o[d][e], w.o[d][e + 1]);
    if (!__any_sync(~0u, !(most < INFINITY))) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int end[2], low[2];  // of the rows that the thread's sums are of
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int from = R::kTurned ? ((2 * t + r) & (M - 1)) * 4 : lane, own = R::kTurned ? 0 : r;
      end[r] = __shfl_sync(~0u, w.end[own], from);
      low[r] = __shfl_sync(~0u, w.low[own], from);
    }
#pragma unroll
    for (int d = 0; d < R::kSums; ++d)
#pragma unroll
      for (int k = 0; k < R::kEach; ++k)
        if (!isfinite(w.o[d][k])) {
          const int r = R::kTurned ? k & 1 : k >> 1, dim = R::kTurned ? 16 * d + g + 8 * (k >> 1) : 8 * d + 2 * t + (k & 1);
          const float odd = not_finite<T>(p, a, head, dim, end[r], low[r]);
          if (odd != 0.0f) w.o[d][k] = odd;  // 0: finite values whose sum is not
        }
  }
}

// Where the sums of a row's dim `d` meet: rows that are stored together lie in different banks.
template <int D>
__device__ __forceinline__ int meet_at(int row, int d) { return row * D + (d ^ ((row ^ row >> 2) & 3) << 3); }

// A warp's triples to shared memory: maxima and sums by row, o by (row, dim).
template <class T, int D, int M>
__device__ __forceinline__ void put_rows(Rows<T, D, M>& w, float* ms, float* zs, float* joined) {
  using R = Rows<T, D, M>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < R::kOwn; ++r) {
    w.z[r] += __shfl_xor_sync(~0u, w.z[r], 1);
    w.z[r] += __shfl_xor_sync(~0u, w.z[r], 2);
    if (t == 0 && g < M) {
      ms[g + 8 * r] = w.m[r];
      zs[g + 8 * r] = w.z[r];
    }
  }
#pragma unroll
  for (int d = 0; d < R::kSums; ++d) {
    if constexpr (R::kTurned) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (M == 4) w.o[d][e] += __shfl_xor_sync(~0u, w.o[d][e], 2);
        if (2 * t < M) joined[meet_at<D>(2 * t + (e & 1), 16 * d + g + 8 * (e >> 1))] = w.o[d][e];
      }
    } else {
#pragma unroll
      for (int r = 0; r < R::kOwn; ++r)
        if (g < M) *(float2*)(joined + meet_at<D>(g + 8 * r, 8 * d + 2 * t)) = make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
    }
  }
}

// ----------------------------------------------------------------- the kernel

// The new tokens' rows to their pages: a warp per (request, token). The
// attention that reads them waits for this kernel on the device.
template <class T>
__global__ void __launch_bounds__(128) store_kernel(const __grid_constant__ Attend p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const yapd_cache& c = p.a.cache;
  const int lane = threadIdx.x & 31, x = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (x >= p.a.B * p.a.new_tokens) return;
  const int b = x / p.a.new_tokens, i = x - b * p.a.new_tokens;
  // the first rows are on their way while their place is looked up
  constexpr int kVec = 16 / sizeof(T), kFirst = 4;
  const int per = c.head_dim / kVec, all = c.kv_heads * per;
  const T* const k = (const T*)p.a.k + b * p.a.k_stride_req + i * p.a.k_stride_pos;
  const T* const v = (const T*)p.a.v + b * p.a.v_stride_req + i * p.a.v_stride_pos;
  const auto row = [&](const T* rows, int64_t stride_head, int y) {
    const int h = y / per;
    return *(const uint4*)(rows + h * stride_head + (y - h * per) * kVec);
  };
  uint4 kx[kFirst], vx[kFirst];
#pragma unroll
  for (int u = 0; u < kFirst; ++u)
    if (lane + 32 * u < all) {
      kx[u] = row(k, p.a.k_stride_head, lane + 32 * u);
      vx[u] = row(v, p.a.v_stride_head, lane + 32 * u);
    }
  int slot;
  const int t = slot_len(p, b, slot) - p.a.new_tokens + i;
  // of the requests that name a slot the first one stores
  bool again = false;
  if (p.a.slots) {
    // four at a time where the list lies so (4096 requests: 5 us, one at a time 7; 1024: 1 us)
    const int four = (uintptr_t)p.a.slots % 16 == 0 ? b / 4 : 0;
#pragma unroll 4
    for (int j = lane; j < four; j += 32) {
      const int4 s = ((const int4*)p.a.slots)[j];
      again |= s.x == slot || s.y == slot || s.z == slot || s.w == slot;
    }
#pragma unroll 4
    for (int j = four * 4 + lane; j < b; j += 32) again |= p.a.slots[j] == slot;
  }
  again = __any_sync(~0u, again);
  uint32_t wrong = 0;
  int g = -1, q = 0;
  if (slot < 0 || again) {
    wrong = YAPD_STATUS_BAD_SLOT;
  } else if (t < 0) {
    wrong = YAPD_STATUS_BAD_LENGTH;
  } else {
    q = (int)div_floor(t, p.page);
    g = c.page_table[(int64_t)slot * c.max_pages + q];
    if (g < 0 || g >= c.pages)
      wrong = YAPD_STATUS_BAD_PAGE;
    else if (c.refs[g] > 1)
      wrong = YAPD_STATUS_SHARED_PAGE;
  }
  if (wrong) {
    if (lane == 0) set_status(c.workspace, wrong);
    return;
  }
  T* const to = (T*)c.kv + p.a.layer * c.stride_layer + g * c.stride_page +
                (int64_t)(t - q * c.page_size) * c.kv_heads * c.head_dim;
  T* const to_v = to + (int64_t)c.page_size * c.kv_heads * c.head_dim;
#pragma unroll
  for (int u = 0; u < kFirst; ++u)
    if (lane + 32 * u < all) {
      *(uint4*)(to + (int64_t)(lane + 32 * u) * kVec) = kx[u];
      *(uint4*)(to_v + (int64_t)(lane + 32 * u) * kVec) = vx[u];
    }
#pragma unroll 4
  for (int y = lane + 32 * kFirst; y < all; y += 32) {
    const uint4 ky = row(k, p.a.k_stride_head, y), vy = row(v, p.a.v_stride_head, y);
    *(uint4*)(to + (int64_t)y * kVec) = ky;
    *(uint4*)(to_v + (int64_t)y * kVec) = vy;
  }
}

template <class T>
__device__ __forceinline__ void write_row(const Attend& p, int b, int head, int row, int d, float4 o, float rz) {
  const int i = (int)div_floor(row, p.groups), h = head * p.group + row - i * p.group;
  T* out = (T*)p.a.out + b * p.a.out_stride_req + i * p.a.out_stride_pos + h * p.a.out_stride_head + d;
  if constexpr (sizeof(T) == 4) {
    *(float4*)out = make_float4(o.x * rz, o.y * rz, o.z * rz, o.w * rz);
  } else {
    uint2 x;
    x.x = pack2<T>(o.x * rz, o.y * rz);
    x.y = pack2<T>(o.z * rz, o.w * rz);
    *(uint2*)out = x;
  }
}
__device__ __forceinline__ void write_lse(const Attend& p, int b, int head, int row, float m, float z) {
  if (!p.a.lse) return;
  const int i = (int)div_floor(row, p.groups), h = head * p.group + row - i * p.group;
  p.a.lse[((int64_t)b * p.a.new_tokens + i) * p.a.heads + h] =
      z == 0.0f ? -INFINITY : m * 0.69314718055994531f + logf(z);
}

// The kernel. Its bound is the rate of the pages' reads: a token's key and value
// row, 4 D bytes at 16 bits, meet 4 D rows operations, so up to about 100 query
// rows of a key head the products are the smaller part; they run on the
// mma.sync pipe, at a tenth of its rate for one row (from 16 rows on a tcgen05
// tile with the keys or the queries on its 128 rows would shorten the steps). What it took to get there, 256 requests of
// 16 heads of 64 and 20 to 1250 tokens (692 MB; 106 us at the copy rate):
//   every warp copying its share of a stage, 255 registers       217 us
//   products by the number of rows, four CTAs per SM             169 us
//   one fetching warp, a 512-byte bulk copy to a token           161 us (17 ns a copy and SM)
//   one fetching warp, 16 bytes a lane                           184 us
//   one fetching warp, boxes of 16 tokens                        125 us
// and 4 requests of 95k tokens with 8 key heads of 128 (1.63 GB) 247 to 255 us, the
// copy rate. One request of 417 tokens, a tile to a CTA, takes 10 us: 3.3
// us to the first box, 1 us for the tile, 2 us for what the warps and the joining
// kernel add up, the rest for the three launches.

// What the fetching warp says of a tile.
struct Tile {
  int b, head0, rb, len, k0;  // request, first key head, row block, tokens, first token
  int tile, tiles;            // of the piece
  bool mixed, last;  // some row may not see some key; the share's or the piece's last tile
};

template <class T, int D, int M>
struct Shared {
  using S = Shape<T, D, M>;
  uint64_t full[S::kStages], empty[S::kStages], met;
  Tile tile[S::kStages];
  uint32_t known[S::kStages][S::kWords];   // which keys of a tile are tokens
  float m[kWarps * M], z[kWarps * M];      // maxima and sums that meet
  long long sums[kThreads / 32];
  int found[3];
  int given_up;
};

template <class T, int D, int M>
__global__ void __launch_bounds__(kThreads, Shape<T, D, M>::kFit) attend_kernel(const __grid_constant__ Attend p,
                                                                                const __grid_constant__ CUtensorMap map) {
  using S = Shape<T, D, M>;
  extern __shared__ __align__(1024) char smem[];
  char* const ring = smem;
  __shared__ Shared<T, D, M> sh;

  const yapd_cache& c = p.a.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.boxes && tid == kWarps * 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  const int shift = 31 - __clz(S::kRows / p.hg), keys = 1 << shift;  // keys of a tile
  const int pairs = p.head_groups * p.row_blocks;
  const int group_bytes = p.hg * 16 * S::kBytes;

  // every CTA of the grid runs: those of the joining kernel may take the place of the ones that end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // all units, and where this CTA's share begins
  const int per = (p.a.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.a.B), b1 = min(b0 + per, p.a.B);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    int slot;
    const int len = slot_len(p, b, slot);
    mine += (long long)span_of(p, len, shift).tiles * pairs;
    if (blockIdx.x == 0) {
      if (slot < 0)
        set_status(c.workspace, YAPD_STATUS_BAD_SLOT);
      else if (!fits(c, c.kv_len[slot]))
        set_status(c.workspace, YAPD_STATUS_BAD_LENGTH);
    }
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(~0u, upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 31) sh.sums[warp] = upto;
  if (tid == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      yapd::mbar_init(&sh.full[s], 33);  // the fetching warp's copies, and its word on the tile
      yapd::mbar_init(&sh.empty[s], kWarps);
    }
    yapd::mbar_init(&sh.met, kWarps);
    yapd::fence_mbar_init();
    sh.given_up = 0;
    p.pieces[blockIdx.x] = Piece{0, 0, 0, 0, 0};
  }
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) upto += total;
    total += sh.sums[w];
  }
  const long long chunk = (total + gridDim.x - 1) / gridDim.x;
  const long long u0 = min(chunk * blockIdx.x, total), u1 = min(u0 + chunk, total);
  const int units = (int)(u1 - u0);  // 2^31 tiles of one CTA would take it an hour
  if (units > 0 && upto - mine <= u0 && u0 < upto) {
    long long at = upto - mine;
    for (int b = b0;; ++b) {
      int slot;
      const int tiles = span_of(p, slot_len(p, b, slot), shift).tiles;
      const long long n = (long long)tiles * pairs;
      if (u0 < at + n) {
        const long long r = u0 - at;
        sh.found[0] = b;
        sh.found[1] = (int)(r / tiles);
        sh.found[2] = (int)(r % tiles);
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  constexpr int kPart = kMaxRows * (D + 2);

  if (warp == kWarps) {
    // ---------------------------------------------------------------- fetch
    // Lane y (and y + 32, ...) looks key y up: the table entry is read while the
    // tile before it is on its way. Where pages are whole groups of 16 tokens a
    // group's first lane copies it as two boxes; of other pages the warp copies
    // token by token, 16 bytes a lane.
    constexpr int kPer = S::kRows / 32;
    constexpr int kNone = INT32_MIN;
    constexpr int kVec = 16 / sizeof(T), kChunks = S::kBytes / 16, kIn = S::kInner / 16;
    const int chunks = p.hg * kChunks;                      // of a token's keys
    const int at_once = chunks >= 32 ? 1 : 32 / chunks;     // tokens of one instruction
    const int my_token = chunks >= 32 ? 0 : lane / chunks, my_chunk = lane - my_token * chunks;
    const bool copying = my_token < at_once;
    static_assert(kChunks * S::kMaxHeads <= 64, "two chunks of a token to a lane");
    const int64_t to_v = (int64_t)c.page_size * c.kv_heads * D;
    // where the lane's one or two chunks of a token lie in a group
    const auto slab_of = [&](int x) { return (x % kChunks / kIn * p.hg + x / kChunks) * S::kSlab; };
    const int chunk2 = my_chunk + 32, slab1 = slab_of(my_chunk), slab2 = slab_of(chunk2);
    const int in1 = my_chunk % kChunks % kIn << 4, in2 = chunk2 % kChunks % kIn << 4;
    const bool two = chunk2 < chunks;
    int entry[kPer];
    Cursor at;
    auto ask = [&]() {
      const int k0 = tile_start(at, shift), low = first_low(p, at.len), sinks = sinks_of(p);
      const int32_t* const row = c.page_table + (int64_t)at.slot * c.max_pages;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int y = lane + 32 * e, j = k0 + y;
        entry[e] = kNone;
        if (y < keys && j < at.len && (j >= low || j < sinks)) entry[e] = max(row[div_floor(j, p.page)], -1);
      }
    };
    int head0 = 0, rb = 0;
    if (units > 0) {
      at.b = sh.found[0];
      at.hr = sh.found[1];
      at.tile = sh.found[2];
      enter(p, at, shift);
      head0 = at.hr / p.row_blocks * p.hg;
      rb = at.hr % p.row_blocks;
      ask();
    }
    // the pages are read from here on
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
    bool bad = false;
    int it = 0;
    for (int stage = 0, phase = 1; it < units; ++it) {
      // a stage's first use needs no wait: the phase before the first counts as over
      if (!warp_wait(&sh.empty[stage], phase, it < S::kStages ? kWaitNs : p.wait_ns)) break;
      const int k0 = tile_start(at, shift);
      const uint32_t to = smem_addr(ring + stage * S::kStage);
      uint32_t tokens[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const bool wrong = entry[e] != kNone && (entry[e] < 0 || entry[e] >= c.pages);
        if (__any_sync(~0u, wrong)) {
          bad = true;
          if (wrong) {
            entry[e] = kNone;
            set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
          }
        }
        tokens[e] = __ballot_sync(~0u, entry[e] != kNone);
      }
      if (lane == 0) {
        Tile& t = sh.tile[stage];
        t.b = at.b;
        t.head0 = head0;
        t.rb = rb;
        t.len = at.len;
        t.k0 = k0;
        t.tile = at.tile;
        t.tiles = at.span.tiles;
        // every row sees every key of the tile unless
        const int first_end = p.a.causal ? at.len - p.a.new_tokens + 1 : at.len;
        const int64_t last_low = p.a.window > 0 ? (int64_t)at.len - p.a.window : 0;
        t.mixed = bad || k0 + keys > first_end || (k0 < last_low && k0 + keys > p.a.sinks);
        t.last = at.tile + 1 == at.span.tiles || it + 1 == units;
#pragma unroll
        for (int e = 0; e < kPer; ++e) sh.known[stage][e] = tokens[e];
        int groups = 0;
        if (p.boxes)
#pragma unroll
          for (int e = 0; e < kPer; ++e) groups += ((tokens[e] & 0xffffu) != 0) + (tokens[e] >> 16 != 0);
        yapd::mbar_arrive_expect_tx(&sh.full[stage], 2 * groups * group_bytes);
      }
      __syncwarp();
      if (p.boxes) {
        // a group's tokens are all of one page; hidden ones come along
        yapd::fence_proxy_async_smem();
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const uint32_t mine = lane < 16 ? tokens[e] & 0xffffu : tokens[e] & 0xffff0000u;
          const int g = __shfl_sync(~0u, entry[e], mine ? __ffs(mine) - 1 : lane);
          if ((lane & 15) == 0 && mine) {
            const int y = lane + 32 * e, j = k0 + y, r = j - (int)div_floor(j, p.page) * c.page_size;
            const uint32_t d = to + (y >> 4) * group_bytes;
            copy_group(d, &map, &sh.full[stage], r, head0, g);
            copy_group(d + S::kHalf, &map, &sh.full[stage], c.page_size + r, head0, g);
          }
        }
      } else {
        const T* const base = (const T*)c.kv + p.a.layer * c.stride_layer + head0 * D;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int j = k0 + lane + 32 * e, r = j - (int)div_floor(j, p.page) * c.page_size;
          const int64_t place = entry[e] == kNone ? -1 : entry[e] * c.stride_page + (int64_t)r * c.kv_heads * D;
          const int turns = min(32, keys - 32 * e) / at_once;
#pragma unroll 4
          for (int i = 0; i < turns; ++i) {
            const int from_lane = i * at_once + my_token, y = 32 * e + from_lane, tok = y & 15;
            const int64_t from = __shfl_sync(~0u, place, from_lane);
            if (!copying || from < 0) continue;
            const T* const k = base + from + my_chunk * kVec;
            const uint32_t row = to + (y >> 4) * group_bytes + tok * S::kInner, d = row + slab1 + (in1 ^ S::turn(tok));
            copy16(d, k);
            copy16(d + S::kHalf, k + to_v);
            if (two) {
              const uint32_t d2 = row + slab2 + (in2 ^ S::turn(tok));
              copy16(d2, k + 32 * kVec);
              copy16(d2 + S::kHalf, k + 32 * kVec + to_v);
            }
          }
        }
      }
      copies_arrive(&sh.full[stage]);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
      if (it + 1 < units) {
        const int hr = at.hr;
        advance(p, at, shift);
        if (at.hr != hr) {
          head0 = at.hr / p.row_blocks * p.hg;
          rb = at.hr % p.row_blocks;
        }
        ask();
      }
    }
    // What is on its way lands before the CTA ends and its shared memory is
    // another one's, whichever side gave up: the last stages' copies are waited for
    // here as well (they have landed where the other warps did not give up).
    copies_wait();
    for (int n = max(it - S::kStages, 0); n < it; ++n)
      warp_wait(&sh.full[n % S::kStages], n / S::kStages & 1, kWaitNs);
    if (it < units && lane == 0) {
      set_status(c.workspace, YAPD_STATUS_WAIT_TIMEOUT);
      atomicExch(&sh.given_up, 1);
    }
  } else {
    // -------------------------------------------------------------- multiply
    // requests without a token
    for (int b = blockIdx.x; b < p.a.B; b += gridDim.x) {
      int slot;
      if (slot_len(p, b, slot) > 0) continue;
      for (int x = tid; x < p.a.new_tokens * p.a.heads * (D / 4); x += kWarps * 32) {
        const int r = x / (D / 4), h = r % p.a.heads, i = r / p.a.heads, head = h / p.group;
        const int row = i * p.group + h - head * p.group;
        write_row<T>(p, b, head, row, x % (D / 4) * 4, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 1.0f);
        if (x % (D / 4) == 0) write_lse(p, b, head, row, 0.0f, 0.0f);
      }
    }
    const int wk_all = kWarps / p.wr, wk = warp / p.wr, wrow = warp - wk * p.wr;
    const int parts = wk_all / p.hg;                       // warps that share a head's keys
    const int head_in = wk / parts, part = wk - head_in * parts;
    const int span = keys / parts;                         // keys of this warp
    // the warp's keys: from the group's start on, and whole steps of 16 in groups of their own
    const int mine_at = (part * span >> 4) * group_bytes + head_in * S::kSlab;
    float* const my_qs = (float*)(smem + S::kStages * S::kStage) + warp * S::kQuery;
    bool ok = true;
    int meetings = 0;
    // the multiplying warps wait for one another
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) yapd::mbar_arrive(&sh.met);
      ok = ok && warp_wait(&sh.met, meetings++ & 1, p.wait_ns);
    };
    Rows<T, D, M> w;
    bool fresh = true, whole = true;
    int tile0 = 0;  // the piece's first one here
    for (int it = 0, stage = 0, phase = 0; it < units; ++it) {
      if (!(ok = warp_wait(&sh.full[stage], phase, p.wait_ns))) break;
      const Tile& t = sh.tile[stage];
      const int head0 = t.head0, rb = t.rb;
      if (fresh) {
        whole = t.tile == 0;
        tile0 = t.tile;
        Cursor x;
        x.b = t.b;
        x.len = t.len;
        begin_rows<T, D, M>(p, w, x, head0 + head_in, (rb * p.wr + wrow) * M, my_qs);
        fresh = false;
      }
      {
        Place at;
        at.keys = ring + stage * S::kStage + mine_at;
        at.first = part * span & 15;
        at.slab = p.hg * S::kSlab;
        at.group = group_bytes;
        const bool mixed = t.mixed;
        const int j0 = t.k0 + part * span, len = t.len;
        for (int x = 0; x < span; x += S::kStep) {
          if (j0 + x >= len) break;
          step<T, D, M, S::kStep>(p, w, at, my_qs, j0 + x, mixed, sh.known[stage], part * span + x);
          if constexpr (S::kStep < 16) {
            at.first += S::kStep;
            if (at.first == 16) {
              at.first = 0;
              at.keys += group_bytes;
            }
          } else {
            at.keys += S::kStep / 16 * group_bytes;
          }
        }
      }
      if (t.last) {
        // the warps' triples meet in the stage that was just read
        const bool done = t.tile + 1 == t.tiles;
        whole = whole && done;
        const int b = t.b;
        const long long start = u0 + it - t.tile, end = start + t.tiles;
        make_good<T, D, M>(p, w, Added{b, t.len, shift, tile0, t.tile, part * span, span}, head0 + head_in);
        meet();
        if (!ok) break;
        float* const joined = (float*)(ring + stage * S::kStage);
        put_rows<T, D, M>(w, sh.m + warp * M, sh.z + warp * M, joined + warp * M * D);
        meet();
        if (!ok) break;
        const int block_rows = p.wr * M, rows_here = min(block_rows, p.rows - rb * block_rows);
        float* const left_at = p.partials + ((int64_t)blockIdx.x * 2 + (start > u0 ? 1 : 0)) * kPart;
        for (int x = tid; x < p.hg * rows_here * (D / 4); x += kWarps * 32) {
          const int rr = x / (D / 4), d = x - rr * (D / 4), hi = rr / rows_here, row = rr - hi * rows_here;
          const int rm = row & (M - 1), first = (hi * parts) * p.wr + row / M;
          float m = -INFINITY;
          for (int k = 0; k < parts; ++k) m = fmaxf(m, sh.m[(first + k * p.wr) * M + rm]);
          const float base = m == -INFINITY ? 0.0f : m;
          float z = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int k = 0; k < parts; ++k) {
            const int y = (first + k * p.wr) * M + rm;
            const float f = ex2(sh.m[y] - base);
            const float4 v = *(const float4*)(joined + y / M * M * D + meet_at<D>(rm, 4 * d));
            z = fmaf(f, sh.z[y], z);
            o.x = fmaf(f, v.x, o.x);
            o.y = fmaf(f, v.y, o.y);
            o.z = fmaf(f, v.z, o.z);
            o.w = fmaf(f, v.w, o.w);
          }
          if (whole) {
            const float rz = z == 0.0f ? 0.0f : 1.0f / (kUp<T> * z);
            write_row<T>(p, b, head0 + hi, rb * block_rows + row, 4 * d, o, rz);
            if (d == 0) write_lse(p, b, head0 + hi, rb * block_rows + row, m, z);
          } else {
            *(float4*)(left_at + 4 * x) = o;
            if (d == 0) *(float2*)(left_at + kMaxRows * D + 2 * rr) = make_float2(m, z);
          }
        }
        yapd::fence_proxy_async_smem();  // the stage is a box's target again
        if (!whole && start >= u0 && tid == 0) {
          // the piece begins here: where the parts are, for the kernel that joins them
          const long long c0 = start / chunk;
          p.pieces[blockIdx.x] = Piece{b, head0, rb, (int)((end - 1) / chunk - c0) + 1, start > u0};
        }
        fresh = true;
      }
      __syncwarp();
      if (lane == 0) yapd::mbar_arrive(&sh.empty[stage]);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok && lane == 0) {
      set_status(c.workspace, YAPD_STATUS_WAIT_TIMEOUT);
      atomicExch(&sh.given_up, 1);
    }
  }

  // A CTA that gave up leaves no numbers to the pieces that it shares.
  __syncthreads();
  if (sh.given_up)
    for (int r = tid; r < 2 * kMaxRows; r += kThreads)
      *(float2*)(p.partials + ((int64_t)blockIdx.x * 2 + r / kMaxRows) * kPart + kMaxRows * D + r % kMaxRows * 2) =
          make_float2(0.0f, NAN);
}

// Joins the parts of the piece that begins in a CTA's share, in their order:
// four dims of a row to a thread, and where that leaves threads over, the parts
// are shared out over groups of them. Time is the latency of the reads, so a
// thread has eight parts' under way.
constexpr int kJoinThreads = 256;
template <class T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Attend p, int block_rows) {
  constexpr int64_t kPart = kMaxRows * (D + 2);
  __shared__ float2 mzs[kJoinThreads];
  __shared__ float4 os[kJoinThreads];
  const int tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Piece piece = p.pieces[blockIdx.x];
  if (piece.parts == 0) return;
  const int rows_here = min(block_rows, p.rows - piece.rb * block_rows), items = p.hg * rows_here * (D / 4);
  const int groups = max(1, min(min(kJoinThreads / items, 8), piece.parts / 4));
  const int group = groups > 1 ? tid / items : 0;
  // the first CTA's part is its second one unless its share begins with the piece
  const auto part_at = [&](int k) { return p.partials + ((int64_t)(blockIdx.x + k) * 2 + (k == 0 ? piece.second : 0)) * kPart; };
  const auto add = [](float& m, float& z, float4& o, float2 mz, float4 v) {
    const float top = fmaxf(m, mz.x), base = top == -INFINITY ? 0.0f : top, f0 = ex2(m - base), f = ex2(mz.x - base);
    z = fmaf(f, mz.y, z * f0);
    o.x = fmaf(f, v.x, o.x * f0);
    o.y = fmaf(f, v.y, o.y * f0);
    o.z = fmaf(f, v.z, o.z * f0);
    o.w = fmaf(f, v.w, o.w * f0);
    m = top;
  };
  for (int x = groups > 1 ? tid - group * items : tid; x < items; x += kJoinThreads) {
    float m = -INFINITY, z = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = group; k0 < piece.parts && group < groups; k0 += 8 * groups) {
      float2 mz[8];
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k0 + k * groups < piece.parts) {
          const float* const y = part_at(k0 + k * groups);
          mz[k] = __ldcg((const float2*)(y + kMaxRows * D + x / (D / 4) * 2));
          v[k] = __ldcg((const float4*)(y + 4 * x));
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k * groups < piece.parts) add(m, z, o, mz[k], v[k]);
    }
    if (groups > 1) {
      mzs[tid] = make_float2(m, z);
      os[tid] = o;
      __syncthreads();  // every thread comes here once: the items are fewer than the threads
      if (group) break;
      for (int g = 1; g < groups; ++g) add(m, z, o, mzs[g * items + x], os[g * items + x]);
    }
    const int rr = x / (D / 4), d = x - rr * (D / 4), hi = rr / rows_here;
    const int full = piece.rb * block_rows + rr - hi * rows_here;
    write_row<T>(p, piece.b, piece.head0 + hi, full, 4 * d, o, z == 0.0f ? 0.0f : 1.0f / (kUp<T> * z));
    if (d == 0) write_lse(p, piece.b, piece.head0 + hi, full, m, z);
  }
}

// ------------------------------------------------------------------ the host

// The kernel's grid on the current device: every CTA that fits at once.
template <class T, int D, int M>
int grid_of(int& grid) {
  constexpr int kSmem = Shape<T, D, M>::kSmem;
  static std::atomic<int> grids[64];  // per device, found at its first call
  int dev = 0, sms = 0, fit = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return YAPD_ERR_NO_DEVICE;
  grid = grids[dev].load(std::memory_order_relaxed);
  if (grid) return YAPD_OK;
  if (cudaFuncSetAttribute(attend_kernel<T, D, M>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, attend_kernel<T, D, M>, kThreads, kSmem) != cudaSuccess ||
      fit < 1)
    return YAPD_ERR_LAUNCH;
  grid = sms * fit < kMaxCtas ? sms * fit : kMaxCtas;
  grids[dev].store(grid, std::memory_order_relaxed);
  return YAPD_OK;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}

// The layer's pages as (row of a slab, token of both halves, head, slab of a
// head, page); a box is 16 tokens of the unit's heads.
template <class T, int D, int M>
bool encode(const Attend& p, CUtensorMap& map) {
  using S = Shape<T, D, M>;
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const yapd_cache& c = p.a.cache;
  const cuuint32_t inner = S::kInner / sizeof(T);
  const int64_t block = (int64_t)2 * c.page_size * c.kv_heads * D;
  const cuuint64_t dims[5] = {inner, (cuuint64_t)2 * c.page_size, (cuuint64_t)c.kv_heads, S::kSlabs, (cuuint64_t)c.pages};
  const cuuint64_t strides[4] = {(cuuint64_t)c.kv_heads * S::kBytes, S::kBytes, S::kInner,
                                 (cuuint64_t)(c.pages > 1 ? c.stride_page : block) * sizeof(T)};
  const cuuint32_t box[5] = {inner, 16, (cuuint32_t)p.hg, S::kSlabs, 1}, step[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : p.a.cache.dtype == YAPD_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(&map, type, 5, (T*)c.kv + p.a.layer * c.stride_layer, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            S::kInner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, int M>
int launch(Attend& p, cudaStream_t st) {
  int grid = 0;
  const int rc = grid_of<T, D, M>(grid);
  if (rc != YAPD_OK) return rc;
  p.wr = M < 16 || p.rows <= 16 ? 1 : p.rows <= 32 ? 2 : 4;
  p.row_blocks = (p.rows + M * p.wr - 1) / (M * p.wr);
  p.boxes = p.a.cache.page_size % 16 == 0;
  // Key heads of a unit: the rows of several heads of a token lie side by side
  // in its page, and a piece has more tiles (256 requests of 16 heads: 169 us
  // with four, 182 with two, 218 with one).  Few requests are shared out by
  // heads first, so that fewer CTAs hold parts of the same sums (64 requests:
  // 44 us with four heads; 48 requests of 4 heads: 49 us with one, 54 with two).
  const int kvh = p.a.cache.kv_heads;
  p.hg = Shape<T, D, M>::kMaxHeads >= p.wr ? Shape<T, D, M>::kMaxHeads / p.wr : 1;
  const int64_t pieces = p.boxes ? grid / 4 : 0;
  while (p.hg > 1 && (kvh % p.hg || (int64_t)p.a.B * (kvh / p.hg) * p.row_blocks < pieces)) p.hg /= 2;
  p.head_groups = kvh / p.hg;
  CUtensorMap map{};
  if (p.boxes && !encode<T, D, M>(p, map)) return YAPD_ERR_LAUNCH;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shape<T, D, M>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  if (p.a.k) {
    const int rows = p.a.B * p.a.new_tokens;
    store_kernel<T><<<(rows + 3) / 4, 128, 0, st>>>(p);
    // the attention's CTAs start beside the stores and wait for them where they read the pages
    cfg.attrs = &early;
    cfg.numAttrs = 1;
  }
  if (cudaLaunchKernelEx(&cfg, attend_kernel<T, D, M>, p, map) != cudaSuccess) return YAPD_ERR_LAUNCH;
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p, M * p.wr) != cudaSuccess) return YAPD_ERR_LAUNCH;
  return launched();
}

template <class T, int D>
int launch_rows(Attend& p, cudaStream_t st) {
  if (sizeof(T) == 2 && p.rows <= 4) return launch<T, D, sizeof(T) == 2 ? 4 : 8>(p, st);
  if (p.rows <= 8) return launch<T, D, 8>(p, st);
  return launch<T, D, 16>(p, st);
}

template <class T>
int launch_dim(Attend& p, cudaStream_t st) {
  switch (p.a.cache.head_dim) {
    case 32: return launch_rows<T, 32>(p, st);
    case 64: return launch_rows<T, 64>(p, st);
    case 96: return launch_rows<T, 96>(p, st);
    default: return launch_rows<T, 128>(p, st);
  }
}

bool rows_aligned(const void* base, int64_t r, int64_t p, int64_t h, int dtype) {
  const int64_t vec = 16 / dtype_size(dtype);
  return (uintptr_t)base % 16 == 0 && r % vec == 0 && p % vec == 0 && h % vec == 0;
}

}  // namespace

size_t attend_scratch_bytes(const yapd_cache& c) {
  return round_up(kMaxCtas * sizeof(Piece), 256) + (size_t)kMaxCtas * 2 * kMaxRows * (c.head_dim + 2) * 4;
}

}  // namespace serve

using namespace serve;

extern "C" int yapd_attend(const yapd_attend_args* args, void* stream) {
  if (!args) return YAPD_ERR_NULL_POINTER;
  const yapd_attend_args& a = *args;
  const int rc = check_cache(a.cache);
  if (rc != YAPD_OK) return rc;
  const int kvh = a.cache.kv_heads;
  if (a.B < 0 || a.B > 65535 || a.new_tokens < 1 || a.new_tokens > YAPD_MAX_NEW_TOKENS || a.heads < 1 ||
      a.heads % kvh || a.heads > 1024 || (!a.slots && a.B > a.cache.slots))
    return YAPD_ERR_BAD_SHAPE;
  if (a.layer < 0 || a.layer >= a.cache.layers || a.sinks < 0 || !(a.scale == a.scale)) return YAPD_ERR_BAD_ARG;
  if (a.B == 0) return YAPD_OK;
  if (!a.q || !a.out || !a.k != !a.v) return YAPD_ERR_NULL_POINTER;
  const int dt = a.cache.dtype;
  if (!rows_aligned(a.q, a.q_stride_req, a.q_stride_pos, a.q_stride_head, dt) ||
      !rows_aligned(a.out, a.out_stride_req, a.out_stride_pos, a.out_stride_head, dt) ||
      (a.k && (!rows_aligned(a.k, a.k_stride_req, a.k_stride_pos, a.k_stride_head, dt) ||
               !rows_aligned(a.v, a.v_stride_req, a.v_stride_pos, a.v_stride_head, dt))))
    return YAPD_ERR_MISALIGNED;
  Attend p;
  p.a = a;
  p.page = make_div((uint32_t)a.cache.page_size);
  p.group = a.heads / kvh;
  p.groups = make_div((uint32_t)p.group);
  p.rows = a.new_tokens * p.group;
  // A negative scale is a positive one of the negative queries, and a scale of 0
  // any other one of queries that are 0: hidden scores are -inf before the scale.
  p.keep = a.scale == 0.0f ? 0u : ~0u;
  p.negate = std::signbit(a.scale) ? dt == YAPD_DTYPE_F32 ? 0x80000000u : 0x80008000u : 0u;
  p.scale_log2 = a.scale == 0.0f ? 1.0f : std::fabs(a.scale) * 1.4426950408889634f;
  p.wait_ns = a.wait_limit_ns ? a.wait_limit_ns : kWaitNs;
  char* const scratch = (char*)a.cache.workspace + kHeaderBytes + pages_scratch_bytes(a.cache);
  p.pieces = (Piece*)scratch;
  p.partials = (float*)(scratch + round_up(kMaxCtas * sizeof(Piece), 256));
  switch (dt) {
    case YAPD_DTYPE_F32: return launch_dim<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch_dim<__half>(p, (cudaStream_t)stream);
    default: return launch_dim<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
