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
// workspace, and the CTA that arrives last joins them in their order.  No CTA
// waits for another one.
#include <atomic>
#include <cmath>

#include "serve_common.cuh"

namespace serve {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxRows = 64;  // query rows times key heads of a unit at most

struct Attend {
  yapd_attend_args a;
  Div page;
  Div groups;        // query heads per key head
  int group;
  int rows;          // new_tokens * group: query rows that share a key head
  int wr;            // warps along the rows: 1, 2, 4 (1 unless M = 16)
  int hg;            // key heads of a unit: 1, 2, 4
  int head_groups, row_blocks;
  uint32_t negate;   // sign bits of the queries to turn
  float scale_log2;  // not negative
  int* counters;     // (gridDim): arrivals at a cut piece that starts in the CTA
  float* partials;   // (gridDim, 2, kMaxRows, D + 2)
};

// ------------------------------------------------------------ shapes by type

// M: query rows of a warp, 4, 8 or 16.
template <class T, int D, int M>
struct Shape {
  // rows of keys in a stage, and as many of values
  static constexpr int kRows = sizeof(T) == 2 ? (D == 32 ? 128 : 64) : (D == 32 ? 64 : 32);
  static constexpr int kStep = kRows / kWarps < 32 ? kRows / kWarps : 32;  // keys of one softmax step
  static constexpr int kPitch = D * sizeof(T) + 16;  // bytes: eight rows' 16-byte chunks fall in different banks
  static constexpr int kHalf = kRows * kPitch;
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kStages = 3;
  static constexpr int kChunks = D * sizeof(T) / 16;
  static constexpr int kLoads = kRows * kChunks / kThreads;
  static constexpr int kJoinPitch = D + 4;           // floats
  static constexpr int kWords = kRows / 32;          // of a mask of keys
  static constexpr int kQuery = sizeof(T) == 4 ? M * (D + 4) : 0;  // floats of a warp's queries in shared memory
  static constexpr int kSmem = kStages * kStage + kWarps * kQuery * 4 + 2 * kRows * 8;
  // CTAs of an SM: as many as its 228 KB hold, and no more than leave a thread the registers of its sums
  static constexpr int kRoom = 228 * 1024 / (kSmem + 1024 + 512), kMost = M == 16 ? 3 : 4;
  static constexpr int kFit = kRoom < kMost ? kRoom : kMost;
  static_assert(kWarps * M * kJoinPitch * 4 <= kStage, "the warps' triples meet in a stage");
  static_assert(kRows * kChunks % kThreads == 0 && kRows <= kThreads, "");
};

// ----------------------------------------------------------------- the cache

__device__ __forceinline__ int slot_len(const Attend& p, int b, int& slot) {
  const yapd_cache& c = p.a.cache;
  slot = p.a.slots ? p.a.slots[b] : b;
  if (slot < 0 || slot >= c.slots) {
    slot = -1;
    return 0;
  }
  const int64_t n = c.kv_len[slot], most = (int64_t)c.max_pages * c.page_size;
  return (int)(n < 0 ? 0 : n > most ? most : n);
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

// ------------------------------------------------------------------- copies

__device__ __forceinline__ uint32_t smem_addr(const void* x) { return (uint32_t)__cvta_generic_to_shared(x); }

// 16 bytes to shared memory, or zeros where `from` is not to be read.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

__device__ __forceinline__ uint32_t pack(__nv_bfloat16 lo, __nv_bfloat16 hi) {
  __nv_bfloat162 x(lo, hi);
  return *reinterpret_cast<uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t pack(__half lo, __half hi) {
  __half2 x(lo, hi);
  return *reinterpret_cast<uint32_t*>(&x);
}
// x and y as the sums of two T each
template <class T>
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
  const T hx = from_f32<T>(x), hy = from_f32<T>(y);
  high = pack(hx, hy);
  low = pack(from_f32<T>(x - to_f32(hx)), from_f32<T>(y - to_f32(hy)));
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
              row < p.rows ? *(const uint32_t*)(q + 16 * k + 8 * e + 2 * t) ^ p.negate : 0u;
    }
  } else {
    __syncwarp();
    for (int x = lane; x < M * (D / 4); x += 32) {
      const int r = x / (D / 4), d = x % (D / 4) * 4, row = row0 + r;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row < p.rows) v = *(const float4*)(query_at<T>(p, c.b, head, row) + d);
      if (p.negate) v = make_float4(-v.x, -v.y, -v.z, -v.w);
      *(float4*)(qs + r * (D + 4) + d) = v;
    }
    __syncwarp();
  }
}

// Scores of N keys whose rows start at `keys`: s[n][2 r + e] is row r's, key 8n + 2t + e.
template <class T, int D, int M, int N>
__device__ __forceinline__ void scores(const Rows<T, D, M>& w, float (&s)[N / 8][4], const char* keys, const float* qs) {
  constexpr int kPitch = Shape<T, D, M>::kPitch;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
  if constexpr (sizeof(T) == 2) {
    const uint32_t at = smem_addr(keys) + ((lane >> 4) * 8 + (lane & 7)) * kPitch + (lane >> 3 & 1) * 16;
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
#pragma unroll
      for (int n = 0; n < N / 16; ++n) {
        uint32_t f[4];
        load_x4(f, at + n * 16 * kPitch + k * 32);
        mma<T>(s[2 * n], a, f[0], f[1]);
        mma<T>(s[2 * n + 1], a, f[2], f[3]);
      }
    }
  } else {
    const int g = lane >> 2, t = lane & 3, row = row_of(lane, M, 0);
    (void)g;
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      const float4 q0 = *(const float4*)(qs + row * (D + 4) + d);
      float4 q1 = q0;
      if constexpr (M == 16) q1 = *(const float4*)(qs + (row + 8) * (D + 4) + d);
#pragma unroll
      for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 k = *(const float4*)(keys + (8 * n + 2 * t + e) * kPitch + d * 4);
          s[n][e] = fmaf(q0.w, k.w, fmaf(q0.z, k.z, fmaf(q0.y, k.y, fmaf(q0.x, k.x, s[n][e]))));
          if constexpr (M == 16)
            s[n][2 + e] = fmaf(q1.w, k.w, fmaf(q1.z, k.z, fmaf(q1.y, k.y, fmaf(q1.x, k.x, s[n][2 + e]))));
        }
    }
  }
}

__device__ __forceinline__ bool any_nonfinite(uint32_t x, __nv_bfloat16) {
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ bool any_nonfinite(uint32_t x, __half) {
  return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ bool any_nonfinite(uint32_t x, float) { return (x & 0x7f800000u) == 0x7f800000u; }

template <int S, int E>
struct Sums {
  float o[S][E];
};
template <int N>
struct Weights {
  float s[N / 8][4];
  uint32_t see;  // bit 4n + e: s[n][e] is of a visible token
};

// o += s v with the weight 0 of a hidden token kept away from its value, which
// may be anything: element by element.
template <class T, int D, int M, int N>
__device__ __noinline__ Sums<Rows<T, D, M>::kSums, Rows<T, D, M>::kEach> values_one_by_one(
    Sums<Rows<T, D, M>::kSums, Rows<T, D, M>::kEach> sums, Weights<N> w, const char* vals) {
  using R = Rows<T, D, M>;
  constexpr int kPitch = Shape<T, D, M>::kPitch;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const T* v = (const T*)(vals + (8 * n + 2 * x + e) * kPitch);
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
            if constexpr (R::kTurned) {
              if (see[k & 1] && 2 * t < M) sums.o[d][k] = fmaf(p[k & 1], to_f32(v[16 * d + g + 8 * (k >> 1)]), sums.o[d][k]);
            } else {
              if (see[k >> 1]) sums.o[d][k] = fmaf(p[k >> 1], to_f32(v[8 * d + 2 * t + (k & 1)]), sums.o[d][k]);
            }
          }
      }
  return sums;
}

// o += s v.  In 16 bits the weights enter as sums of two halves: one rounding
// of 2^-9 to each weight would cost as much precision as the output's own.
template <class T, int D, int M, int N>
__device__ __forceinline__ void values(Rows<T, D, M>& w, const float (&s)[N / 8][4], const char* vals) {
  constexpr int kPitch = Shape<T, D, M>::kPitch;
  const int lane = threadIdx.x & 31;
  if constexpr (sizeof(T) == 2 && M <= 8) {
    // values (dims x keys) times weights (keys x rows)
    const uint32_t at = smem_addr(vals) + ((lane >> 4) * 8 + (lane & 7)) * kPitch + (lane >> 3 & 1) * 16;
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
        load_x4_turned(f, at + n * 16 * kPitch + d * 32);
        mma<T>(w.o[d], f, h0, h1);
        if (M != 4) mma<T>(w.o[d], f, l0, l1);
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    const uint32_t at = smem_addr(vals) + (lane & 15) * kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < N / 16; ++n) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        split<T>(s[2 * n + (e >> 1)][2 * (e & 1)], s[2 * n + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t f[4];
        load_x4_turned(f, at + n * 16 * kPitch + d * 32);
        mma<T>(w.o[2 * d], hi, f[0], f[1]);
        mma<T>(w.o[2 * d + 1], hi, f[2], f[3]);
        mma<T>(w.o[2 * d], lo, f[0], f[1]);
        mma<T>(w.o[2 * d + 1], lo, f[2], f[3]);
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
          const char* v = vals + (8 * n + 2 * x + e) * kPitch + 8 * t;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            const float2 f = *(const float2*)(v + 32 * d);
            w.o[d][0] = fmaf(p0, f.x, w.o[d][0]);
            w.o[d][1] = fmaf(p0, f.y, w.o[d][1]);
            if constexpr (M == 16) {
              w.o[d][2] = fmaf(p1, f.x, w.o[d][2]);
              w.o[d][3] = fmaf(p1, f.y, w.o[d][3]);
            }
          }
        }
  }
}

// One softmax step: N keys, the first of them token `j0`.  `mixed`: some row
// may not see some of them (`known`, from bit `bit0` on: the keys that are tokens).
template <class T, int D, int M, int N>
__device__ __forceinline__ void step(const Attend& p, Rows<T, D, M>& w, const char* keys, const char* vals,
                                     const float* qs, int j0, bool mixed, const uint32_t* known, int bit0) {
  using R = Rows<T, D, M>;
  const int lane = threadIdx.x & 31, t = lane & 3;
  float s[N / 8][4];
  scores<T, D, M, N>(w, s, keys, qs);
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
    const float m = fmaxf(w.m[r], top * p.scale_log2);  // the scale is not negative (see `negate`)
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
    constexpr int kPitch = Shape<T, D, M>::kPitch, kPer = D * (int)sizeof(T) / 4;
    bool careful = false;
    for (int x = lane; x < N * kPer; x += 32)
      careful |= any_nonfinite(*(const uint32_t*)(vals + x / kPer * kPitch + x % kPer * 4), T());
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
      sums = values_one_by_one<T, D, M, N>(sums, weights, vals);
#pragma unroll
      for (int d = 0; d < R::kSums; ++d)
#pragma unroll
        for (int e = 0; e < R::kEach; ++e) w.o[d][e] = sums.o[d][e];
      return;
    }
  }
  values<T, D, M, N>(w, s, vals);
}

// A warp's triples to shared memory: maxima and sums by row, o by (row, dim).
template <class T, int D, int M>
__device__ __forceinline__ void put_rows(Rows<T, D, M>& w, float* ms, float* zs, float* joined) {
  using R = Rows<T, D, M>;
  constexpr int kJoin = Shape<T, D, M>::kJoinPitch;
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
        if (2 * t < M) joined[(2 * t + (e & 1)) * kJoin + 16 * d + g + 8 * (e >> 1)] = w.o[d][e];
      }
    } else {
#pragma unroll
      for (int r = 0; r < R::kOwn; ++r)
        if (g < M) *(float2*)(joined + (g + 8 * r) * kJoin + 8 * d + 2 * t) = make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
    }
  }
}

// ----------------------------------------------------------------- the kernel

// Stores one new token's rows (all heads) in its page.
template <class T>
__device__ void store_token(const Attend& p, int b, int i) {
  const yapd_cache& c = p.a.cache;
  int slot;
  const int t = slot_len(p, b, slot) - p.a.new_tokens + i;
  uint32_t wrong = 0;
  int g = -1, q = 0;
  if (slot < 0) {
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
    if (threadIdx.x == 0) set_status(c.workspace, wrong);
    return;
  }
  constexpr int kVec = 16 / sizeof(T);
  const int per = c.head_dim / kVec, all = c.kv_heads * per;
  T* to = (T*)c.kv + p.a.layer * c.stride_layer + g * c.stride_page + (int64_t)(t - q * c.page_size) * c.kv_heads * c.head_dim;
  T* to_v = to + (int64_t)c.page_size * c.kv_heads * c.head_dim;
  for (int x = threadIdx.x; x < all; x += kThreads) {
    const int h = x / per, d = (x - h * per) * kVec;
    const uint4 k = *(const uint4*)((const T*)p.a.k + b * p.a.k_stride_req + i * p.a.k_stride_pos + h * p.a.k_stride_head + d);
    const uint4 v = *(const uint4*)((const T*)p.a.v + b * p.a.v_stride_req + i * p.a.v_stride_pos + h * p.a.v_stride_head + d);
    *(uint4*)(to + (int64_t)x * kVec) = k;
    *(uint4*)(to_v + (int64_t)x * kVec) = v;
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
    x.x = pack(from_f32<T>(o.x * rz), from_f32<T>(o.y * rz));
    x.y = pack(from_f32<T>(o.z * rz), from_f32<T>(o.w * rz));
    *(uint2*)out = x;
  }
}
__device__ __forceinline__ void write_lse(const Attend& p, int b, int head, int row, float m, float z) {
  if (!p.a.lse) return;
  const int i = (int)div_floor(row, p.groups), h = head * p.group + row - i * p.group;
  p.a.lse[((int64_t)b * p.a.new_tokens + i) * p.a.heads + h] =
      z == 0.0f ? -INFINITY : m * 0.69314718055994531f + logf(z);
}

template <class T, int D, int M>
__global__ void __launch_bounds__(kThreads, Shape<T, D, M>::kFit) attend_kernel(const __grid_constant__ Attend p) {
  using S = Shape<T, D, M>;
  extern __shared__ __align__(128) char smem[];
  char* const ring = smem;
  float* const qs = (float*)(smem + S::kStages * S::kStage);
  int64_t* const places = (int64_t*)(qs + kWarps * S::kQuery);  // [2][kRows]
  __shared__ uint32_t known[S::kStages + 1][S::kWords];  // which keys of a tile are tokens
  __shared__ float ms[kWarps * M], zs[kWarps * M];       // maxima and sums that meet
  __shared__ long long sums[kWarps];
  __shared__ int found[3];
  __shared__ int arrived, bad;  // bad: some table entry so far is no page

  const yapd_cache& c = p.a.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = 31 - __clz(S::kRows / p.hg), keys = 1 << shift;  // keys of a tile
  const int pairs = p.head_groups * p.row_blocks;

  // all units, and where this CTA's share begins
  const int per = (p.a.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.a.B), b1 = min(b0 + per, p.a.B);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    int slot;
    const int len = slot_len(p, b, slot);
    mine += (long long)span_of(p, len, shift).tiles * pairs;
    if (slot < 0 && blockIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_SLOT);
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(~0u, upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 31) sums[warp] = upto;
  if (tid == 0) bad = 0;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) upto += total;
    total += sums[w];
  }
  const long long chunk = (total + gridDim.x - 1) / gridDim.x;
  const long long u0 = min(chunk * blockIdx.x, total), u1 = min(u0 + chunk, total);
  if (u0 < u1 && upto - mine <= u0 && u0 < upto) {
    long long at = upto - mine;
    for (int b = b0;; ++b) {
      int slot;
      const int tiles = span_of(p, slot_len(p, b, slot), shift).tiles;
      const long long n = (long long)tiles * pairs;
      if (u0 < at + n) {
        const long long r = u0 - at;
        found[0] = b;
        found[1] = (int)(r / tiles);
        found[2] = (int)(r % tiles);
        break;
      }
      at += n;
    }
  }
  __syncthreads();

  // requests without a token
  for (int b = blockIdx.x; b < p.a.B; b += gridDim.x) {
    int slot;
    if (slot_len(p, b, slot) > 0) continue;
    for (int x = tid; x < p.a.new_tokens * p.a.heads * (D / 4); x += kThreads) {
      const int r = x / (D / 4), h = r % p.a.heads, i = r / p.a.heads, head = h / p.group;
      const int row = i * p.group + h - head * p.group;
      write_row<T>(p, b, head, row, x % (D / 4) * 4, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 1.0f);
      if (x % (D / 4) == 0) write_lse(p, b, head, row, 0.0f, 0.0f);
    }
  }

  const long long units = u1 - u0;
  Cursor get, load, look;  // the tile that is multiplied, fetched, looked up
  get.b = found[0];
  get.hr = found[1];
  get.tile = found[2];
  if (units > 0) enter(p, get, shift);
  load = look = get;

  // Looking a tile up is two halves, so that the read of the page table is on
  // its way during a product: thread y holds key y's table entry, then notes the
  // token's place, in elements from the layer's start (-1: no token, -2 - i: new
  // token i, read from the call's rows).
  constexpr int kNone = INT32_MIN;
  int entry;
  auto ask = [&](const Cursor& x) {
    const int j = tile_start(x, shift) + tid, low = first_low(p, x.len), sinks = sinks_of(p);
    entry = kNone;
    if (tid < keys && j < x.len && (j >= low || j < sinks))
      entry = max(c.page_table[(int64_t)x.slot * c.max_pages + div_floor(j, p.page)], -1);
  };
  auto note = [&](const Cursor& x, int tile) {
    const int j = tile_start(x, shift) + tid, i = j - (x.len - p.a.new_tokens);
    int64_t place = -1;
    if (entry != kNone) {
      if (p.a.k && i >= 0) {
        place = -2 - i;
      } else if (entry >= 0 && entry < c.pages) {
        const int r = j - (int)div_floor(j, p.page) * c.page_size;
        place = entry * c.stride_page + (int64_t)r * c.kv_heads * D;
      } else {
        bad = 1;
        set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
      }
    }
    if (tid < S::kRows) {
      places[(tile & 1) * S::kRows + tid] = place;
      const uint32_t mask = __ballot_sync(~0u, place != -1);
      if (lane == 0) known[tile & S::kStages][warp] = mask;
    }
  };
  static_assert(S::kStages == 3, "a ring of four masks");
  const int64_t to_v = (int64_t)c.page_size * c.kv_heads * D;
  auto fetch = [&](const Cursor& x, int stage, int tile) {
    const int head0 = x.hr / p.row_blocks * p.hg;
    const T* const base = (const T*)c.kv + p.a.layer * c.stride_layer + head0 * D;
    const int64_t* const at = places + (tile & 1) * S::kRows;
    const uint32_t to = smem_addr(ring + stage * S::kStage);
    constexpr int kVec = 16 / sizeof(T);
    if (!p.a.k || tile_start(x, shift) + keys <= x.len - p.a.new_tokens) {
#pragma unroll
      for (int e = 0; e < S::kLoads; ++e) {
        const int y = tid + e * kThreads, row = y / S::kChunks, ch = y - row * S::kChunks;
        const int64_t place = at[row & (keys - 1)];
        const T* const k = base + max(place, (int64_t)0) + (row >> shift) * D + ch * kVec;
        const uint32_t d = to + row * S::kPitch + ch * 16;
        copy16(d, k, place >= 0);
        copy16(d + S::kHalf, k + to_v, place >= 0);
      }
    } else {
      for (int e = 0; e < S::kLoads; ++e) {
        const int y = tid + e * kThreads, row = y / S::kChunks, ch = y - row * S::kChunks, h = row >> shift;
        const int64_t place = at[row & (keys - 1)];
        const T *k = base, *v = base;
        if (place >= 0) {
          k = base + place + h * D + ch * kVec;
          v = k + to_v;
        } else if (place < -1) {
          const int i = (int)(-2 - place);
          k = (const T*)p.a.k + x.b * p.a.k_stride_req + i * p.a.k_stride_pos + (head0 + h) * p.a.k_stride_head + ch * kVec;
          v = (const T*)p.a.v + x.b * p.a.v_stride_req + i * p.a.v_stride_pos + (head0 + h) * p.a.v_stride_head + ch * kVec;
        }
        const uint32_t d = to + row * S::kPitch + ch * 16;
        copy16(d, k, place != -1);
        copy16(d + S::kHalf, v, place != -1);
      }
    }
  };

  // the pipeline fills: two tiles under way, the third looked up
  for (int s = 0; s < S::kStages; ++s) {
    if (s < units) {
      ask(look);
      note(look, s);
      advance(p, look, shift);
    }
    __syncthreads();
    if (s < S::kStages - 1) {
      if (s < units) {
        fetch(load, s, s);
        advance(p, load, shift);
      }
      copies_commit();
    }
  }
  if (p.a.k)
    for (int x = blockIdx.x; x < p.a.B * p.a.new_tokens; x += gridDim.x)
      store_token<T>(p, x / p.a.new_tokens, x % p.a.new_tokens);

  const int wk_all = kWarps / p.wr, wk = warp / p.wr, wrow = warp - wk * p.wr;
  const int span = S::kRows / wk_all;                    // stage rows of this warp
  const int parts = wk_all / p.hg;                       // warps that share a head's keys
  const int head_in = wk / parts, part = wk - head_in * parts;
  float* const my_qs = qs + warp * S::kQuery;
  Rows<T, D, M> w;
  bool fresh = true, whole = true;
  int stage = 0;
  for (long long it = 0; it < units; ++it) {
    copies_wait<S::kStages - 2>();
    __syncthreads();
    if (it + S::kStages - 1 < units) {
      fetch(load, stage == 0 ? S::kStages - 1 : stage - 1, (int)(it + S::kStages - 1));
      advance(p, load, shift);
    }
    copies_commit();
    const bool more = it + S::kStages < units;
    if (more) ask(look);
    const int head0 = get.hr / p.row_blocks * p.hg, rb = get.hr % p.row_blocks;
    if (fresh) {
      whole = get.tile == 0;
      begin_rows<T, D, M>(p, w, get, head0 + head_in, (rb * p.wr + wrow) * M, my_qs);
      fresh = false;
    }
    {
      const int k0 = tile_start(get, shift);
      // every row sees every key of the tile
      const int first_end = p.a.causal ? get.len - p.a.new_tokens + 1 : get.len;
      const int64_t last_low = p.a.window > 0 ? (int64_t)get.len - p.a.window : 0;
      const bool mixed = bad || k0 + keys > first_end || (k0 < last_low && k0 + keys > p.a.sinks);
      const char* rows = ring + stage * S::kStage + wk * span * S::kPitch;
      for (int x = 0; x < span; x += S::kStep) {
        const int j0 = k0 + part * span + x;
        if (j0 >= get.len) break;
        step<T, D, M, S::kStep>(p, w, rows + x * S::kPitch, rows + S::kHalf + x * S::kPitch, my_qs, j0, mixed,
                                known[it & S::kStages], part * span + x);
      }
    }
    if (more) {
      note(look, (int)(it + S::kStages));
      advance(p, look, shift);
    }
    const bool last_tile = get.tile + 1 == get.span.tiles;
    if (last_tile || it + 1 == units) {
      // the warps' triples meet in the stage that was just read
      whole = whole && last_tile;
      __syncthreads();
      float* const joined = (float*)(ring + stage * S::kStage);
      put_rows<T, D, M>(w, ms + warp * M, zs + warp * M, joined + warp * M * S::kJoinPitch);
      __syncthreads();
      const int block_rows = p.wr * M, rows_here = min(block_rows, p.rows - rb * block_rows);
      // which CTAs hold parts of this (request, head group, row block)
      const long long u = u0 + it, start = u - get.tile, end = start + get.span.tiles;
      const int c0 = (int)(start / chunk), c1 = (int)((end - 1) / chunk);
      constexpr int64_t kPart = kMaxRows * (D + 2);
      float* const mine_at = p.partials + ((int64_t)blockIdx.x * 2 + (start > u0 ? 1 : 0)) * kPart;
      for (int x = tid; x < p.hg * rows_here * (D / 4); x += kThreads) {
        const int rr = x / (D / 4), d = x - rr * (D / 4), hi = rr / rows_here, row = rr - hi * rows_here;
        const int rm = row & (M - 1), first = (hi * parts) * p.wr + row / M;
        float m = -INFINITY;
        for (int k = 0; k < parts; ++k) m = fmaxf(m, ms[(first + k * p.wr) * M + rm]);
        const float base = m == -INFINITY ? 0.0f : m;
        float z = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < parts; ++k) {
          const int y = (first + k * p.wr) * M + rm;
          const float f = ex2(ms[y] - base);
          const float4 v = *(const float4*)(joined + y * S::kJoinPitch + 4 * d);
          z = fmaf(f, zs[y], z);
          o.x = fmaf(f, v.x, o.x);
          o.y = fmaf(f, v.y, o.y);
          o.z = fmaf(f, v.z, o.z);
          o.w = fmaf(f, v.w, o.w);
        }
        if (whole) {
          const float rz = z == 0.0f ? 0.0f : 1.0f / z;
          write_row<T>(p, get.b, head0 + hi, rb * block_rows + row, 4 * d, o, rz);
          if (d == 0) write_lse(p, get.b, head0 + hi, rb * block_rows + row, m, z);
        } else {
          float* const to = mine_at + rr * (D + 2);
          *(float2*)(to + 4 * d) = make_float2(o.x, o.y);
          *(float2*)(to + 4 * d + 2) = make_float2(o.z, o.w);
          if (d == 0) *(float2*)(to + D) = make_float2(m, z);
        }
      }
      if (!whole) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const int before = atomicAdd(p.counters + c0, 1);
          arrived = before == c1 - c0;
          if (arrived) p.counters[c0] = 0;  // for the next call; nobody else comes
        }
        __syncthreads();
        if (arrived) {
          __threadfence();
          // the parts in their order: CTA c0's is its second unless its share begins with it
          const int n = c1 - c0 + 1;
          const float* const parts0 = p.partials + (c0 * 2 + (start > c0 * chunk ? 1 : 0)) * kPart;
          const float* const parts1 = p.partials + (int64_t)c0 * 2 * kPart;
          auto part_at = [&](int k) { return k == 0 ? parts0 : parts1 + k * 2 * kPart; };
          // maxima and sums: a warp per row, lanes over the parts
          for (int rr = warp; rr < p.hg * rows_here; rr += kWarps) {
            float m = -INFINITY, z = 0.0f;
            for (int k = lane; k < n; k += 32) m = fmaxf(m, __ldcg(part_at(k) + rr * (D + 2) + D));
#pragma unroll
            for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
            const float base = m == -INFINITY ? 0.0f : m;
            for (int k = lane; k < n; k += 32) {
              const float2 mz = __ldcg((const float2*)(part_at(k) + rr * (D + 2) + D));
              z = fmaf(ex2(mz.x - base), mz.y, z);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) z += __shfl_xor_sync(~0u, z, d);
            if (lane == 0) {
              const int hi = rr / rows_here;
              ms[rr] = base;
              zs[rr] = z == 0.0f ? 0.0f : 1.0f / z;
              write_lse(p, get.b, head0 + hi, rb * block_rows + rr - hi * rows_here, m, z);
            }
          }
          __syncthreads();
          for (int x = tid; x < p.hg * rows_here * (D / 2); x += kThreads) {
            const int rr = x / (D / 2), d = x - rr * (D / 2), hi = rr / rows_here;
            const float base = ms[rr], rz = zs[rr];
            float2 o = make_float2(0.0f, 0.0f);
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
              const float* const y = part_at(k) + rr * (D + 2);
              const float f = ex2(__ldcg(y + D) - base);
              const float2 v = __ldcg((const float2*)(y + 2 * d));
              o.x = fmaf(f, v.x, o.x);
              o.y = fmaf(f, v.y, o.y);
            }
            const int full = rb * block_rows + rr - hi * rows_here, i = (int)div_floor(full, p.groups);
            const int h = (head0 + hi) * p.group + full - i * p.group;
            T* const out = (T*)p.a.out + get.b * p.a.out_stride_req + i * p.a.out_stride_pos + h * p.a.out_stride_head + 2 * d;
            if constexpr (sizeof(T) == 4)
              *(float2*)out = make_float2(o.x * rz, o.y * rz);
            else
              *(uint32_t*)out = pack(from_f32<T>(o.x * rz), from_f32<T>(o.y * rz));
          }
        }
      }
      fresh = true;
    }
    advance(p, get, shift);
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
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

template <class T, int D, int M>
int launch(Attend& p, cudaStream_t st) {
  int grid = 0;
  const int rc = grid_of<T, D, M>(grid);
  if (rc != YAPD_OK) return rc;
  p.wr = M < 16 || p.rows <= 16 ? 1 : p.rows <= 32 ? 2 : 4;
  p.row_blocks = (p.rows + M * p.wr - 1) / (M * p.wr);
  // Key heads of a unit: the rows of several heads of a token lie side by side
  // in its page.  Few requests are shared out by heads first, so that fewer
  // CTAs hold parts of the same sums.
  const int kvh = p.a.cache.kv_heads;
  p.hg = 4 / p.wr;
  while (p.hg > 1 && (kvh % p.hg || (int64_t)p.a.B * (kvh / p.hg) * p.row_blocks < grid / 2)) p.hg /= 2;
  p.head_groups = kvh / p.hg;
  attend_kernel<T, D, M><<<grid, kThreads, Shape<T, D, M>::kSmem, st>>>(p);
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
  return round_up(kMaxCtas * 4, 256) + (size_t)kMaxCtas * 2 * kMaxRows * (c.head_dim + 2) * 4;
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
  // a negative scale is a positive one of the negative queries
  p.negate = std::signbit(a.scale) ? dt == YAPD_DTYPE_F32 ? 0x80000000u : 0x80008000u : 0u;
  p.scale_log2 = std::fabs(a.scale) * 1.4426950408889634f;
  char* const scratch = (char*)a.cache.workspace + kHeaderBytes + pages_scratch_bytes(a.cache);
  p.counters = (int*)scratch;
  p.partials = (float*)(scratch + round_up(kMaxCtas * 4, 256));
  switch (dt) {
    case YAPD_DTYPE_F32: return launch_dim<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch_dim<__half>(p, (cudaStream_t)stream);
    default: return launch_dim<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
