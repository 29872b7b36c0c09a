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
  int wr;            // warps along the rows: 1, 2, 4
  int hg;            // key heads of a unit: 1, 2, 4
  int head_groups, row_blocks;
  float scale_log2;
  int* counters;     // (gridDim): arrivals at a cut piece that starts in the CTA
  float* partials;   // (gridDim, 2, kMaxRows, D + 2)
};

// ------------------------------------------------------------ shapes by type

template <class T, int D>
struct Shape {
  // rows of keys in a stage, and as many of values
  static constexpr int kRows = sizeof(T) == 2 ? (D <= 64 ? 128 : 64) : (D == 32 ? 64 : 32);
  static constexpr int kStep = kRows / kWarps < 32 ? kRows / kWarps : 32;  // keys of one softmax step
  static constexpr int kPitch = D * sizeof(T) + 16;  // bytes: eight rows' 16-byte chunks fall in different banks
  static constexpr int kHalf = kRows * kPitch;
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kStages = 3;
  static constexpr int kChunks = D * sizeof(T) / 16;
  static constexpr int kLoads = kRows * kChunks / kThreads;
  static constexpr int kJoinPitch = D + 4;           // floats
  static constexpr int kQ = sizeof(T) == 4 ? kWarps * 16 * (D + 4) * 4 : 0;
  static constexpr int kMaxKeys = kRows;             // keys of a tile: kRows / hg
  static constexpr int kSmem = kStages * kStage + kQ + (kStages + 1) * kMaxKeys * 8 + 2 * kWarps * 16 * 4;
  static_assert(kWarps * 16 * kJoinPitch * 4 <= kStage, "the join fits a stage");
  static_assert(kRows * kChunks % kThreads == 0, "");
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

// One thread's share of a warp's 16 rows, as the matrix instructions lay an
// accumulator out: rows g and g + 8, columns 8n + 2t and 8n + 2t + 1
// (g = lane / 4, t = lane % 4).
template <class T, int D>
struct Rows {
  uint32_t q[sizeof(T) == 2 ? D / 16 : 1][4];
  float o[D / 8][4];
  float m[2], z[2];
  int end[2], low[2];  // visible: [low, end) and [0, sinks)
};

template <class T, int D>
__device__ __forceinline__ const T* query_at(const Attend& p, int b, int head, int row) {
  const int i = (int)div_floor(row, p.groups), h = head * p.group + row - i * p.group;
  return (const T*)p.a.q + b * p.a.q_stride_req + i * p.a.q_stride_pos + h * p.a.q_stride_head;
}

// The queries of 16 rows from `row0` on (rows past the last one: zeros).
template <class T, int D>
__device__ __forceinline__ void begin_rows(const Attend& p, Rows<T, D>& w, const Cursor& c, int head, int row0,
                                           float* qs) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) w.o[n][e] = 0.0f;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + g + 8 * r, i = (int)div_floor(row, p.groups);
    const int place = c.len - p.a.new_tokens + i;
    w.m[r] = -INFINITY;
    w.z[r] = 0.0f;
    w.end[r] = p.a.causal ? min(c.len, place + 1) : c.len;
    const int64_t low = p.a.window > 0 ? place - p.a.window + 1 : 0;
    w.low[r] = low > 0 ? (int)low : 0;
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row0 + g + 8 * r;
      const T* q = query_at<T, D>(p, c.b, head, row);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w.q[k][r + 2 * e] = row < p.rows ? *(const uint32_t*)(q + 16 * k + 8 * e + 2 * t) : 0u;
    }
  } else {
    __syncwarp();
    for (int x = lane; x < 16 * (D / 4); x += 32) {
      const int r = x / (D / 4), d = x % (D / 4) * 4, row = row0 + r;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row < p.rows) v = *(const float4*)(query_at<T, D>(p, c.b, head, row) + d);
      *(float4*)(qs + r * (D + 4) + d) = v;
    }
    __syncwarp();
  }
}

// Scores of N/8 * 8 keys whose rows start at `keys`.
template <class T, int D, int N>
__device__ __forceinline__ void scores(const Rows<T, D>& w, float (&s)[N / 8][4], const char* keys, const float* qs) {
  constexpr int kPitch = Shape<T, D>::kPitch;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
  if constexpr (sizeof(T) == 2) {
    const uint32_t at = smem_addr(keys) + ((lane >> 4) * 8 + (lane & 7)) * kPitch + (lane >> 3 & 1) * 16;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int n = 0; n < N / 16; ++n) {
        uint32_t f[4];
        load_x4(f, at + n * 16 * kPitch + k * 32);
        mma<T>(s[2 * n], w.q[k], f[0], f[1]);
        mma<T>(s[2 * n + 1], w.q[k], f[2], f[3]);
      }
  } else {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      const float4 q0 = *(const float4*)(qs + g * (D + 4) + d), q1 = *(const float4*)(qs + (g + 8) * (D + 4) + d);
#pragma unroll
      for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 k = *(const float4*)(keys + (8 * n + 2 * t + e) * kPitch + d * 4);
          s[n][e] = fmaf(q0.w, k.w, fmaf(q0.z, k.z, fmaf(q0.y, k.y, fmaf(q0.x, k.x, s[n][e]))));
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

template <int N>
struct Weights {
  float s[N / 8][4];
  bool see[N / 8][4];
};

// o += s v with the weight 0 of a hidden token kept away from its value, which
// may be anything: element by element.
template <int D>
struct Sums {
  float o[D / 8][4];
};
template <class T, int D, int N>
__device__ __noinline__ Sums<D> values_one_by_one(Sums<D> sums, Weights<N> weights, const char* vals) {
  constexpr int kPitch = Shape<T, D>::kPitch;
  auto& o = sums.o;
  auto& s = weights.s;
  auto& see = weights.see;
  const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int from = (lane & ~3) + x;  // the lane that holds columns 2x, 2x + 1 of these rows
        const float p0 = __shfl_sync(~0u, s[n][e], from), p1 = __shfl_sync(~0u, s[n][2 + e], from);
        const bool s0 = __shfl_sync(~0u, (int)see[n][e], from), s1 = __shfl_sync(~0u, (int)see[n][2 + e], from);
        const T* v = (const T*)(vals + (8 * n + 2 * x + e) * kPitch);
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f = to_f32(v[8 * d + 2 * t + c]);
            if (s0) o[d][c] = fmaf(p0, f, o[d][c]);
            if (s1) o[d][2 + c] = fmaf(p1, f, o[d][2 + c]);
          }
      }
  return sums;
}

// o += s v, the weights as sums of two 16-bit halves: one rounding of 2^-9 to
// each weight would cost as much precision as the output's own.
template <class T, int D, int N>
__device__ __forceinline__ void values(float (&o)[D / 8][4], const float (&s)[N / 8][4], const char* vals) {
  constexpr int kPitch = Shape<T, D>::kPitch;
  const int lane = threadIdx.x & 31;
  if constexpr (sizeof(T) == 2) {
    const uint32_t at = smem_addr(vals) + (lane & 15) * kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < N / 16; ++n) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split<T>(s[2 * n + (e >> 1)][2 * (e & 1)], s[2 * n + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t f[4];
        load_x4_turned(f, at + n * 16 * kPitch + d * 32);
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
          const float p0 = __shfl_sync(~0u, s[n][e], from), p1 = __shfl_sync(~0u, s[n][2 + e], from);
          const char* v = vals + (8 * n + 2 * x + e) * kPitch + 8 * t;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            const float2 f = *(const float2*)(v + 32 * d);
            o[d][0] = fmaf(p0, f.x, o[d][0]);
            o[d][1] = fmaf(p0, f.y, o[d][1]);
            o[d][2] = fmaf(p1, f.x, o[d][2]);
            o[d][3] = fmaf(p1, f.y, o[d][3]);
          }
        }
  }
}

// One softmax step: N keys, the first of them token `j0`.  `mixed`: some row
// may not see some of them (`known`: offsets of the keys, negative: no token).
template <class T, int D, int N>
__device__ __forceinline__ void step(const Attend& p, Rows<T, D>& w, const char* keys, const char* vals, const float* qs,
                                     int j0, bool mixed, const int64_t* known) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  float s[N / 8][4];
  scores<T, D, N>(w, s, keys, qs);
  bool see[N / 8][4];
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
  if (mixed) {
    const int sinks = sinks_of(p);
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int x = 8 * n + 2 * t + (e & 1), j = j0 + x, r = e >> 1;
        see[n][e] = known[x] != -1 && j < w.end[r] && (j >= w.low[r] || j < sinks);
        if (!see[n][e]) s[n][e] = -INFINITY;
      }
  }
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
  float fix[2], base[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 1));
    top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 2));
    const float m = fmaxf(w.m[r], top[r]);
    base[r] = m == -INFINITY ? 0.0f : m;
    fix[r] = ex2(w.m[r] - base[r]);
    w.m[r] = m;
  }
  if (__any_sync(~0u, fix[0] != 1.0f || fix[1] != 1.0f)) {
#pragma unroll
    for (int r = 0; r < 2; ++r) w.z[r] *= fix[r];
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) w.o[d][e] *= fix[e >> 1];
  }
#pragma unroll
  for (int n = 0; n < N / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[n][e] = ex2(s[n][e] - base[e >> 1]);
      w.z[e >> 1] += s[n][e];
    }
  bool careful = false;
  if (mixed) {
    // a value that is not finite reaches only the rows that see its token
    constexpr int kPitch = Shape<T, D>::kPitch;
    for (int x = lane; x < N * (D * (int)sizeof(T) / 4); x += 32) {
      const int r = x / (D * (int)sizeof(T) / 4), d = x % (D * (int)sizeof(T) / 4);
      const uint32_t f = *(const uint32_t*)(vals + r * kPitch + 4 * d);
      if constexpr (sizeof(T) == 2)
        careful |= any_nonfinite(f, T());
      else
        careful |= (f & 0x7f800000u) == 0x7f800000u;
    }
    careful = __any_sync(~0u, careful);
  }
  if (careful) {
    // by value: nothing of the common path has an address
    Sums<D> sums;
    Weights<N> weights;
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums.o[d][e] = w.o[d][e];
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        weights.s[n][e] = s[n][e];
        weights.see[n][e] = see[n][e];
      }
    sums = values_one_by_one<T, D, N>(sums, weights, vals);
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) w.o[d][e] = sums.o[d][e];
  } else {
    values<T, D, N>(w.o, s, vals);
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

template <class T, int D>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const __grid_constant__ Attend p) {
  using S = Shape<T, D>;
  extern __shared__ __align__(128) char smem[];
  char* const ring = smem;
  float* const qs = (float*)(smem + S::kStages * S::kStage);
  int64_t* const known = (int64_t*)(smem + S::kStages * S::kStage + S::kQ);  // [kStages + 1][kMaxKeys]
  float* const ms = (float*)(known + (S::kStages + 1) * S::kMaxKeys);        // [kWarps][16], then z
  float* const zs = ms + kWarps * 16;
  __shared__ long long sums[kWarps + 1];
  __shared__ int found[4];
  __shared__ int arrived, bad;  // bad: some table entry so far is no page

  const yapd_cache& c = p.a.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = 31 - __clz(S::kRows / p.hg);  // keys of a tile, as a power of two
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
  Cursor get, put;  // the tile to be multiplied, the tile whose tokens are looked up
  get.b = found[0];
  get.hr = found[1];
  get.tile = found[2];
  if (units > 0) enter(p, get, shift);
  put = get;
  Cursor load = get;  // the tile to be fetched

  // the places of a tile's tokens: elements from the layer's start, -1: none,
  // -2 - i: new token i, read from the call's rows
  constexpr int kLook = S::kMaxKeys > kThreads ? S::kMaxKeys / kThreads : 1;
  int page_of[kLook];
  auto look = [&](const Cursor& x) {
    const int k0 = tile_start(x, shift), low = first_low(p, x.len), sinks = sinks_of(p);
#pragma unroll
    for (int e = 0; e < kLook; ++e) {
      const int j = k0 + tid + e * kThreads;
      page_of[e] = INT32_MIN;  // no token
      if (tid + e * kThreads < (1 << shift) && j < x.len && (j >= low || j < sinks)) {
        page_of[e] = c.page_table[(int64_t)x.slot * c.max_pages + div_floor(j, p.page)];
        if (page_of[e] == INT32_MIN) page_of[e] = -1;
      }
    }
  };
  auto note = [&](const Cursor& x, int at) {
    const int k0 = tile_start(x, shift);
    bool wrong = false;
#pragma unroll
    for (int e = 0; e < kLook; ++e) {
      const int y = tid + e * kThreads;
      if (y >= (1 << shift)) break;
      const int g = page_of[e], j = k0 + y, i = j - (x.len - p.a.new_tokens);
      int64_t place = -1;
      if (g != INT32_MIN) {
        if (p.a.k && i >= 0) {
          place = -2 - i;
        } else if (g >= 0 && g < c.pages) {
          const int r = j - (int)div_floor(j, p.page) * c.page_size;
          place = g * c.stride_page + (int64_t)r * c.kv_heads * D;
        } else {
          wrong = true;
        }
      }
      known[at * S::kMaxKeys + y] = place;
    }
    if (wrong) {
      bad = 1;
      set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
    }
  };
  auto fetch = [&](const Cursor& x, int stage, int at) {
    const int head0 = x.hr / p.row_blocks * p.hg;
    const T* base = (const T*)c.kv + p.a.layer * c.stride_layer;
    const int64_t to_v = (int64_t)c.page_size * c.kv_heads * D;
    const uint32_t to = smem_addr(ring + stage * S::kStage);
#pragma unroll 4
    for (int e = 0; e < S::kLoads; ++e) {
      const int y = tid + e * kThreads, row = y / S::kChunks, ch = y - row * S::kChunks;
      const int kk = row & ((1 << shift) - 1), h = head0 + (row >> shift);
      const int64_t place = known[at * S::kMaxKeys + kk];
      const T* k = base + h * D;
      const T* v = k;
      if (place >= 0) {
        k += place;
        v = k + to_v;
      } else if (place < -1) {
        const int i = (int)(-2 - place);
        k = (const T*)p.a.k + x.b * p.a.k_stride_req + i * p.a.k_stride_pos + h * p.a.k_stride_head;
        v = (const T*)p.a.v + x.b * p.a.v_stride_req + i * p.a.v_stride_pos + h * p.a.v_stride_head;
      }
      const uint32_t d = to + row * S::kPitch + ch * 16;
      copy16(d, k + ch * (16 / sizeof(T)), place != -1);
      copy16(d + S::kHalf, v + ch * (16 / sizeof(T)), place != -1);
    }
  };

  // the pipeline fills: tiles 0 .. kStages - 2 are under way, the next is looked up
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int s = 0; s < S::kStages; ++s)
    if (s < units) {
      look(put);
      note(put, s);
      advance(p, put, shift);
    }
  __syncthreads();
  for (int s = 0; s < S::kStages - 1; ++s) {
    if (s < units) {
      fetch(load, s, s);
      advance(p, load, shift);
    }
    copies_commit();
  }
  if (p.a.k)
    for (int x = blockIdx.x; x < p.a.B * p.a.new_tokens; x += gridDim.x)
      store_token<T>(p, x / p.a.new_tokens, x % p.a.new_tokens);

  const int wk_all = kWarps / p.wr, wk = warp / p.wr, wrow = warp - wk * p.wr;
  const int span = S::kRows / wk_all;                    // stage rows of this warp
  const int parts = wk_all / p.hg;                       // warps that share a head's keys
  const int head_in = wk / parts, part = wk - head_in * parts;
  float* const my_qs = qs + warp * 16 * (D + 4);
  Rows<T, D> w;
  bool fresh = true, whole = true;
  for (long long it = 0; it < units; ++it) {
    copies_wait<S::kStages - 2>();
    __syncthreads();
    const int stage = (int)(it % S::kStages), at = (int)(it % (S::kStages + 1));
    if (it + S::kStages - 1 < units) {
      fetch(load, (int)((it + S::kStages - 1) % S::kStages), (int)((it + S::kStages - 1) % (S::kStages + 1)));
      advance(p, load, shift);
    }
    copies_commit();
    const bool more = it + S::kStages < units;
    if (more) look(put);
    const int head0 = get.hr / p.row_blocks * p.hg, rb = get.hr % p.row_blocks;
    const int row0 = (rb * p.wr + wrow) * 16;
    if (fresh) {
      whole = get.tile == 0;
      begin_rows<T, D>(p, w, get, head0 + head_in, row0, my_qs);
      fresh = false;
    }
    {
      const int k0 = tile_start(get, shift), keys = 1 << shift;
      // every row sees every key of the tile
      const int first_end = p.a.causal ? get.len - p.a.new_tokens + 1 : get.len;
      const int64_t last_low = p.a.window > 0 ? (int64_t)get.len - p.a.window : 0;
      const bool mixed = bad || k0 + keys > first_end || (k0 < last_low && k0 + keys > p.a.sinks);
      const char* rows = ring + stage * S::kStage + wk * span * S::kPitch;
      const int64_t* places = known + at * S::kMaxKeys + part * span;
      for (int x = 0; x < span; x += S::kStep) {
        const int j0 = k0 + part * span + x;
        if (j0 >= get.len) break;
        step<T, D, S::kStep>(p, w, rows + x * S::kPitch, rows + S::kHalf + x * S::kPitch, my_qs, j0, mixed, places + x);
      }
    }
    if (more) {
      const int to = (int)((it + S::kStages) % (S::kStages + 1));
      note(put, to);  // the place of tile it - 1: every warp has passed this iteration's barrier
      advance(p, put, shift);
    }
    const bool last_tile = get.tile + 1 == get.span.tiles;
    if (last_tile || it + 1 == units) {
      // the warps' triples meet in the stage that was just read
      whole = whole && last_tile;
      __syncthreads();
      float* const joined = (float*)(ring + stage * S::kStage);
      {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          w.z[r] += __shfl_xor_sync(~0u, w.z[r], 1);
          w.z[r] += __shfl_xor_sync(~0u, w.z[r], 2);
          if (t == 0) {
            ms[warp * 16 + g + 8 * r] = w.m[r];
            zs[warp * 16 + g + 8 * r] = w.z[r];
          }
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *(float2*)(joined + (warp * 16 + g + 8 * r) * S::kJoinPitch + 8 * d + 2 * t) =
                make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
        }
      }
      __syncthreads();
      const int rows_here = min(p.wr * 16, p.rows - rb * p.wr * 16);
      // which CTAs hold parts of this (request, head group, row block)
      const long long u = u0 + it, start = u - get.tile, end = start + get.span.tiles;
      const long long c0 = start / chunk, c1 = (end - 1) / chunk;
      float* const mine_at =
          p.partials + ((int64_t)blockIdx.x * 2 + (start > u0 ? 1 : 0)) * kMaxRows * (D + 2);
      for (int x = tid; x < p.hg * rows_here * (D / 4); x += kThreads) {
        const int rr = x / (D / 4), d = x - rr * (D / 4), hi = rr / rows_here, row = rr - hi * rows_here;
        const int r16 = row & 15, first = (hi * parts) * p.wr + (row >> 4);
        float m = -INFINITY;
        for (int k = 0; k < parts; ++k) m = fmaxf(m, ms[(first + k * p.wr) * 16 + r16]);
        const float base = m == -INFINITY ? 0.0f : m;
        float z = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < parts; ++k) {
          const int y = (first + k * p.wr) * 16 + r16;
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
          write_row<T>(p, get.b, head0 + hi, rb * p.wr * 16 + row, 4 * d, o, rz);
          if (d == 0) write_lse(p, get.b, head0 + hi, rb * p.wr * 16 + row, m, z);
        } else {
          float* const to = mine_at + (hi * rows_here + row) * (D + 2);
          *(float2*)(to + 4 * d) = make_float2(o.x, o.y);
          *(float2*)(to + 4 * d + 2) = make_float2(o.z, o.w);
          if (d == 0) *(float2*)(to + D) = make_float2(m, z);
        }
      }
      if (!whole) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const int n = (int)(c1 - c0) + 1, before = atomicAdd(p.counters + c0, 1);
          arrived = before == n - 1;
          if (arrived) p.counters[c0] = 0;  // for the next call; nobody else comes
        }
        __syncthreads();
        if (arrived) {
          __threadfence();
          // CTA c0 left it in its second place unless the piece begins with it
          const float* const from0 = p.partials + (c0 * 2 + (start > c0 * chunk ? 1 : 0)) * kMaxRows * (D + 2);
          const float* const rest = p.partials + (c0 + 1) * 2 * kMaxRows * (D + 2);
          const int n = (int)(c1 - c0);
          for (int x = tid; x < p.hg * rows_here * (D / 2); x += kThreads) {
            const int rr = x / (D / 2), d = x - rr * (D / 2), hi = rr / rows_here, row = rr - hi * rows_here;
            const float* const a = from0 + rr * (D + 2);
            const float* const b = rest + rr * (D + 2);
            float m = __ldcg(a + D);
            for (int k = 0; k < n; ++k) m = fmaxf(m, __ldcg(b + (int64_t)k * 2 * kMaxRows * (D + 2) + D));
            const float base = m == -INFINITY ? 0.0f : m;
            float z = 0.0f;
            float2 o = make_float2(0.0f, 0.0f);
#pragma unroll 4
            for (int k = -1; k < n; ++k) {
              const float* const y = k < 0 ? a : b + (int64_t)k * 2 * kMaxRows * (D + 2);
              const float2 mz = __ldcg((const float2*)(y + D)), v = __ldcg((const float2*)(y + 2 * d));
              const float f = ex2(mz.x - base);
              z = fmaf(f, mz.y, z);
              o.x = fmaf(f, v.x, o.x);
              o.y = fmaf(f, v.y, o.y);
            }
            const float rz = z == 0.0f ? 0.0f : 1.0f / z;
            const int full = rb * p.wr * 16 + row, i = (int)div_floor(full, p.groups);
            const int h = (head0 + hi) * p.group + full - i * p.group;
            T* const out = (T*)p.a.out + get.b * p.a.out_stride_req + i * p.a.out_stride_pos + h * p.a.out_stride_head + 2 * d;
            if constexpr (sizeof(T) == 4)
              *(float2*)out = make_float2(o.x * rz, o.y * rz);
            else
              *(uint32_t*)out = pack(from_f32<T>(o.x * rz), from_f32<T>(o.y * rz));
            if (d == 0) write_lse(p, get.b, head0 + hi, full, m, z);
          }
        }
      }
      fresh = true;
    }
    advance(p, get, shift);
  }
}

// ------------------------------------------------------------------ the host

template <class T, int D>
int launch(Attend& p, cudaStream_t st) {
  using S = Shape<T, D>;
  int dev = 0, sms = 0, fit = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return YAPD_ERR_NO_DEVICE;
  static std::atomic<int> grids[64];  // per device, found at its first call
  if (dev >= 64) return YAPD_ERR_NO_DEVICE;
  int grid = grids[dev].load(std::memory_order_relaxed);
  if (!grid) {
    if (cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, attend_kernel<T, D>, kThreads, S::kSmem) != cudaSuccess ||
        fit < 1)
      return YAPD_ERR_LAUNCH;
    grid = sms * fit < kMaxCtas ? sms * fit : kMaxCtas;
    grids[dev].store(grid, std::memory_order_relaxed);
  }
  attend_kernel<T, D><<<grid, kThreads, S::kSmem, st>>>(p);
  return launched();
}

template <class T>
int launch_dim(Attend& p, cudaStream_t st) {
  switch (p.a.cache.head_dim) {
    case 32: return launch<T, 32>(p, st);
    case 64: return launch<T, 64>(p, st);
    case 96: return launch<T, 96>(p, st);
    default: return launch<T, 128>(p, st);
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
  p.wr = p.rows <= 16 ? 1 : p.rows <= 32 ? 2 : 4;
  p.row_blocks = (p.rows + 16 * p.wr - 1) / (16 * p.wr);
  const int most = kWarps / p.wr;
  p.hg = most >= 4 && kvh % 4 == 0 ? 4 : most >= 2 && kvh % 2 == 0 ? 2 : 1;
  p.head_groups = kvh / p.hg;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  char* const scratch = (char*)a.cache.workspace + kHeaderBytes + pages_scratch_bytes(a.cache);
  p.counters = (int*)scratch;
  p.partials = (float*)(scratch + round_up(kMaxCtas * 4, 256));
  switch (dt) {
    case YAPD_DTYPE_F32: return launch_dim<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch_dim<__half>(p, (cudaStream_t)stream);
    default: return launch_dim<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
