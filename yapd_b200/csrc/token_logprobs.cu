// Log probabilities of given tokens, the entropy and the most likely tokens.
//
// With m the largest logit, t = sum e^(x - m) over all tokens but one that has it,
// and w = sum e^(x - m) (x - m): log p = x - m - ln(1 + t) and the entropy is
// ln(1 + t) - w / (1 + t). Where one token has nearly all the mass, t is the
// result: no sum of it has a 1 in it, whose last place would be the error. The alternatives need
// no sort of the row: of the maxima of P disjoint parts of it, the n-th largest
// has n tokens at or above it, so only tokens that reach it can be among the
// first n. In a row without structure -P ln(1 - n / P) do, 9 for n = 8 and P = 32;
// they are listed and ranked.
//
// A warp holds up to 1056 vectors of 16 bytes in its registers and makes all
// passes over them alone; the parts are its lanes. A longer row, or few rows,
// are shared out over the warps of a CTA or of a cluster; the parts are then the
// lanes of a CTA, and the CTAs' tokens are merged at the end.
#include <cooperative_groups.h>

#include "select_common.cuh"
#include "serve_common.cuh"

namespace serve {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kFit = 3;             // CTAs of an SM: 168 registers a thread
constexpr int kVecs = 33;           // vectors of a lane at a time
constexpr int kSome = 18;           // of a lane of a longer row's share, four CTAs to an SM
constexpr int kSomeFit = 4;
constexpr int kFew = 3;             // of a lane of a short share: less code to fetch
constexpr int kGroup = 3;           // vectors between two looks at the end
constexpr int kList = 256;          // tokens that are ranked at once
constexpr int kKept = 64;           // vectors that are kept for it
constexpr int kMaxCtas = 8;         // of a cluster
constexpr int kMaxTop = YAPD_LOGPROBS_MAX_TOP;

using Key = unsigned long long;  // (logit, lower id first) in ascending order; 0: none

struct Logprobs {
  yapd_logprobs_args a;
  int warps;  // of a row: 1, or kWarps times the cluster's CTAs
};

__device__ __forceinline__ Key key_of(float f, uint32_t id) {
  const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);  // -0 and 0 are equal
  return (Key)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | ~id;
}
__device__ __forceinline__ float logit_of(Key k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int id_of(Key k) { return (int)~(uint32_t)k; }

// The elements of a vector as pairs of 32-bit numbers.
template <class T>
struct Pairs;
template <>
struct Pairs<float> {
  static constexpr int kCount = 2;
  __device__ static float2 get(const uint4& v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  __device__ static uint32_t hidden() { return 0xff800000u; }
  // the larger halves of two words, and a word's largest number
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ static float largest(uint32_t a) { return __uint_as_float(a); }
  // all ones in the halves of `a` that are above those of `b`
  __device__ static uint32_t above(uint32_t a, uint32_t b) { return __uint_as_float(a) > __uint_as_float(b) ? ~0u : 0u; }
};
template <>
struct Pairs<__nv_bfloat16> {
  static constexpr int kCount = 4;
  __device__ static float2 get(const uint4& v, int i) {
    const uint32_t u = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  __device__ static uint32_t hidden() { return 0xff80ff80u; }
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float largest(uint32_t a) {
    return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
  }
  __device__ static uint32_t above(uint32_t a, uint32_t b) {
    return __hgt2_mask(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  }
};
template <>
struct Pairs<__half> {
  static constexpr int kCount = 4;
  __device__ static float2 get(const uint4& v, int i) {
    uint32_t u = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  __device__ static uint32_t hidden() { return 0xfc00fc00u; }
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float largest(uint32_t a) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&a));
    return fmaxf(f.x, f.y);
  }
  __device__ static uint32_t above(uint32_t a, uint32_t b) {
    return __hgt2_mask(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Sums over a part of a row against its own maximum: w = sum e^(x - m) (x - m),
// tail = sum e^(x - m) without one token that has the maximum.
struct Part {
  float m, tail, w;
};
// `b` joins `a`: both against the larger maximum.
__device__ __forceinline__ Part join(const Part& a, const Part& b) {
  const bool left = a.m >= b.m;
  const Part &big = left ? a : b, &small = left ? b : a;
  if (small.m == -INFINITY) return Part{big.m, a.tail + b.tail, a.w + b.w};  // nothing, or NaN
  const float d = fmaxf(small.m - big.m, -1e30f), f = expf(d), z = 1.0f + small.tail;
  return Part{big.m, fmaf(f, z, big.tail), fmaf(f, fmaf(d, z, small.w), big.w)};
}

// A lane's largest logit, and the first of the group of vectors that has it.
constexpr int kRim = -1, kNowhere = -2;
struct Most {
  float value;
  int group;
};

// A row's vectors: its first one begins at the 16-byte boundary at or below the
// row, its last one ends at or after the row's end.
template <class T>
struct Row {
  static constexpr int kVec = 16 / (int)sizeof(T);
  const uint4* base;
  const T* x;
  int lead, V, vectors;  // lead: elements of the first vector before the row

  __device__ Row(const yapd_logprobs_args& a, int r) {
    x = (const T*)a.logits + (int64_t)r * a.stride_row;
    lead = (int)((uintptr_t)x % 16 / sizeof(T));
    base = (const uint4*)((uintptr_t)x & ~(uintptr_t)15);
    V = a.V;
    vectors = (V + lead + kVec - 1) / kVec;
  }
  // A vector that ends outside the row: what is not of the row is hidden, and not read.
  __device__ uint4 edge(int j) const {
    const int first = j * kVec - lead;
    union {
      uint4 v;
      T e[kVec];
    } u;
    u.v.x = u.v.y = u.v.z = u.v.w = Pairs<T>::hidden();
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (first + i >= 0 && first + i < V) u.e[i] = x[first + i];
    return u.v;
  }
};

// Element e of a word.
template <class T>
__device__ __forceinline__ float word_part(uint32_t w, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const float2 f = Pairs<T>::get(make_uint4(w, 0, 0, 0), 0);
    return e ? f.y : f.x;
  }
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
  return x;
}

// Vectors of a row in a warp's registers, the k-th of a lane k * 32 + lane from v0 on.
template <class T, int kVecs>
struct Tile {
  static constexpr int kVec = Row<T>::kVec, kPairs = Pairs<T>::kCount;
  uint4 x[kVecs];
  uint4 rim;  // lane 0: the row's first vector if it begins before it; lane 1: its last if it ends after it
  int v0, v1, end;
  bool rimmed;  // whether a lane has one

  __device__ __forceinline__ void load(const Row<T>& row, int from, int to) {
    v0 = from;
    v1 = min(to, from + kVecs * 32);
    const int lane = threadIdx.x & 31;
    const int inner0 = row.lead ? 1 : 0, inner1 = (row.V + row.lead) / kVec;  // vectors wholly of the row
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const uint32_t h = Pairs<T>::hidden();
      x[k] = make_uint4(h, h, h, h);
    }
#pragma unroll
    for (int g = 0; g < kVecs; g += kGroup)
      if (v0 + g * 32 < v1)
#pragma unroll
        for (int k = g; k < g + kGroup; ++k) {
          const int j = v0 + k * 32 + lane;
          if (j >= inner0 && j < min(inner1, v1)) x[k] = __ldg(row.base + j);
        }
    const bool head = v0 == 0 && v1 > 0 && inner0, tail = inner1 < row.vectors && inner1 >= max(v0, inner0) && inner1 < v1;
    rimmed = head || tail;
    end = inner1;
    rim = make_uint4(Pairs<T>::hidden(), Pairs<T>::hidden(), Pairs<T>::hidden(), Pairs<T>::hidden());
    if ((head && lane == 0) || (tail && lane == 1)) rim = row.edge(lane == 0 ? 0 : inner1);
  }

  __device__ __forceinline__ static uint32_t word_of(const uint4& v) {
    return Pairs<T>::larger(Pairs<T>::larger(v.x, v.y), Pairs<T>::larger(v.z, v.w));
  }
  // The lane's largest logit. In 16 bits a word holds two maxima, and `at` the group of each.
  __device__ __forceinline__ Most largest() {
    constexpr uint32_t kBoth = sizeof(T) == 2 ? 0x10001u : 1u, kRimAt = kVecs / kGroup;
    uint32_t word = Pairs<T>::hidden(), at = 0;
    const auto see = [&](uint32_t w, uint32_t g) {
      const uint32_t more = Pairs<T>::above(w, word);
      at = (at & ~more) | (g * kBoth & more);
      word = Pairs<T>::larger(word, w);
    };
#pragma unroll
    for (int g = 0; g < kVecs; g += kGroup)
      if (v0 + g * 32 < v1) {
        uint32_t w = word_of(x[g]);
#pragma unroll
        for (int k = g + 1; k < g + kGroup; ++k) w = Pairs<T>::larger(w, word_of(x[k]));
        see(w, g / kGroup);
      }
    if (rimmed) see(word_of(rim), kRimAt);
    // 16-bit elements are converted anew: kept as 32-bit numbers they would not fit the registers.
    if constexpr (sizeof(T) == 2)
#pragma unroll
      for (int k = 0; k < kVecs; ++k) asm volatile("" : "+r"(x[k].x), "+r"(x[k].y), "+r"(x[k].z), "+r"(x[k].w));
    if constexpr (sizeof(T) == 2) {
      const float2 f = Pairs<T>::get(make_uint4(word, 0, 0, 0), 0);
      at = f.x >= f.y ? at & 0xffffu : at >> 16;
    }
    return Most{Pairs<T>::largest(word), at == kRimAt ? kRim : v0 + (int)at * kGroup * 32};
  }
  // Adds the lane's sums against `base`: two each, for the even and the odd elements. Group `skip` is left out of z2.
  __device__ __forceinline__ void add(float base, int skip, unsigned long long& z2, unsigned long long& w2) const {
    const unsigned long long minus = yapd::f2_pack(-base, -base), log2e = yapd::f2_pack(yapd::kLog2e, yapd::kLog2e);
    const auto one = [&](const uint4& v) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 f = Pairs<T>::get(v, i);
        float dx, dy, tx, ty;
        const unsigned long long d = yapd::f2_add(yapd::f2_pack(f.x, f.y), minus);
        yapd::f2_unpack(d, dx, dy);
        yapd::f2_unpack(f2_mul(d, log2e), tx, ty);
        const unsigned long long e = yapd::f2_pack(ex2(tx), ex2(ty));
        z2 = yapd::f2_add(z2, e);
        // a hidden token adds 0 and not 0 times infinity
        w2 = yapd::f2_fma(e, yapd::f2_pack(fmaxf(dx, -1e30f), fmaxf(dy, -1e30f)), w2);
      }
    };
#pragma unroll
    for (int g = 0; g < kVecs; g += kGroup)
      if (v0 + g * 32 < v1) {
        const unsigned long long before = z2;
#pragma unroll
        for (int k = g; k < g + kGroup; ++k) one(x[k]);
        if (v0 + g * 32 == skip) z2 = before;
      }
    if (rimmed) {
      const unsigned long long before = z2;
      one(rim);
      if (skip == kRim) z2 = before;
    }
  }
  // The lane's second largest logit (the largest one again if two are equal).
  __device__ __forceinline__ float second() const {
    float a = -INFINITY, b = -INFINITY;
    const auto see = [&](const uint4& v) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 f = Pairs<T>::get(v, i);
        b = fmaxf(b, fminf(a, f.x));
        a = fmaxf(a, f.x);
        b = fmaxf(b, fminf(a, f.y));
        a = fmaxf(a, f.y);
      }
    };
#pragma unroll
    for (int k = 0; k < kVecs; ++k) see(x[k]);
    if (rimmed) see(rim);
    return b;
  }
  // Calls f(vector, its number) for each vector with a token that reaches `reach`.
  template <class F>
  __device__ __forceinline__ void reaching(float reach, F f) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < kVecs; g += kGroup)
      if (v0 + g * 32 < v1)
#pragma unroll
        for (int k = g; k < g + kGroup; ++k) {
          const float most = Pairs<T>::largest(word_of(x[k]));
          if (most >= reach && most > -INFINITY) f(x[k], v0 + k * 32 + lane);
        }
    const float most = Pairs<T>::largest(word_of(rim));
    if (most >= reach && most > -INFINITY) f(rim, lane == 0 ? 0 : end);
  }
};

// The token of a warp's vectors that its tail leaves out: one lane that has the
// maximum leaves its group out of its sum, and the warp adds the group's other
// tokens, one to a lane (five more instructions to a group of vectors and a read that the
// sums hide: 2 us of 52 for 8192 rows of 8194).
template <class T>
struct Apart {
  static constexpr int kVec = Row<T>::kVec;
  static_assert(kGroup * kVec <= 32, "a token to a lane");
  float m;
  int skip;     // the lane's group that is left out
  float other;  // the lane's token of that group

  // `most`: the lane's, of vectors [.., to) of the row.
  __device__ __forceinline__ Apart(const Row<T>& row, const Most& most, int to) {
    const int lane = threadIdx.x & 31;
    m = warp_max(most.value);
    const uint32_t have = __ballot_sync(~0u, most.value == m);
    // nothing but -inf and NaN: none is left out
    const int owner = m > -INFINITY ? __ffs(have) - 1 : -1, group = __shfl_sync(~0u, most.group, max(owner, 0));
    skip = lane == owner ? group : kNowhere;
    other = -INFINITY;
    const int inner0 = row.lead ? 1 : 0, inner1 = (row.V + row.lead) / kVec, i = lane / kVec;
    int j = group + i * 32 + owner, first = inner0, end = i < kGroup ? min(inner1, to) : 0;
    if (group == kRim) {
      j = owner == 0 ? 0 : inner1;
      first = 0;
      end = i == 0 ? row.vectors : 0;
    }
    const int id = j * kVec - row.lead + lane % kVec;
    if (owner >= 0 && j >= first && j < end && id >= 0 && id < row.V) other = to_f32(row.x[id]);
  }

  // The warp's sums from its lanes'.
  __device__ __forceinline__ Part join(unsigned long long z2, unsigned long long w2) const {
    const int lane = threadIdx.x & 31, out = __ffs(__ballot_sync(~0u, other == m)) - 1;
    Part p{m, lane == out || other == -INFINITY ? 0.0f : ex2((other - m) * yapd::kLog2e), 0.0f};
    float x, y;
    yapd::f2_unpack(z2, x, y);
    p.tail += x + y;
    yapd::f2_unpack(w2, p.w, y);
    p.w += y;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      p.tail += __shfl_xor_sync(~0u, p.tail, d);
      p.w += __shfl_xor_sync(~0u, p.w, d);
    }
    return p;
  }
};

// What the threads of a row put together for its alternatives: a warp's, or a CTA's.
struct Candidates {
  uint4 data[kKept];
  int number[kKept];   // of the vector
  Key list[kList];
  Key top[kMaxTop];
  int vectors, count;  // as many as reach the threshold, held or not
};

// The 32 largest of two lists, one ascending over the lanes and one descending: ascending.
__device__ __forceinline__ float merge_top(float up, float down) {
  const int lane = threadIdx.x & 31;
  float x = fmaxf(up, down);
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float y = __shfl_xor_sync(~0u, x, d);
    x = lane & d ? fmaxf(x, y) : fminf(x, y);
  }
  return x;
}

// The n largest of `count` keys, in their order, to `top`: all different (but
// for 0, none), each one's place is the number of those above it.
template <int kSize>
__device__ __forceinline__ void place(const Key* keys, int count, int n, Key* top, int rank) {
  for (int i = rank; i < count; i += kSize) {
    const Key k = keys[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) above += keys[j] > k;
    if (k && above < n) top[above] = k;
  }
}

// The most likely tokens of vectors [v0, v1) of a row, by `kSize` threads that
// `sync` brings together: to c.top. `tile(f)` calls f for the vectors that reach
// `reach`, the n-th largest maximum of the parts.
template <class T, int kSize, class Sync, class Tiles>
__device__ __forceinline__ void find_top(const Row<T>& row, int v0, int v1, int n, float reach, Candidates& c, int rank,
                                         Sync sync, Tiles tiles) {
  constexpr int kWord = 4 / (int)sizeof(T), kVec = Row<T>::kVec;
  if (rank < kMaxTop) c.top[rank] = 0;
  if (rank == 0) c.vectors = c.count = 0;
  sync();
  tiles([&](const uint4& v, int j) {
    const int at = atomicAdd(&c.vectors, 1);
    if (at < kKept) {
      c.data[at] = v;
      c.number[at] = j;
    }
  });
  sync();
  // their tokens, a word of a vector to a thread
  for (int i = rank; i < min(c.vectors, kKept) * 4; i += kSize) {
    const uint32_t word = ((const uint32_t*)c.data)[i];
    const int id = c.number[i >> 2] * kVec - row.lead + (i & 3) * kWord;
#pragma unroll
    for (int e = 0; e < kWord; ++e) {
      const float g = word_part<T>(word, e);
      if (g >= reach && g > -INFINITY) {
        const int at = atomicAdd(&c.count, 1);
        if (at < kList) c.list[at] = key_of(g, id + e);
      }
    }
  }
  sync();
  if (c.vectors <= kKept && c.count <= kList) {
    place<kSize>(c.list, c.count, n, c.top, rank);
    sync();
    return;
  }
  // more of them than are held: the largest one below the last, one by one
  Key last = ~0ull;
  for (int k = 0; k < n; ++k) {
    Key best = 0;
    for (int j = v0 + rank; j < v1; j += kSize)
      for (int i = 0; i < kVec; ++i) {
        const int id = j * kVec - row.lead + i;
        const float g = id >= 0 && id < row.V ? to_f32(row.x[id]) : -INFINITY;
        const Key x = key_of(g, id);
        if (g > -INFINITY && x < last && x > best) best = x;
      }
    if (rank == 0) c.top[k] = 0;
    sync();
    atomicMax(&c.top[k], best);
    sync();
    last = c.top[k];
  }
}

// A row's values, by the warp that holds its sums and its tokens.
template <class T>
__device__ __forceinline__ void write(const yapd_logprobs_args& a, const Row<T>& row, int r, const Part& all, Key top) {
  const int lane = threadIdx.x & 31;
  // NaN makes the tail NaN; nothing but -inf leaves no maximum
  const bool fine = all.m > -INFINITY && all.m < INFINITY && all.tail < INFINITY;
  const float lz = log1pf(all.tail);
  if (lane == 0) {
    if (a.targets) {
      const int64_t t = a.targets[r];
      a.logprob[r] = fine && t >= 0 && t < a.V ? to_f32(row.x[t]) - all.m - lz : NAN;
    }
    if (a.entropy) a.entropy[r] = fine ? lz - all.w / (1.0f + all.tail) : NAN;
  }
  if (lane < a.top_n) {
    a.top_ids[(int64_t)r * a.top_n + lane] = fine && top ? id_of(top) : -1;
    a.top_logprobs[(int64_t)r * a.top_n + lane] = !fine ? NAN : top ? logit_of(top) - all.m - lz : -INFINITY;
  }
}

// Rows of one tile: a warp to each, nothing to wait for. 8192 rows of 8194 16-bit
// logits (134 MB; 21 us at the copy rate) take 37 us, with eight alternatives 52
// us: 2500 and 3300 instructions a row at half of the issue slots, since a row in
// registers leaves room for twelve warps to an SM. Four warps to such a row: 53
// and 79 us.
template <class T, bool kTop, int kVecs>
__global__ void __launch_bounds__(kThreads, kFit) rows_kernel(const __grid_constant__ Logprobs p) {
  __shared__ Candidates candidates[kTop ? kWarps : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x * kWarps + warp; r < p.a.R; r += (int64_t)gridDim.x * kWarps) {
    const Row<T> row(p.a, (int)r);
    Tile<T, kVecs> tile;
    tile.load(row, 0, row.vectors);
    const Most most = tile.largest();
    const Apart<T> apart(row, most, row.vectors);
    const float mine = most.value, m = apart.m;
    unsigned long long z2 = 0, w2 = 0;
    tile.add(m == -INFINITY ? 0.0f : m, apart.skip, z2, w2);
    Key top = 0;
    if (kTop) {
      const int n = p.a.top_n;
      const float firsts = yapd::warp_bitonic_asc_f(mine);
      float reach = __shfl_sync(~0u, firsts, 32 - n);
      if (n > (kVecs == kFew ? 8 : 20)) {
        // The n-th largest of the lanes' 64 first and second logits lies closer to the
        // n-th largest of all, where n comes near the number of lanes or the lanes
        // have few tokens (7312 rows of 459, 32 alternatives: 24 us, and 105 us with
        // the first ones alone, which every token reached). It is the largest, over
        // all i, of the smaller of the i-th first and the (n - i)-th second one.
        const float seconds = yapd::warp_bitonic_asc_f(tile.second());
        const int rest = n - lane;  // lane i takes i first ones
        const float f = __shfl_sync(~0u, firsts, (32 - lane) & 31), g = __shfl_sync(~0u, seconds, (32 - rest) & 31);
        const float both = fminf(lane ? f : INFINITY, rest > 0 ? g : INFINITY);
        reach = fmaxf(reach, warp_max(rest >= 0 ? both : -INFINITY));
      }
      Candidates& c = candidates[warp];
      find_top<T, 32>(row, 0, row.vectors, n, reach, c, lane, [] { __syncwarp(); }, [&](auto f) { tile.reaching(reach, f); });
      top = c.top[lane];
    }
    write(p.a, row, (int)r, apart.join(z2, w2), top);
    __syncwarp();
  }
}

struct Meeting {
  float mine[kThreads];
  Part part[kWarps];
  Part all;          // what the cluster's first CTA reads of this one, with c.top
  Part parts[kMaxCtas];
  Candidates c;
  Key lists[kMaxCtas * kMaxTop];
  Key sorted[kMaxTop];
};

// A CTA or a cluster to each row, a warp to each share of its vectors. kOnce: a
// tile holds the share. 4096 rows of 8192 32-bit logits (134 MB) take 31 us, 66 % of
// the copy rate; 384 rows of 128256 16-bit ones, read twice and a third time for
// the alternatives, take 38 us without them and 52 us with them (15 us at the copy
// rate); one row of 6563 takes 6 us, two meetings of the cluster's CTAs and launch.
template <class T, bool kTop, int kVecs, bool kOnce>
__global__ void __launch_bounds__(kThreads, kSomeFit) row_kernel(const __grid_constant__ Logprobs p) {
  __shared__ Meeting mt;
  const yapd_logprobs_args& a = p.a;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), me = cluster.block_rank(), n = a.top_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x / ctas;
  const Row<T> row(a, r);
  const int share = (row.vectors + p.warps - 1) / p.warps;
  const auto first = [&](int w) { return min((me * kWarps + w) * share, row.vectors); };
  const int v0 = first(warp), v1 = first(warp + 1);
  Tile<T, kVecs> tile;
  // f() for each tile of the share
  const auto tiles = [&](auto f) {
    if (kOnce) {
      f();
    } else {
      for (int v = v0; v < v1; v += kVecs * 32) {
        tile.load(row, v, v1);
        f();
      }
    }
  };
  if (kOnce) tile.load(row, v0, v1);
  Most most{-INFINITY, kNowhere};
  tiles([&] {
    const Most x = tile.largest();
    if (x.value > most.value) most = x;
  });
  if (kTop) mt.mine[tid] = yapd::warp_bitonic_asc_f(most.value);
  const Apart<T> apart(row, most, v1);
  const float m = apart.m;
  unsigned long long z2 = 0, w2 = 0;
  tiles([&] { tile.add(m == -INFINITY ? 0.0f : m, apart.skip, z2, w2); });
  Part part = apart.join(z2, w2);
  if (lane == 0) mt.part[warp] = part;
  __syncthreads();
  if (kTop) {
    // the 32 largest of the lanes' maxima
    static_assert(kWarps == 4, "two and two");
    const float a0 = merge_top(mt.mine[lane], mt.mine[63 - lane]), a1 = merge_top(mt.mine[64 + lane], mt.mine[127 - lane]);
    const float reach = __shfl_sync(~0u, merge_top(a0, __shfl_sync(~0u, a1, 31 - lane)), 32 - n);
    find_top<T, kThreads>(row, first(0), first(kWarps), n, reach, mt.c, tid, [] { __syncthreads(); },
                          [&](auto f) { tiles([&] { tile.reaching(reach, f); }); });
  }
  if (warp == 0)
    for (int w = 1; w < kWarps; ++w) part = join(part, mt.part[w]);
  if (ctas == 1) {
    if (warp == 0) write(a, row, r, part, kTop ? mt.c.top[lane] : 0);
    return;
  }
  if (tid == 0) mt.all = part;
  cluster.sync();
  if (me == 0) {
    if (tid < ctas) mt.parts[tid] = cluster.map_shared_rank(&mt, tid)->all;
    if (kTop) {
      if (tid < kMaxTop) mt.sorted[tid] = 0;
      for (int i = tid; i < ctas * n; i += kThreads) mt.lists[i] = cluster.map_shared_rank(&mt, i / n)->c.top[i % n];
    }
    __syncthreads();
    if (kTop) {
      place<kThreads>(mt.lists, ctas * n, n, mt.sorted, tid);
      __syncthreads();
    }
    if (warp == 0) {
      for (int o = 1; o < ctas; ++o) part = join(part, mt.parts[o]);
      write(a, row, r, part, kTop ? mt.sorted[lane] : 0);
    }
  }
  cluster.sync();  // the others' memory lives until here
}

// The kernel of a configuration by whether there are alternatives.
template <class T, int kVecs>
auto rows_kernel_of(bool top) {
  return top ? rows_kernel<T, true, kVecs> : rows_kernel<T, false, kVecs>;
}
template <class T, int kVecs, bool kOnce>
auto row_kernel_of(bool top) {
  return top ? row_kernel<T, true, kVecs, kOnce> : row_kernel<T, false, kVecs, kOnce>;
}

template <class T>
int launch(Logprobs& p, cudaStream_t st) {
  const yapd_logprobs_args& a = p.a;
  const int64_t vectors = (a.V + 2 * Row<T>::kVec - 2) / Row<T>::kVec;
  constexpr int kSlots = 148 * kFit * kWarps;  // warps that run at once
  // One warp where it holds the row and there are rows for half of the warps,
  // or the row is short; else a CTA, and a cluster for so few rows that they
  // leave half of the GPU idle, as long as every lane has four vectors. (With
  // 384 rows of 128256: clusters of four that hold the rows take 58 us, single
  // CTAs that read them again out of L2 52 us; 4096 rows of 8192 in 32 bits: 31 us
  // with 18 vectors to a lane, 39 with 33, 37 with 9.)
  constexpr int kTile = kVecs * 32;
  if (vectors <= kTile && (a.R >= kSlots / 2 || vectors <= 64)) {
    const int ctas = (a.R + kWarps - 1) / kWarps, most = 148 * kFit;
    const auto kernel = vectors <= kFew * 32 ? rows_kernel_of<T, kFew>(a.top_n) : rows_kernel_of<T, kVecs>(a.top_n);
    kernel<<<ctas < most ? ctas : most, kThreads, 0, st>>>(p);
    return launched();
  }
  int ctas = 1;
  while (ctas < kMaxCtas && (int64_t)a.R * ctas < 148 * kSomeFit / 2 && vectors > (int64_t)ctas * kWarps * 128) ctas *= 2;
  if ((int64_t)a.R * ctas > INT32_MAX) return YAPD_ERR_BAD_SHAPE;
  p.warps = ctas * kWarps;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.R * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute size{};
  size.id = cudaLaunchAttributeClusterDimension;
  size.val.clusterDim.x = ctas;
  size.val.clusterDim.y = size.val.clusterDim.z = 1;
  cfg.attrs = &size;
  cfg.numAttrs = ctas > 1;
  const int64_t share = (vectors + p.warps - 1) / p.warps;
  const auto kernel = share <= kFew * 32 ? row_kernel_of<T, kFew, true>(a.top_n)
                      : share <= kSome * 32 ? row_kernel_of<T, kSome, true>(a.top_n)
                                            : row_kernel_of<T, kSome, false>(a.top_n);
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return YAPD_ERR_LAUNCH;
  return launched();
}

}  // namespace
}  // namespace serve

using namespace serve;

extern "C" int yapd_token_logprobs(const yapd_logprobs_args* args, void* stream) {
  if (!args) return YAPD_ERR_NULL_POINTER;
  const yapd_logprobs_args& a = *args;
  if (a.R < 0 || a.V < 1 || a.top_n < 0 || a.top_n > YAPD_LOGPROBS_MAX_TOP) return YAPD_ERR_BAD_SHAPE;
  if (a.V > YAPD_LOGPROBS_MAX_V) return YAPD_ERR_V_TOO_LARGE;
  if (a.logits_dtype != YAPD_DTYPE_F32 && a.logits_dtype != YAPD_DTYPE_BF16 && a.logits_dtype != YAPD_DTYPE_F16)
    return YAPD_ERR_BAD_DTYPE;
  if (a.R > 1 && a.stride_row < a.V) return YAPD_ERR_BAD_SHAPE;
  if (a.R == 0) return YAPD_OK;
  if (!a.logits || (a.targets && !a.logprob) || (a.top_n && (!a.top_logprobs || !a.top_ids)))
    return YAPD_ERR_NULL_POINTER;
  if ((uintptr_t)a.logits % dtype_size(a.logits_dtype)) return YAPD_ERR_MISALIGNED;
  Logprobs p{a, 1};
  switch (a.logits_dtype) {
    case YAPD_DTYPE_F32: return launch<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch<__half>(p, (cudaStream_t)stream);
    default: return launch<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
