// Log probabilities of given tokens, the entropy and the most likely tokens.
//
// With m the largest logit, z = sum e^(x - m) and w = sum e^(x - m) (x - m):
// log p(t) = x_t - m - ln z and the entropy is ln z - w / z, which has no
// cancellation where one token has nearly all the mass. The alternatives need
// no sort of the row: of the maxima of 64 disjoint parts of it, the n-th largest
// has n tokens at or above it, so only tokens that reach it can be among the
// first n. About 1.2 n do in a row without structure; they are listed and
// ranked against one another.
//
// A row is held in the registers of one CTA, or of a cluster of up to eight that
// meet in the first one's shared memory, so it is read once; a row too long for
// that is read a second time, out of L2.
#include <cooperative_groups.h>

#include "select_common.cuh"
#include "serve_common.cuh"

namespace serve {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kVecs = 8;         // 16-byte vectors of a thread at a time
constexpr int kBuckets = kThreads / 4;
constexpr int kList = 512;       // tokens that can be ranked at once
constexpr int kMaxCluster = 8;
constexpr int kMaxTop = YAPD_LOGPROBS_MAX_TOP;

using Key = unsigned long long;  // (logit, lower id first) in ascending order; 0: none

struct Logprobs {
  yapd_logprobs_args a;
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
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of a part of a row against its own maximum.
struct Part {
  float m, z, w;
};
// `b` joins `a`: both against the larger maximum.
__device__ __forceinline__ Part join(const Part& a, const Part& b) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -INFINITY) return Part{r.m, a.z + b.z, a.w + b.w};
  const float da = fmaxf(a.m - r.m, -1e30f), db = fmaxf(b.m - r.m, -1e30f);  // a factor of 0 and not of NaN
  const float fa = expf(da), fb = expf(db);
  r.z = fmaf(fa, a.z, fb * b.z);
  r.w = fa * fmaf(da, a.z, a.w) + fb * fmaf(db, b.z, b.w);
  return r;
}

// A row's vectors: its first one begins at the 16-byte boundary at or below the
// row, its last one ends at or after the row's end.
template <class T>
struct Row {
  static constexpr int kVec = 16 / (int)sizeof(T);
  const uint4* base;
  const T* x;
  int lead, V, vectors;  // elements of the first vector before the row

  __device__ Row(const yapd_logprobs_args& a, int r) {
    x = (const T*)a.logits + (int64_t)r * a.stride_row;
    lead = (int)((uintptr_t)x % 16 / sizeof(T));
    base = (const uint4*)((uintptr_t)x & ~(uintptr_t)15);
    V = a.V;
    vectors = (V + lead + kVec - 1) / kVec;
  }
  // Vector j; what is not of the row is hidden, and not read.
  __device__ uint4 get(int j) const {
    const int first = j * kVec - lead;
    if (first >= 0 && first + kVec <= V) return __ldg(base + j);
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

struct Shared {
  float bucket[kBuckets];
  float z[kThreads / 32], w[kThreads / 32];
  float threshold;
  int listed;
  Key list[kList];
  // what the cluster's first CTA reads of this one
  Part part;
  Key top[kMaxTop];
  Key all[kMaxCluster * kMaxTop];
  Key best[kThreads / 32];
};

// Ranks `n` keys of `from`, all different: the k-th largest to to[k], k < most.
__device__ __forceinline__ void rank(const Key* from, int n, Key* to, int most) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const Key mine = from[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += from[j] > mine;
    if (mine && above < most) to[above] = mine;
  }
}

template <class T, bool kOnce, bool kTop>
__global__ void __launch_bounds__(kThreads, 4) row_kernel(const __grid_constant__ Logprobs p) {
  __shared__ Shared sh;
  const yapd_logprobs_args& a = p.a;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), me = cluster.block_rank();
  const int r = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> row(a, r);
  constexpr int kVec = Row<T>::kVec, kPairs = Pairs<T>::kCount, kTile = kThreads * kVecs;
  const int share = (row.vectors + ctas - 1) / ctas, v0 = me * share, v1 = min(v0 + share, row.vectors);

  uint4 x[kVecs];
  auto load = [&](int first) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int j = first + k * kThreads + tid;
      const uint32_t h = Pairs<T>::hidden();
      x[k] = make_uint4(h, h, h, h);
      if (j < v1) x[k] = row.get(j);
    }
  };
  // The passes convert the elements anew: kept from one to the next as 32-bit
  // numbers they would not fit the registers.
  auto forget = [&]() {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) asm volatile("" : "+r"(x[k].x), "+r"(x[k].y), "+r"(x[k].z), "+r"(x[k].w));
  };
  // whether any lane of the warp has a k-th vector
  auto any = [&](int first, int k) { return first + k * kThreads + warp * 32 < v1; };

  // the largest logit, by thread, by four threads, of all
  uint32_t word = Pairs<T>::hidden();
  for (int first = v0; first < v1; first += kTile) {
    load(first);
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      if (any(first, k))
        word = Pairs<T>::larger(word, Pairs<T>::larger(Pairs<T>::larger(x[k].x, x[k].y), Pairs<T>::larger(x[k].z, x[k].w)));
  }
  const float mine = Pairs<T>::largest(word);
  float top = fmaxf(mine, __shfl_xor_sync(~0u, mine, 1));
  top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
  if ((lane & 3) == 0) sh.bucket[tid >> 2] = top;
  if (tid == 0) {
    sh.listed = 0;
    sh.threshold = -INFINITY;
  }
  __syncthreads();
  float m = fmaxf(sh.bucket[lane], sh.bucket[lane + 32]);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  if (kTop) {
    // the four threads of a bucket compare it with a quarter of the others each
    int above = 0;
#pragma unroll
    for (int j = 0; j < kBuckets / 4; ++j) {
      const int o = j * 4 + (tid & 3);
      const float f = sh.bucket[o];
      above += f > top || (f == top && o < tid >> 2);
    }
    above += __shfl_xor_sync(~0u, above, 1);
    above += __shfl_xor_sync(~0u, above, 2);
    if (above == a.top_n - 1) sh.threshold = top;
    __syncthreads();
  }

  // sums, and the tokens that reach the threshold
  const float reach = kTop ? sh.threshold : 0.0f, base = m == -INFINITY ? 0.0f : m;
  unsigned long long z2 = 0, w2 = 0;  // two sums each, for the even and the odd elements
  const unsigned long long minus = yapd::f2_pack(-base, -base), log2e = yapd::f2_pack(yapd::kLog2e, yapd::kLog2e);
  for (int first = v0; first < v1; first += kTile) {
    if (!kOnce) load(first);
    forget();
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      if (any(first, k))
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float2 f = Pairs<T>::get(x[k], i);
          float dx, dy, tx, ty;
          const unsigned long long d = yapd::f2_add(yapd::f2_pack(f.x, f.y), minus);
          yapd::f2_unpack(d, dx, dy);
          asm("{.reg .b64 t; mul.rn.f32x2 t, %2, %3; mov.b64 {%0, %1}, t;}" : "=f"(tx), "=f"(ty) : "l"(d), "l"(log2e));
          const unsigned long long e = yapd::f2_pack(ex2(tx), ex2(ty));
          z2 = yapd::f2_add(z2, e);
          // a hidden token adds 0 and not 0 times infinity
          w2 = yapd::f2_fma(e, yapd::f2_pack(fmaxf(dx, -1e30f), fmaxf(dy, -1e30f)), w2);
        }
    if (kTop) {
      // the warp looks through the vectors of each of its threads that has a candidate
      uint32_t some = __ballot_sync(~0u, mine >= reach && mine > -INFINITY);
      for (; some; some &= some - 1) {
        const int from = __ffs(some) - 1;
#pragma unroll
        for (int y = lane; y < kVecs * kVec; y += 32) {
          const int j = first + y / kVec * kThreads + warp * 32 + from, id = j * kVec - row.lead + y % kVec;
          if (j < v1 && id >= 0 && id < row.V) {
            const float g = to_f32(row.x[id]);
            if (g >= reach && g > -INFINITY) {
              const int at = atomicAdd(&sh.listed, 1);
              if (at < kList) sh.list[at] = key_of(g, id);
            }
          }
        }
      }
    }
  }
  float z, w, y;
  yapd::f2_unpack(z2, z, y);
  z += y;
  yapd::f2_unpack(w2, w, y);
  w += y;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    z += __shfl_xor_sync(~0u, z, d);
    w += __shfl_xor_sync(~0u, w, d);
  }
  if (lane == 0) {
    sh.z[warp] = z;
    sh.w[warp] = w;
  }
  if (kTop && tid < kMaxTop) sh.top[tid] = 0;
  __syncthreads();
  if (kTop) {
    const int n = sh.listed;
    if (n <= kList) {
      rank(sh.list, n, sh.top, a.top_n);
    } else {
      // more equal logits than the list holds: the largest below the last one, one by one
      Key last = ~0ull;
      for (int k = 0; k < a.top_n; ++k) {
        Key best = 0;
#pragma unroll 1
        for (int j = v0 + tid; j < v1; j += kThreads) {
          const uint4 v = row.get(j);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float2 f = Pairs<T>::get(v, i);
            const Key c = key_of(f.x, j * kVec - row.lead + 2 * i), d = key_of(f.y, j * kVec - row.lead + 2 * i + 1);
            if (f.x > -INFINITY && c < last && c > best) best = c;
            if (f.y > -INFINITY && d < last && d > best) best = d;
          }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
          const Key o = __shfl_xor_sync(~0u, best, d);
          best = o > best ? o : best;
        }
        if (lane == 0) sh.best[warp] = best;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < kThreads / 32; ++v) best = sh.best[v] > best ? sh.best[v] : best;
        if (tid == 0) sh.top[k] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  if (tid == 0) {
    Part part{m, 0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < kThreads / 32; ++v) {
      part.z += sh.z[v];
      part.w += sh.w[v];
    }
    sh.part = part;
  }

  // the cluster's first CTA puts the row together
  const Key* best = sh.top;
  Part all;
  if (ctas > 1) {
    cluster.sync();
    if (me == 0) {
      if (kTop) {
        for (int i = tid; i < ctas * a.top_n; i += kThreads)
          sh.all[i] = cluster.map_shared_rank(&sh, i / a.top_n)->top[i % a.top_n];
        __syncthreads();
        if (tid < kMaxTop) sh.list[tid] = 0;
        __syncthreads();
        rank(sh.all, ctas * a.top_n, sh.list, a.top_n);
        best = sh.list;
      }
      all = sh.part;
      for (int o = 1; o < ctas; ++o) all = join(all, cluster.map_shared_rank(&sh, o)->part);
    }
    cluster.sync();  // the others' memory lives until here
    if (me != 0) return;
  } else {
    __syncthreads();
    all = sh.part;
  }
  // NaN or +inf make z NaN; nothing but -inf leaves no maximum
  const bool fine = all.m > -INFINITY && all.z > 0.0f && all.z < INFINITY;
  const float lz = logf(all.z);
  if (tid == 0) {
    if (a.targets) {
      const int64_t t = a.targets[r];
      a.logprob[r] = fine && t >= 0 && t < a.V ? to_f32(row.x[t]) - all.m - lz : NAN;
    }
    if (a.entropy) a.entropy[r] = fine ? lz - all.w / all.z : NAN;
  }
  if (kTop && tid < a.top_n) {
    const Key k = best[tid];
    a.top_ids[(int64_t)r * a.top_n + tid] = fine && k ? id_of(k) : -1;
    a.top_logprobs[(int64_t)r * a.top_n + tid] = !fine ? NAN : k ? logit_of(k) - all.m - lz : -INFINITY;
  }
}

template <class T>
int launch(const Logprobs& p, cudaStream_t st) {
  const yapd_logprobs_args& a = p.a;
  const int64_t vectors = (a.V + 2 * Row<T>::kVec - 2) / Row<T>::kVec;
  // Few rows: a cluster to each, as long as every thread has a vector of it;
  // a row that one CTA's registers do not hold: as many as do.
  int ctas = 1;
  while (ctas < kMaxCluster && (vectors > (int64_t)ctas * kThreads * kVecs ||
                                ((int64_t)a.R * ctas < 2 * 148 && vectors > (int64_t)ctas * kThreads)))
    ctas *= 2;
  if ((int64_t)a.R * ctas > INT32_MAX) return YAPD_ERR_BAD_SHAPE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.R * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute size{};
  size.id = cudaLaunchAttributeClusterDimension;
  size.val.clusterDim.x = ctas;
  size.val.clusterDim.y = size.val.clusterDim.z = 1;
  cfg.attrs = &size;
  cfg.numAttrs = 1;
  const bool once = (vectors + ctas - 1) / ctas <= kThreads * kVecs;
  const auto kernel = once ? a.top_n ? row_kernel<T, true, true> : row_kernel<T, true, false>
                           : a.top_n ? row_kernel<T, false, true> : row_kernel<T, false, false>;
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
  const Logprobs p{a};
  switch (a.logits_dtype) {
    case YAPD_DTYPE_F32: return launch<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch<__half>(p, (cudaStream_t)stream);
    default: return launch<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
