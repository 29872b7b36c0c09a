// Log probabilities of given tokens, the entropy and the most likely tokens.
#include "serve_common.cuh"

namespace serve {
namespace {

constexpr int kThreads = 256;

struct Logprobs {
  yapd_logprobs_args a;
};

__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <class V, class F>
__device__ V block_reduce(V x, F f, V* sh) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x = f(x, __shfl_xor_sync(~0u, x, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
  __syncthreads();
  x = sh[0];
  for (int w = 1; w < kThreads / 32; ++w) x = f(x, sh[w]);
  return x;
}

// One block per row: the maximum, the sums, then the alternatives one by one.
template <class T>
__global__ void __launch_bounds__(kThreads) row_kernel(Logprobs p) {
  __shared__ unsigned long long sh[kThreads / 32];
  const yapd_logprobs_args& a = p.a;
  const int r = blockIdx.x, tid = threadIdx.x;
  const T* x = (const T*)a.logits + r * a.stride_row;
  float m = -INFINITY;
  bool bad = false;
  for (int v = tid; v < a.V; v += kThreads) {
    const float f = to_f32(x[v]);
    bad |= f != f;
    m = fmaxf(m, f);
  }
  m = block_reduce(m, [](float u, float w) { return fmaxf(u, w); }, (float*)sh);
  bad = __syncthreads_or(bad) || !(fabsf(m) < INFINITY);
  float z = 0.0f, w = 0.0f;
  for (int v = tid; v < a.V; v += kThreads) {
    const float d = to_f32(x[v]) - m, e = expf(d);
    z += e;
    if (e > 0.0f) w = fmaf(e, d, w);
  }
  auto add = [](float u, float y) { return u + y; };
  z = block_reduce(z, add, (float*)sh);
  w = block_reduce(w, add, (float*)sh);
  const float lz = logf(z);
  if (tid == 0) {
    if (a.targets) {
      const int64_t t = a.targets[r];
      a.logprob[r] = bad || t < 0 || t >= a.V ? NAN : to_f32(x[t]) - m - lz;
    }
    if (a.entropy) a.entropy[r] = bad ? NAN : lz - w / z;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top_n; ++k) {
    unsigned long long best = 0;
    for (int v = tid; v < a.V && !bad; v += kThreads) {
      const float f = to_f32(x[v]);
      const unsigned long long key = (unsigned long long)order_of(f == 0.0f ? 0.0f : f) << 32 | (uint32_t)~v;
      if (f > -INFINITY && key < last && key > best) best = key;
    }
    best = block_reduce(best, [](unsigned long long u, unsigned long long y) { return u > y ? u : y; }, sh);
    last = best;
    if (tid == 0) {
      const int id = best ? (int)~(uint32_t)best : -1;
      a.top_ids[(int64_t)r * a.top_n + k] = id;
      a.top_logprobs[(int64_t)r * a.top_n + k] = bad ? NAN : id < 0 ? -INFINITY : to_f32(x[id]) - m - lz;
    }
  }
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
  Logprobs p{a};
  cudaStream_t st = (cudaStream_t)stream;
  switch (a.logits_dtype) {
    case YAPD_DTYPE_F32: row_kernel<float><<<a.R, kThreads, 0, st>>>(p); break;
    case YAPD_DTYPE_F16: row_kernel<__half><<<a.R, kThreads, 0, st>>>(p); break;
    default: row_kernel<__nv_bfloat16><<<a.R, kThreads, 0, st>>>(p); break;
  }
  return launched();
}
