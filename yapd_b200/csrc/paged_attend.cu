// Attention of new tokens over a paged key-value cache.
#include "serve_common.cuh"

namespace serve {
namespace {

struct Attend {
  yapd_attend_args a;
  Div page;
  int group;  // query heads per key head
};

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

// Elements from the layer's start to a token's key row of head 0, or -1.
__device__ __forceinline__ int64_t token_at(const Attend& p, int slot, int t) {
  const yapd_cache& c = p.a.cache;
  const int q = (int)div_floor(t, p.page), r = t - q * c.page_size;
  const int g = c.page_table[(int64_t)slot * c.max_pages + q];
  if (g < 0 || g >= c.pages) return -1;
  return g * c.stride_page + (int64_t)r * c.kv_heads * c.head_dim;
}

// The new tokens' rows to their pages: a warp per (request, token, head).
template <class T>
__global__ void __launch_bounds__(256) store_kernel(Attend p) {
  const yapd_cache& c = p.a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.a.B * p.a.new_tokens * c.kv_heads;
  for (int64_t w = blockIdx.x * 8ll + (threadIdx.x >> 5); w < rows; w += gridDim.x * 8ll) {
    const int h = (int)(w % c.kv_heads), i = (int)(w / c.kv_heads % p.a.new_tokens);
    const int b = (int)(w / c.kv_heads / p.a.new_tokens);
    int slot;
    const int t = slot_len(p, b, slot) - p.a.new_tokens + i;
    if (slot < 0 || t < 0) {
      if (lane == 0) set_status(c.workspace, slot < 0 ? YAPD_STATUS_BAD_SLOT : YAPD_STATUS_BAD_LENGTH);
      continue;
    }
    const int64_t at = token_at(p, slot, t);
    if (at < 0 || c.refs[at / c.stride_page] > 1) {
      if (lane == 0) set_status(c.workspace, at < 0 ? YAPD_STATUS_BAD_PAGE : YAPD_STATUS_SHARED_PAGE);
      continue;
    }
    T* key = (T*)c.kv + p.a.layer * c.stride_layer + at + h * c.head_dim;
    T* val = key + (int64_t)c.page_size * c.kv_heads * c.head_dim;
    const T* k = (const T*)p.a.k + b * p.a.k_stride_req + i * p.a.k_stride_pos + h * p.a.k_stride_head;
    const T* v = (const T*)p.a.v + b * p.a.v_stride_req + i * p.a.v_stride_pos + h * p.a.v_stride_head;
    for (int d = lane; d < c.head_dim; d += 32) {
      key[d] = k[d];
      val[d] = v[d];
    }
  }
}

// One warp per query row: lanes over the head dimension, tokens one by one
// with the running maximum and sum of a softmax.
template <class T, int D>
__global__ void __launch_bounds__(32) row_kernel(Attend p) {
  constexpr int E = D / 32;
  const yapd_cache& c = p.a.cache;
  const int lane = threadIdx.x, h = blockIdx.x % p.a.heads, i = blockIdx.x / p.a.heads, b = blockIdx.y;
  int slot;
  const int n = slot_len(p, b, slot), place = n - p.a.new_tokens + i;
  const T* q = (const T*)p.a.q + b * p.a.q_stride_req + i * p.a.q_stride_pos + h * p.a.q_stride_head;
  float qf[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = to_f32(q[lane + 32 * e]) * p.a.scale;
    o[e] = 0.0f;
  }
  float m = -INFINITY, z = 0.0f;
  const int end = p.a.causal ? min(n, place + 1) : n;
  const int64_t low = p.a.window > 0 ? place - p.a.window + 1 : 0;
  for (int t = 0; t < end; ++t) {
    if (t < low && t >= p.a.sinks) {
      t = (int)min(low, (int64_t)end) - 1;
      continue;
    }
    const int64_t at = token_at(p, slot, t);
    if (at < 0) {
      if (lane == 0) set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
      continue;
    }
    const T* key = (const T*)c.kv + p.a.layer * c.stride_layer + at + (h / p.group) * D;
    const T* val = key + (int64_t)c.page_size * c.kv_heads * D;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qf[e], to_f32(key[lane + 32 * e]), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    if (s == -INFINITY) continue;
    const float mn = fmaxf(m, s), r = expf(m - mn), e1 = expf(s - mn);
    m = mn;
    z = fmaf(z, r, e1);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], r, e1 * to_f32(val[lane + 32 * e]));
  }
  const float rz = z == 0.0f ? 0.0f : 1.0f / z;
  T* out = (T*)p.a.out + b * p.a.out_stride_req + i * p.a.out_stride_pos + h * p.a.out_stride_head;
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane + 32 * e] = from_f32<T>(o[e] * rz);
  if (p.a.lse && lane == 0)
    p.a.lse[((int64_t)b * p.a.new_tokens + i) * p.a.heads + h] = z == 0.0f ? -INFINITY : m + logf(z);
}

template <class T>
int launch(const Attend& p, cudaStream_t st) {
  const yapd_attend_args& a = p.a;
  if (a.k) {
    const int64_t rows = (int64_t)a.B * a.new_tokens * a.cache.kv_heads;
    store_kernel<T><<<(int)((rows + 7) / 8 < 2048 ? (rows + 7) / 8 : 2048), 256, 0, st>>>(p);
  }
  const dim3 grid(a.heads * a.new_tokens, a.B);
  switch (a.cache.head_dim) {
    case 32: row_kernel<T, 32><<<grid, 32, 0, st>>>(p); break;
    case 64: row_kernel<T, 64><<<grid, 32, 0, st>>>(p); break;
    case 96: row_kernel<T, 96><<<grid, 32, 0, st>>>(p); break;
    default: row_kernel<T, 128><<<grid, 32, 0, st>>>(p); break;
  }
  return launched();
}

bool rows_aligned(const void* base, int64_t r, int64_t p, int64_t h, int dtype) {
  const int64_t vec = 16 / dtype_size(dtype);
  return (uintptr_t)base % 16 == 0 && r % vec == 0 && p % vec == 0 && h % vec == 0;
}

}  // namespace

size_t attend_scratch_bytes(const yapd_cache&) { return 0; }

}  // namespace serve

using namespace serve;

extern "C" int yapd_attend(const yapd_attend_args* args, void* stream) {
  if (!args) return YAPD_ERR_NULL_POINTER;
  const yapd_attend_args& a = *args;
  const int rc = check_cache(a.cache);
  if (rc != YAPD_OK) return rc;
  if (a.B < 0 || a.B > 65535 || a.new_tokens < 1 || a.new_tokens > YAPD_MAX_NEW_TOKENS || a.heads < 1 ||
      a.heads % a.cache.kv_heads || a.heads > 1024 || (!a.slots && a.B > a.cache.slots))
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
  p.group = a.heads / a.cache.kv_heads;
  switch (dt) {
    case YAPD_DTYPE_F32: return launch<float>(p, (cudaStream_t)stream);
    case YAPD_DTYPE_F16: return launch<__half>(p, (cudaStream_t)stream);
    default: return launch<__nv_bfloat16>(p, (cudaStream_t)stream);
  }
}
