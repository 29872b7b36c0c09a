// What the serving kernels share: element types, the cache's host checks and
// its workspace, division by the page size.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "yapd_cache.h"

namespace serve {

// -------------------------------------------------------------------- types

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline int dtype_size(int dtype) { return dtype == YAPD_DTYPE_F32 ? 4 : 2; }

// ----------------------------------------------------------------- division

// t / d for 0 <= t < 2^31: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d),
// m*d exceeds 2^(31+s) by less than 2^s, so (t*m) >> (31+s) is exact.
struct Div {
  uint32_t d, m;
  int s;
};
inline Div make_div(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return Div{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ __forceinline__ uint32_t div_floor(uint32_t t, const Div& v) {
  return (uint32_t)(((uint64_t)t * v.m) >> v.s);
}

// ---------------------------------------------------------------- the cache

// Workspace: the status word, then integer scratch of the page operations,
// then the attention's.
constexpr size_t kHeaderBytes = 256;
// Attention: CTAs of one launch at most, and the floats that one of them may
// leave for others to join.
constexpr int kMaxCtas = 148 * 4;

inline size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }
// slots: per listed slot; pages: per page (see paged_pages.cu)
inline size_t pages_scratch_bytes(const yapd_cache& c) {
  return round_up(((size_t)c.slots * 8 + (size_t)c.pages * 2 + 64) * 4, 256);
}
size_t attend_scratch_bytes(const yapd_cache& c);

inline int check_cache_shape(const yapd_cache& c) {
  if (c.layers < 1 || c.pages < 1 || c.page_size < 1 || c.kv_heads < 1 || c.slots < 1 || c.max_pages < 1)
    return YAPD_ERR_BAD_SHAPE;
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 96 && c.head_dim != 128) return YAPD_ERR_BAD_SHAPE;
  if (c.kv_heads > 1024 || c.page_size > 65536) return YAPD_ERR_BAD_SHAPE;
  // the copies count the 16-byte vectors of half a page in 31 bits
  if ((int64_t)c.page_size * c.kv_heads * c.head_dim * dtype_size(c.dtype) > (int64_t)1 << 34) return YAPD_ERR_BAD_SHAPE;
  // positions, rounded up to pages and tiles, stay below 2^31
  if ((int64_t)c.max_pages * c.page_size >= ((int64_t)1 << 31) - (1 << 17)) return YAPD_ERR_BAD_SHAPE;
  if (c.dtype != YAPD_DTYPE_F32 && c.dtype != YAPD_DTYPE_BF16 && c.dtype != YAPD_DTYPE_F16)
    return YAPD_ERR_BAD_DTYPE;
  return YAPD_OK;
}

inline int check_cache(const yapd_cache& c) {
  const int rc = check_cache_shape(c);
  if (rc != YAPD_OK) return rc;
  if (!c.kv || !c.page_table || !c.kv_len || !c.refs || !c.workspace) return YAPD_ERR_NULL_POINTER;
  const int64_t block = (int64_t)2 * c.page_size * c.kv_heads * c.head_dim;
  const int64_t vec = 16 / dtype_size(c.dtype);
  if ((uintptr_t)c.kv % 16 || c.stride_layer % vec || c.stride_page % vec || (uintptr_t)c.workspace % 16)
    return YAPD_ERR_MISALIGNED;
  if ((c.pages > 1 && c.stride_page < block) || (c.layers > 1 && c.stride_layer < block)) return YAPD_ERR_BAD_SHAPE;
  if (c.workspace_bytes < yapd_cache_workspace_size(&c)) return YAPD_ERR_WORKSPACE;
  return YAPD_OK;
}

// Whether a slot's length is one that its table can hold.
__device__ __forceinline__ bool fits(const yapd_cache& c, int64_t n) {
  return n >= 0 && n <= (int64_t)c.max_pages * c.page_size;
}

__device__ __forceinline__ void set_status(void* workspace, uint32_t bits) {
  atomicOr(static_cast<uint32_t*>(workspace), bits);
}

// Ends a host entry point: a launch that failed leaves its error here.
inline int launched() { return cudaGetLastError() == cudaSuccess ? YAPD_OK : YAPD_ERR_LAUNCH; }

}  // namespace serve
