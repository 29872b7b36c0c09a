// The pages of a key-value cache: reserve, fork, truncate, trim, compact, copy.
//
// The bookkeeping is three arrays (tables, lengths, reference counts) and no
// list: a page is free when its count is 0, and the lowest-numbered free page
// is the next one given out.  Every operation is a function of the arrays and
// its arguments alone, whatever order its threads run in.
#include "serve_common.cuh"

namespace serve {
namespace {

constexpr int kMetaThreads = 1024;

struct Pages {
  yapd_cache c;
  Div page;
  int32_t n;
  const int32_t* slots;
  const int32_t* src;
  const int32_t* dst;
  int64_t tokens;
  const int64_t* tokens_each;
  int64_t window, sinks;
  uint8_t* granted;
  int32_t* live;
  // scratch in the workspace
  int32_t* owner;     // (slots) first list index that names a slot
  int32_t* upto;      // (slots) pages taken by the list up to and including i
  int32_t* tail;      // (slots) page to be copied, or -1
  int32_t* count;     // (slots) pages that i takes; -1: refused
  int32_t* first;     // (slots) first table column that i fills
  int32_t* len;       // (slots) tokens before the call
  int32_t* copy_src;  // pages to copy ...
  int32_t* copy_dst;  // ... to where
  int32_t* copy_tok;  // (slots) tokens of each, or NULL: whole pages
  int32_t* copies;    // how many, or NULL: n
  int32_t* list;      // (pages) free pages / new numbers
};

// Inclusive sum over the block; `total` is its last value.  `sh` has 33 ints.
__device__ int block_scan(int x, int* sh, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < warps ? sh[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(~0u, w, d);
      if (lane >= d) w += y;
    }
    sh[lane] = w;
  }
  __syncthreads();
  total = sh[warps - 1];
  if (warp) x += sh[warp - 1];
  __syncthreads();
  return x;
}

// The slot that list index i names, or -1.
__device__ __forceinline__ int slot_of(const Pages& p, int i) {
  const int s = p.slots ? p.slots[i] : i;
  return s >= 0 && s < p.c.slots ? s : -1;
}

// Tokens of a slot, or -1 where that does not fit its table.
__device__ __forceinline__ int len_of(const Pages& p, int slot) {
  const int64_t n = p.c.kv_len[slot];
  return fits(p.c, n) ? (int)n : -1;
}

__device__ __forceinline__ int64_t tokens_of(const Pages& p, int i) {
  return p.tokens_each ? p.tokens_each[i] : p.tokens;
}

// One block decides the whole list: what each slot needs, who copies a shared
// tail page, which free pages go where.  A few dependent reads of L2 each, so
// latency is all of its time: 6 us with 256 slots of 10000 pages.
__global__ void __launch_bounds__(kMetaThreads) reserve_kernel(Pages p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int sh[33];
  __shared__ int any_shared;
  const yapd_cache& c = p.c;
  const int tid = threadIdx.x;
  if (tid == 0) {
    *p.copies = 0;
    any_shared = 0;
  }
  // the first index that names a slot owns it
  for (int i = tid; i < p.n; i += kMetaThreads) {
    const int s = slot_of(p, i);
    if (s >= 0) p.owner[s] = INT32_MAX;
  }
  __syncthreads();
  for (int i = tid; i < p.n; i += kMetaThreads) {
    const int s = slot_of(p, i);
    if (s >= 0) atomicMin(&p.owner[s], i);
  }
  __syncthreads();
  for (int i = tid; i < p.n; i += kMetaThreads) {
    const int s = slot_of(p, i);
    int need = -1, tail = -1, first = 0, len = 0;
    if (s < 0 || *(volatile int32_t*)&p.owner[s] != i) {
      set_status(c.workspace, YAPD_STATUS_BAD_SLOT);
    } else {
      const int64_t add = tokens_of(p, i);
      len = len_of(p, s);
      if (len < 0 || add < 0 || add > (int64_t)c.max_pages * p.page.d - len) {
        set_status(c.workspace, YAPD_STATUS_BAD_LENGTH);
      } else {
        first = (int)div_floor(len + p.page.d - 1, p.page);
        need = (int)div_floor((uint32_t)(len + add) + p.page.d - 1, p.page) - first;
        if (add > 0 && len % p.page.d) {
          const int t = c.page_table[(int64_t)s * c.max_pages + first - 1];
          if (t < 0 || t >= c.pages) {
            set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
            need = -1;
          } else if (c.refs[t] > 1) {
            tail = t;
            any_shared = 1;
          }
        }
      }
    }
    p.count[i] = need;
    p.tail[i] = tail;
    p.first[i] = first;
    p.len[i] = len;
  }
  __syncthreads();
  // of the h holders of a shared tail page, each listed one copies it until
  // one holder is left: index i does if h less the listed ones before it is > 1
  if (any_shared) {
    for (int i = tid; i < p.n; i += kMetaThreads) {
      const int t = p.tail[i];
      if (t < 0) continue;
      int before = 0;
      for (int j = 0; j < i; ++j) before += p.tail[j] == t;
      const bool copies = c.refs[t] - before > 1;
      p.upto[i] = copies;  // p.tail stays whole until every thread has counted
    }
    __syncthreads();
    for (int i = tid; i < p.n; i += kMetaThreads) {
      if (p.tail[i] < 0) continue;
      if (p.upto[i]) {
        p.count[i] += 1;
        p.first[i] -= 1;
      } else {
        p.tail[i] = -1;
      }
    }
    __syncthreads();
  }
  int wanted = 0;
  for (int base = 0; base < p.n; base += kMetaThreads) {
    const int i = base + tid;
    int total;
    const int x = block_scan(i < p.n ? max(p.count[i], 0) : 0, sh, total);
    if (i < p.n) p.upto[i] = wanted + x;
    wanted += total;
  }
  // the lowest free pages, as many as are wanted
  int found = 0;
  for (int base = 0; base < c.pages && found < wanted; base += kMetaThreads) {
    const int g = base + tid;
    const bool is_free = g < c.pages && c.refs[g] == 0;
    int total;
    const int x = block_scan(is_free, sh, total);
    if (is_free) p.list[found + x - 1] = g;
    found += total;
  }
  __syncthreads();
  for (int i = tid; i < p.n; i += kMetaThreads) {
    const int need = p.count[i];
    const bool ok = need >= 0 && p.upto[i] <= found;
    if (p.granted) p.granted[i] = ok;
    if (need >= 0 && !ok) set_status(c.workspace, YAPD_STATUS_OUT_OF_PAGES);
    if (!ok) continue;
    const int s = slot_of(p, i);
    c.kv_len[s] = p.len[i] + tokens_of(p, i);
    if (p.tail[i] >= 0) {
      const int k = atomicAdd(p.copies, 1);  // any order: the copies are disjoint
      p.copy_src[k] = p.tail[i];
      p.copy_dst[k] = p.list[p.upto[i] - need];
      p.copy_tok[k] = p.len[i] % p.page.d;
      atomicSub(&c.refs[p.tail[i]], 1);
    }
  }
  // page k of those given goes to the first index whose `upto` exceeds k
  const int given = min(found, wanted);
  for (int k = tid; k < given; k += kMetaThreads) {
    int lo = 0, hi = p.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.upto[mid] > k) hi = mid; else lo = mid + 1;
    }
    if (p.upto[lo] > found) continue;  // refused: its pages stay free
    const int g = p.list[k];
    const int column = p.first[lo] + k - (p.upto[lo] - p.count[lo]);
    c.page_table[(int64_t)slot_of(p, lo) * c.max_pages + column] = g;
    c.refs[g] = 1;
  }
}

// Whether an earlier index of the list names `slot` too.
__device__ bool named_before(const Pages& p, int i, int slot) {
  bool dup = false;
  if (p.slots)
    for (int j = threadIdx.x; j < i; j += blockDim.x) dup |= p.slots[j] == slot;
  return __syncthreads_or(dup);
}

__global__ void __launch_bounds__(128) fork_kernel(Pages p) {
  const yapd_cache& c = p.c;
  const int i = blockIdx.x, s = slot_of(p, i), from = p.src[i];
  const bool dup = s < 0 || named_before(p, i, s);
  bool target = from < 0 || from >= c.slots;  // a slot forked is no target of the same call
  for (int j = threadIdx.x; j < p.n; j += blockDim.x) target |= slot_of(p, j) == from;
  target = __syncthreads_or(target);
  if (dup || target || c.kv_len[s] != 0) {
    if (threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_SLOT);
    return;
  }
  __syncthreads();
  const int len = len_of(p, from);
  if (len < 0) {
    if (threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_LENGTH);
    return;
  }
  const int held = (int)div_floor(len + p.page.d - 1, p.page);
  const int32_t* in = c.page_table + (int64_t)from * c.max_pages;
  int32_t* out = c.page_table + (int64_t)s * c.max_pages;
  for (int j = threadIdx.x; j < held; j += blockDim.x) {
    const int g = in[j];
    out[j] = g;
    if (g >= 0 && g < c.pages) atomicAdd(&c.refs[g], 1);
  }
  if (threadIdx.x == 0) c.kv_len[s] = len;
}

__device__ __forceinline__ void give_up(const yapd_cache& c, int32_t* entry) {
  const int g = *entry;
  if (g < 0) return;
  *entry = -1;
  if (g >= c.pages || atomicSub(&c.refs[g], 1) <= 0) set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
}

// Truncate, and trim where `trim`: the pages that no longer hold a token that
// will be seen are given up.
__global__ void __launch_bounds__(128) release_kernel(Pages p, bool trim) {
  const yapd_cache& c = p.c;
  const int i = blockIdx.x, s = slot_of(p, i);
  if (s < 0 || named_before(p, i, s)) {
    if (threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_SLOT);
    return;
  }
  const int64_t take = trim ? 0 : tokens_of(p, i);
  int len = len_of(p, s);
  if (len < 0) {
    if (threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_LENGTH);
    if (take >= 0) return;
    len = c.max_pages * p.page.d;  // freed: whatever the table holds goes
  }
  const int held = (int)div_floor(len + p.page.d - 1, p.page);
  int32_t* row = c.page_table + (int64_t)s * c.max_pages;
  if (trim) {
    // the next token stands at `len` and sees j > len - window, or j < sinks
    const int64_t reach = len + 1 - p.window;
    for (int j = threadIdx.x; j < held; j += blockDim.x)
      if ((int64_t)j * p.page.d >= p.sinks && (int64_t)(j + 1) * p.page.d <= reach) give_up(c, row + j);
    return;
  }
  if (take > len && threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_LENGTH);
  const int keep = take < 0 || take > len ? 0 : len - (int)take;
  __syncthreads();  // every thread has read the length
  for (int j = (int)div_floor(keep + p.page.d - 1, p.page) + threadIdx.x; j < held; j += blockDim.x)
    give_up(c, row + j);
  if (threadIdx.x == 0) c.kv_len[s] = keep;
}

// Pairs the i-th live page numbered `live` or more with the i-th free number
// below it; list[] receives each moved page's new number (-1: not live).
__global__ void __launch_bounds__(kMetaThreads) compact_kernel(Pages p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int sh[33];
  const yapd_cache& c = p.c;
  const int tid = threadIdx.x;
  int live = 0;
  for (int base = 0; base < c.pages; base += kMetaThreads) {
    const int g = base + tid;
    int total;
    block_scan(g < c.pages && c.refs[g] > 0, sh, total);
    live += total;
  }
  int holes = 0, moved = 0;
  for (int base = 0; base < c.pages; base += kMetaThreads) {
    const int g = base + tid;
    const bool used = g < c.pages && c.refs[g] > 0;
    const bool hole = g < live && !used, mover = g >= live && used;
    int total;
    const int h = block_scan(hole, sh, total);
    if (hole) p.copy_dst[holes + h - 1] = g;
    holes += total;
    const int m = block_scan(mover, sh, total);
    if (mover) p.copy_src[moved + m - 1] = g;
    moved += total;
    if (g < c.pages) p.list[g] = used ? g : -1;
  }
  __syncthreads();
  for (int k = tid; k < moved; k += kMetaThreads) {
    const int a = p.copy_src[k], b = p.copy_dst[k];
    p.list[a] = b;
    c.refs[b] = c.refs[a];
    c.refs[a] = 0;
  }
  if (tid == 0) {
    *p.copies = moved;
    if (p.live) *p.live = live;
  }
}

__global__ void __launch_bounds__(256) renumber_kernel(Pages p) {
  const int64_t all = (int64_t)p.c.slots * p.c.max_pages;
  for (int64_t k = blockIdx.x * 256ll + threadIdx.x; k < all; k += gridDim.x * 256ll) {
    const int g = p.c.page_table[k];
    if (g >= 0 && g < p.c.pages) p.c.page_table[k] = p.list[g];
  }
}

// Copies page (or token) ranges in all layers: work item = (pair, layer, half
// of the block), 16 bytes a thread, four at a time. It starts beside the kernel
// that lists the copies and waits for it on the device. Bound by memory: 302 us
// for 1.65 GB read and written, 84 % of the copy rate.
__global__ void __launch_bounds__(256) copy_kernel(Pages p, int esize, bool check) {
  const yapd_cache& c = p.c;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int copies = p.copies ? *p.copies : p.n;
  const int64_t row = (int64_t)c.kv_heads * c.head_dim * esize;  // bytes of a token in one half
  const int64_t items = (int64_t)copies * c.layers * 2;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int half = (int)(it & 1), layer = (int)((it >> 1) % c.layers), k = (int)((it >> 1) / c.layers);
    const int a = p.copy_src[k], b = p.copy_dst[k];
    if (check && (a < 0 || a >= c.pages || b < 0 || b >= c.pages)) {
      if (threadIdx.x == 0) set_status(c.workspace, YAPD_STATUS_BAD_PAGE);
      continue;
    }
    const int64_t bytes = (p.copy_tok ? p.copy_tok[k] : c.page_size) * row;
    const int64_t at = (layer * c.stride_layer) * esize + half * c.page_size * row;
    const uint4* in = (const uint4*)((const char*)c.kv + at + a * c.stride_page * esize);
    uint4* out = (uint4*)((char*)c.kv + at + b * c.stride_page * esize);
#pragma unroll 4
    for (int x = threadIdx.x; x < (int)(bytes / 16); x += 256) out[x] = in[x];
  }
}

constexpr int kCopyCtas = 148 * 8;

// A kernel that may start while the one before it in the stream ends.
template <class... Args>
int launch_early(void (*kernel)(Args...), int ctas, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? YAPD_OK : YAPD_ERR_LAUNCH;
}

enum class Need { kSlots, kSrc, kPages };

int set_up(const yapd_pages_args* a, Need need, Pages& p) {
  if (!a) return YAPD_ERR_NULL_POINTER;
  const int rc = check_cache(a->cache);
  if (rc != YAPD_OK) return rc;
  if (a->n < 0 || a->n > (need == Need::kPages ? a->cache.pages : a->cache.slots)) return YAPD_ERR_BAD_SHAPE;
  if (need == Need::kSrc && a->n && (!a->src || !a->slots)) return YAPD_ERR_NULL_POINTER;
  if (need == Need::kPages && a->n && (!a->src || !a->dst)) return YAPD_ERR_NULL_POINTER;
  const yapd_cache& c = a->cache;
  p = Pages{};
  p.c = c;
  p.page = make_div((uint32_t)c.page_size);
  p.n = a->n;
  p.slots = a->slots;
  p.src = a->src;
  p.dst = a->dst;
  p.tokens = a->tokens;
  p.tokens_each = a->tokens_each;
  p.window = a->window;
  p.sinks = a->sinks;
  p.granted = a->granted;
  p.live = a->live;
  int32_t* w = (int32_t*)((char*)c.workspace + kHeaderBytes);
  p.copies = w;
  w += 64;
  int32_t** per_slot[] = {&p.owner, &p.upto, &p.tail, &p.count, &p.first, &p.len, &p.copy_tok, &p.copy_src};
  for (int32_t** q : per_slot) {
    *q = w;
    w += c.slots;
  }
  p.list = w;
  p.copy_dst = w + c.pages;  // a reserve copies at most min(slots, pages) pages
  return YAPD_OK;
}

}  // namespace
}  // namespace serve

using namespace serve;

extern "C" {

size_t yapd_cache_workspace_size(const yapd_cache* cache) {
  if (!cache || check_cache_shape(*cache) != YAPD_OK) return 0;
  return kHeaderBytes + pages_scratch_bytes(*cache) + attend_scratch_bytes(*cache);
}

int yapd_cache_abi_version(void) { return YAPD_CACHE_ABI_VERSION; }

int yapd_pages_reserve(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kSlots, p);
  if (rc != YAPD_OK || args->n == 0) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  reserve_kernel<<<1, kMetaThreads, 0, st>>>(p);
  if (launch_early(copy_kernel, kCopyCtas, st, p, dtype_size(p.c.dtype), false) != YAPD_OK) return YAPD_ERR_LAUNCH;
  return launched();
}

int yapd_pages_fork(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kSrc, p);
  if (rc != YAPD_OK || args->n == 0) return rc;
  fork_kernel<<<args->n, 128, 0, (cudaStream_t)stream>>>(p);
  return launched();
}

int yapd_pages_truncate(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kSlots, p);
  if (rc != YAPD_OK || args->n == 0) return rc;
  release_kernel<<<args->n, 128, 0, (cudaStream_t)stream>>>(p, false);
  return launched();
}

int yapd_pages_trim(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kSlots, p);
  if (rc != YAPD_OK) return rc;
  if (args->window < 1 || args->sinks < 0) return YAPD_ERR_BAD_ARG;
  if (args->n == 0) return rc;
  release_kernel<<<args->n, 128, 0, (cudaStream_t)stream>>>(p, true);
  return launched();
}

int yapd_pages_compact(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kSlots, p);
  if (rc != YAPD_OK) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  p.copy_src = p.copy_dst + (p.c.pages + 1) / 2;  // as many pages move as there are holes: half at most
  p.copy_tok = nullptr;
  compact_kernel<<<1, kMetaThreads, 0, st>>>(p);
  if (launch_early(copy_kernel, kCopyCtas, st, p, dtype_size(p.c.dtype), false) != YAPD_OK) return YAPD_ERR_LAUNCH;
  renumber_kernel<<<148, 256, 0, st>>>(p);
  return launched();
}

int yapd_pages_copy(const yapd_pages_args* args, void* stream) {
  Pages p;
  const int rc = set_up(args, Need::kPages, p);
  if (rc != YAPD_OK || args->n == 0) return rc;
  p.copy_src = const_cast<int32_t*>(args->src);
  p.copy_dst = const_cast<int32_t*>(args->dst);
  p.copy_tok = nullptr;
  p.copies = nullptr;
  copy_kernel<<<kCopyCtas, 256, 0, (cudaStream_t)stream>>>(p, dtype_size(p.c.dtype), true);
  return launched();
}

}  // extern "C"
