/*
 * yapd_cache.h — C ABI of the serving operators around the select step:
 *   attention of new tokens over a paged key-value cache,
 *   the management of that cache's pages,
 *   log probabilities of given tokens with entropy and alternatives.
 *
 * The conventions are those of yapd_select.h: device pointers unless stated,
 * row-major shapes, work enqueued on `stream` and never synchronised, no
 * memory allocated, a negative return value for what the host refuses (nothing
 * was launched).  Conditions that only the device can see set bits of the
 * status word at the start of the cache's workspace (yapd_read_status,
 * yapd_clear_status); no such condition reads or writes out of range.
 */
#ifndef YAPD_CACHE_H_
#define YAPD_CACHE_H_

#include "yapd_select.h"

#ifdef __cplusplus
extern "C" {
#endif

#define YAPD_CACHE_ABI_VERSION 1

/* With enum yapd_dtype: half precision, for the entry points of this header. */
#define YAPD_DTYPE_F16 2

/* Status bits of a cache's workspace. */
#define YAPD_STATUS_OUT_OF_PAGES 16u  /* a reserve was refused: the pool is full */
#define YAPD_STATUS_BAD_PAGE 32u      /* a table entry outside the pool, or none
                                         where a token should be (such a token
                                         is not seen, such a store not made) */
#define YAPD_STATUS_SHARED_PAGE 64u   /* a store into a page that other requests
                                         hold too was not made */
#define YAPD_STATUS_BAD_SLOT 128u     /* a slot out of range, listed twice, or a
                                         fork's target that is not empty */
#define YAPD_STATUS_BAD_LENGTH 256u   /* a length or a reserve of more tokens than
                                         the slot's table holds, a negative one,
                                         a truncate of more tokens than there are,
                                         a store of more than there are (those
                                         before the slot's first are not made) */

/* New tokens per request of one attention call. */
#define YAPD_MAX_NEW_TOKENS 32
/* Largest vocabulary and number of alternatives of yapd_token_logprobs. */
#define YAPD_LOGPROBS_MAX_V 1048576
#define YAPD_LOGPROBS_MAX_TOP 32

/*
 * yapd_cache — a pool of pages and the requests' tables into it.
 *
 * kv is (layers, pages) blocks of (2, page_size, kv_heads, head_dim): keys,
 * then values, the page layout of the reference's FlashInfer engine
 * (chatterbox_flash/engines/flashinfer.py:110-115).  A block is contiguous;
 * stride_layer and stride_page (elements, multiples of 16 bytes) place the
 * blocks, so a pool may be layer-major or page-major.  The keys of a page are at
 * most 2^34 bytes.  Token t of slot s is token t % page_size of page page_table[s][t / page_size]; a table entry of
 * -1 is no page (a request that was trimmed has them in its middle).
 * A slot with a length that is negative or more than its table holds is read
 * as an empty one and left as it is (YAPD_STATUS_BAD_LENGTH), but for a truncate
 * with tokens < 0, which empties it.
 * refs[p] is the number of table entries that hold page p; 0: free.  There is
 * no list of free pages: the lowest-numbered free page is always the next one
 * given out, so that a sequence of calls always gives the same tables.
 */
typedef struct yapd_cache {
  int32_t layers, pages, page_size, kv_heads, head_dim;
  int32_t dtype;                /* enum yapd_dtype or YAPD_DTYPE_F16 */
  int32_t slots, max_pages;
  void* kv;                     /* 16-byte aligned */
  int64_t stride_layer, stride_page;
  int32_t* page_table;          /* (slots, max_pages), contiguous */
  int64_t* kv_len;              /* (slots,) tokens of each slot */
  int32_t* refs;                /* (pages,) */
  void* workspace;              /* zero-filled before its first use; its calls
                                   are ordered on one stream, each one's
                                   launches together: one thread at a time */
  size_t workspace_bytes;
} yapd_cache;

/* Workspace bytes a cache needs (its pointers are not looked at); 0 for a
 * cache that the calls would refuse. */
size_t yapd_cache_workspace_size(const yapd_cache* cache);

/*
 * yapd_attend_args — attention of each request's last `new_tokens` tokens.
 *
 * Request b is slot slots[b] (b where slots is NULL); its new tokens are the
 * last new_tokens of the slot's kv_len tokens (reserve them first).  Query i
 * stands at position p = kv_len - new_tokens + i and sees token j when
 *   j < kv_len, and with causal j <= p,
 *   and with window > 0: j > p - window or j < sinks.
 * Query head h reads key head h / (heads / kv_heads).
 *   out = sum_j softmax_j(scale q.k_j) v_j,  lse = ln sum_j exp(scale q.k_j);
 * a query that sees nothing gets out = 0 and lse = -inf, and so does one whose
 * every score is -inf.  Products and sums are in 32 bits.
 *
 * k and v, where given, are the new tokens' rows: the call stores them in the
 * request's pages and attends over them (of the requests that name the same slot
 * only the first one's are stored: YAPD_STATUS_BAD_SLOT).  Rows are q + b*q_stride_req +
 * i*q_stride_pos + h*q_stride_head (elements; likewise k, v, out), head_dim
 * contiguous elements, 16-byte aligned.  The types are the cache's.
 */
typedef struct yapd_attend_args {
  yapd_cache cache;
  int32_t layer, B, new_tokens, heads;
  const int32_t* slots;         /* (B,) or NULL */
  const void* q;
  int64_t q_stride_req, q_stride_pos, q_stride_head;
  const void* k;                /* both or neither */
  int64_t k_stride_req, k_stride_pos, k_stride_head;
  const void* v;
  int64_t v_stride_req, v_stride_pos, v_stride_head;
  void* out;
  int64_t out_stride_req, out_stride_pos, out_stride_head;
  float* lse;                   /* (B, new_tokens, heads) contiguous, or NULL */
  float scale;
  int32_t causal;
  int64_t window, sinks;        /* window <= 0: no window */
  int64_t wait_limit_ns;        /* as in yapd_select_args; a request whose keys
                                   did not arrive has no or NaN outputs, and
                                   YAPD_STATUS_WAIT_TIMEOUT is set */
} yapd_attend_args;

int yapd_attend(const yapd_attend_args* args, void* stream);

/*
 * yapd_pages_args — one change of the pool's bookkeeping.  `n` slots are
 * listed in `slots` (NULL: slots 0 .. n-1); a slot out of range or listed a
 * second time is left alone (YAPD_STATUS_BAD_SLOT).
 */
typedef struct yapd_pages_args {
  yapd_cache cache;
  int32_t n;
  const int32_t* slots;         /* (n,) */
  const int32_t* src;           /* fork: (n,) slots forked; copy: (n,) pages read */
  const int32_t* dst;           /* copy: (n,) pages written */
  int64_t tokens;               /* reserve, truncate: tokens of every slot ... */
  const int64_t* tokens_each;   /* ... or of each, (n,) */
  int64_t window, sinks;        /* trim */
  uint8_t* granted;             /* reserve: (n,) bool, or NULL */
  int32_t* live;                /* compact: (1,), or NULL */
} yapd_pages_args;

/* Adds tokens to each listed slot, in the order of the list.  New pages are
 * the lowest free ones.  A partly filled last page that other slots hold too
 * is replaced by a copy of its tokens in all layers, so that what is stored
 * next touches no other request.  The first slot that the pool has no room
 * for, and all that follow it, are refused unchanged; so is one whose table
 * is too short. */
int yapd_pages_reserve(const yapd_pages_args* args, void* stream);

/* Makes the empty slot slots[i] a copy of slot src[i]: the pages are shared. */
int yapd_pages_fork(const yapd_pages_args* args, void* stream);

/* Takes the last tokens from each listed slot (all that it has where it has
 * fewer, or where tokens < 0) and gives up the pages that no longer hold any. */
int yapd_pages_truncate(const yapd_pages_args* args, void* stream);

/* Gives up each listed slot's pages that the token after its last no longer
 * sees through a window of `window` tokens with the first `sinks` visible. */
int yapd_pages_trim(const yapd_pages_args* args, void* stream);

/* Packs the pool: with m live pages, those numbered m or more move, in their
 * order, to the free numbers below m, in all layers, and every table follows.
 * live receives m. */
int yapd_pages_compact(const yapd_pages_args* args, void* stream);

/* Copies pages src[i] to dst[i] in all layers.  No page may be both read and
 * written, nor written twice. */
int yapd_pages_copy(const yapd_pages_args* args, void* stream);

/*
 * yapd_logprobs_args — how likely given tokens were.
 *
 * For each row x of logits (R, V): log softmax at targets[r] (NaN where the
 * target is outside [0, V)), the entropy in nats, and the top_n most likely
 * tokens, most likely first, equal ones in ascending id.  Masked tokens
 * (-inf) have probability 0 and are no alternatives: the places of
 * alternatives that a row does not have hold id -1 and -inf.  A row with NaN
 * or +inf, or with nothing but -inf, has no distribution: its values are NaN
 * and its ids -1.
 */
typedef struct yapd_logprobs_args {
  int32_t R, V, top_n;
  int32_t logits_dtype;         /* enum yapd_dtype or YAPD_DTYPE_F16 */
  const void* logits;           /* element-aligned */
  int64_t stride_row;
  const int64_t* targets;       /* (R,) or NULL */
  float* logprob;               /* (R,); with targets */
  float* entropy;               /* (R,) or NULL */
  float* top_logprobs;          /* (R, top_n) */
  int32_t* top_ids;             /* (R, top_n) */
} yapd_logprobs_args;

int yapd_token_logprobs(const yapd_logprobs_args* args, void* stream);

/* YAPD_CACHE_ABI_VERSION of the loaded library. */
int yapd_cache_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* YAPD_CACHE_H_ */
