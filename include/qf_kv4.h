/*
 * qf_kv4.h — C ABI of the MI355X (gfx950) operators of a served attention layer over a paged cache held in 4 bits.
 *
 *   qf_step_tables      a step's tables from request lengths: slots, positions, newly taken pages
 *   qf_qk_norm_rope     norms of the query and key heads, the position rotation and the write into the cache
 *   qf_kv4_load         the cache's values at given slots
 *   qf_kv4_attention    attention over the cache: decode, verification and prompt chunks
 *
 * Pointers are device pointers, strides are in elements, the last dimension is contiguous, calls run on `stream` (a
 * hipStream_t, NULL = the null stream) without host synchronisation and may be captured in a HIP graph.  Every entry
 * point checks its arguments before any HIP call and returns a qf_status.  Results do not depend on timing: sums run in
 * a fixed order.  What stands in device memory and cannot be checked by the host (slots, positions, block ids, lengths) is
 * kept inside its tensor by the kernels, as each entry point says.
 *
 * The 4-bit form of a head of D values: blocks of 32 neighbouring values share a power of two 2^e, each value is one of
 * +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} * 2^e (e2m1, nearest, the even code of two, 6 for what is above).  e is the smallest from
 * -125 to 125 with the block's largest magnitude below 7 * 2^e; a block that holds an infinity or NaN is NaN as a whole.  The
 * scale's byte is e + 127 (255: NaN).
 *
 * The cache is bytes [num_blocks, H_kv, page_size / 16, 17 D] (block stride in bytes, a multiple of 16; the rest
 * contiguous; 16-byte aligned; page_size a multiple of 16; D = 64, 128 or 256).  A record of 16 positions holds
 *   [0, 8 D)         the keys' codes [position][D / 2], the even value in the low half of a byte
 *   [8 D, 16 D)      the values' codes [D / (16 w)][position / 4][16][position % 4][w / 2], w = min(D, 128) / 16
 *   [16 D, 16.5 D)   the keys' scales [D / 32][position]
 *   [16.5 D, 17 D)   the values' scales likewise
 * so that a lane of a matrix instruction finds its operand's bytes together.  Slot s is position s % page_size of block
 * s / page_size.
 */
#ifndef QF_KV4_H
#define QF_KV4_H

#include <stddef.h>
#include <stdint.h>

#include "qf_w8a16.h" /* qf_status */

#ifdef __cplusplus
extern "C" {
#endif

#define QF_KV4_ABI_VERSION 1
/* Positions of a cache record; pages are whole multiples of it. */
#define QF_KV4_TILE 16
/* Most requests of qf_step_tables. */
#define QF_STEP_MAX_REQS 4096
/* Most tokens and pages of qf_step_tables. */
#define QF_STEP_MAX_TOKENS (1 << 29)
/* Most requests, and most kv heads, of qf_kv4_attention. */
#define QF_KV4_MAX_REQS 65535
/* Longest packed row tile of the split attention: query tokens of a request * (H / H_kv). */
#define QF_KV4_MAX_ROWS 64

typedef enum qf_cache { QF_CACHE_NONE = 0, QF_CACHE_PAGES = 1, QF_CACHE_KV4 = 2 } qf_cache;

/* ABI version of the loaded library (QF_KV4_ABI_VERSION). */
int qf_kv4_abi_version(void);

/* A step's tables.  Request b has context[b] cached positions, q_lens[b] new tokens and holds held[b] pages, the first
 * entries of its row of block_table int32 [num_reqs, max_blocks] (row stride bt_stride).  It needs
 * ceil((context + q) / page_size) pages; those it lacks are taken from the top of the stack free_blocks[0 .. free_count):
 * in order of requests and pages, the j-th is free_blocks[free_count - 1 - j].  Written:
 *   cu_q [num_reqs + 1]   the first token of each request, then their number
 *   seq_lens [num_reqs]   context + q
 *   positions, slots      int64 [num_tokens]: of each token, request after request; 0 and -1 behind the last one
 *   held_out [num_reqs], free_count_out [1]   what the next step starts from
 *   block_table           the new entries, in place; nothing else of it is touched
 *   fits [1]              1
 * A step that does not fit (more tokens than num_tokens, more pages than the stack or a row of the table holds, a negative
 * length, a sum past 2^31 - 1) takes nothing: cu_q is 0, seq_lens the contexts, slots -1, held and the count as before,
 * fits 0.  The int32 outputs must not overlap the inputs.  num_reqs <= QF_STEP_MAX_REQS; num_tokens, num_free and max_blocks
 * at most QF_STEP_MAX_TOKENS.  An id of the stack is taken as it is. */
int qf_step_tables(const int32_t* context, const int32_t* q_lens, const int32_t* held, int32_t* block_table,
                   int64_t bt_stride, int max_blocks, const int32_t* free_blocks, const int32_t* free_count, int num_free,
                   int num_reqs, int page_size, int num_tokens, int32_t* cu_q, int32_t* seq_lens, int64_t* positions,
                   int64_t* slots, int32_t* held_out, int32_t* free_count_out, int32_t* fits, void* stream);

/* Heads of tokens: [num_tokens, heads, D] bf16, strides in elements (multiples of 8), 16-byte aligned. */
typedef struct qf_heads {
  uint16_t* data;
  int64_t stride_tok, stride_head;
} qf_heads;

/* One of the bf16 pages' tensors: [num_blocks, page_size, H_kv, D], strides in elements (multiples of 8), 16-byte aligned. */
typedef struct qf_pages {
  uint16_t* data;
  int64_t stride_block, stride_tok, stride_head;
} qf_pages;

typedef struct qf_qk_norm_rope_args {
  qf_heads query, key, value;   /* inputs; data NULL: absent (value only together with a cache) */
  qf_heads query_out, key_out;  /* may be the inputs themselves; key_out.data NULL: the cache alone takes the keys */
  const uint16_t *q_weight, *k_weight; /* bf16 [D], 16-byte aligned; NULL: that head is not normalised */
  const int64_t* positions;     /* [num_tokens] */
  const void* cos_sin;          /* [num_positions, rot]: cosines, then sines; contiguous, 16-byte aligned */
  const int64_t* slots;         /* [num_tokens], with a cache */
  void* cache;                  /* QF_CACHE_KV4: the bytes */
  int64_t cache_stride;         /* bytes from block to block */
  qf_pages key_pages, value_pages; /* QF_CACHE_PAGES */
  int64_t num_positions, num_blocks;
  double eps, weight_offset;
  int cos_sin_f32;              /* fp32, else bf16 */
  int rot, interleaved, cache_kind, page_size;
  int num_tokens, num_heads, num_kv_heads, head_size;
} qf_qk_norm_rope_args;

/* n = x * rsqrt(mean(x^2) + eps) * (weight_offset + weight) over each head (x itself where the weight is NULL), then the
 * first `rot` values of a head are turned by the angles of the token's row of cos_sin: pairs (i, i + rot / 2), or (2 i, 2 i
 * + 1) with interleaved, (a, b) -> (a c - b s, b c + a s).  Rounded once to bf16.  With a cache, the rounded key and the
 * value go to the token's slot: as they are (pages), or in the 4-bit form of the bf16 values.  A slot outside
 * [0, num_blocks * page_size) is not written.  Two tokens must not have one slot: of what it then holds some bytes may be the
 * one's and some the other's.  A position is kept inside [0, num_positions).
 * All arithmetic is fp32; that of keys for the 4-bit cache is fp64, so that no code depends on the order of a sum.
 * D = 64, 128 or 256; rot a multiple of 16 up to D, or 0 (no rotation: positions and cos_sin are not read). */
int qf_qk_norm_rope(const qf_qk_norm_rope_args* args, void* stream);

/* key, value bf16 [num_tokens, H_kv, D] (contiguous, 16-byte aligned): what the cache holds at each slot, exactly; zeros for
 * a slot outside the cache. */
int qf_kv4_load(const void* cache, int64_t cache_stride, int64_t num_blocks, int page_size, int num_kv_heads, int head_size,
                const int64_t* slots, int num_tokens, uint16_t* key, uint16_t* value, void* stream);

typedef struct qf_kv4_attention_args {
  qf_heads query, out;          /* [num_tokens, H, D] */
  const void* cache;
  int64_t cache_stride;         /* bytes from block to block */
  int64_t num_blocks;
  const int32_t* block_table;   /* [num_reqs, max_blocks], row stride bt_stride */
  int64_t bt_stride;
  const int32_t* seq_lens;      /* [num_reqs]: cached positions, this step's tokens included */
  const int32_t* cu_q;          /* [num_reqs + 1]: first token of each request; NULL: q_len tokens each */
  float scale;
  int max_blocks, num_tokens, num_reqs;
  int q_len;                    /* tokens of each request, or with cu_q the most that a request has */
  int num_heads, num_kv_heads, head_size, page_size;
} qf_kv4_attention_args;

/* out[t, h] = sum_j softmax_j(scale * q[t, h] . k[j, h / G]) * v[j, h / G], G = H / H_kv, over the cached positions
 * j <= seq_lens[b] - n_b + i of token i of the n_b tokens of request b; zeros where there is none.  This step's keys and
 * values must already be in the cache.  Tokens behind the last request's are left as they were.  Scores, the softmax and the
 * sums are fp32; the cache's values are exact in the products, the softmax weights are rounded to bf16 before they multiply
 * V; the output is rounded once to bf16.
 * Lengths are kept inside the tables (0 <= seq_lens <= max_blocks * page_size, 0 <= cu_q <= num_tokens, at most q_len tokens
 * a request), block ids inside the cache.  out may be query itself.  num_heads % num_kv_heads == 0, num_heads / num_kv_heads *
 * q_len < 2^30, max_blocks * page_size <= 2^31 - 64, at most QF_KV4_MAX_REQS requests and kv heads.
 * Workspace: qf_kv4_attention_workspace_bytes(args); it needs no clearing and is free again when the last launch ends; calls
 * that may run at the same time need distinct ones (16-byte aligned). */
int qf_kv4_attention(const qf_kv4_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace of that call, by its sizes alone (0: none is needed, or the sizes are not served).  Host-only, but for
 * the current device's number of compute units. */
size_t qf_kv4_attention_workspace_bytes(const qf_kv4_attention_args* args);

#ifdef __cplusplus
}
#endif

#endif /* QF_KV4_H */
