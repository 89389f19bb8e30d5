/*
 * Paged-cache operators: quantised rows written by slot and read back, attention of a
 * tree of drafted tokens over the cache, and the verification of the drafts.  They are
 * the forms that scatter, gather, max and sum take in a serving loop, and follow the
 * library's rules: caller-owned buffers, streams and workspace, layouts with axis 0
 * fastest, metadata checked before the launch, a t4a_status returned, nothing
 * allocated and nothing synchronized.
 *
 * The cache is two tensors of pages, K and V, [pages][page_size][heads][dim] with any
 * strides (layout axes 0..3: dim, heads, page_size, pages).  dim is a multiple of 16, at
 * most 256, with unit stride, and every row starts on a 16-byte boundary.  A slot is
 * page * page_size + place.  A quantised kind holds one F32 scale per row (layout axes
 * 0..2: heads, page_size, pages): a row's values are code * scale.  A scale is not below
 * zero; attention gives NaN to whatever sees a V row that has such a one.
 */
#ifndef T4A_B200_CACHE_H_
#define T4A_B200_CACHE_H_

#include <stddef.h>

#include "abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of these operators beside T4A_CUDA_F32; the entries of abi.h and of the
 * reference do not take them. */
typedef enum {
  T4A_F16 = 32,
  T4A_BF16 = 33,
  T4A_I8 = 34,   /* cache only: codes -127..127 */
  T4A_E4M3 = 35  /* cache only: 8-bit floats, 4 exponent and 3 mantissa bits, no infinities */
} t4a_row_dtype;

typedef struct {
  int kind; /* T4A_F16, T4A_BF16, T4A_I8 or T4A_E4M3 */
  int reserved;
  void* k;
  void* v;
  float* k_scale; /* NULL for the 16-bit kinds */
  float* v_scale;
  t4a_cuda_layout k_layout;
  t4a_cuda_layout v_layout;
  t4a_cuda_layout k_scale_layout;
  t4a_cuda_layout v_scale_layout;
  long long k_len; /* elements of each buffer */
  long long v_len;
  long long k_scale_len;
  long long v_scale_len;
} t4a_kv_cache;

/* Rows key[n], value[n] (layout axes: dim, heads, rows; dtype F32, F16 or BF16; unit
 * stride along dim) into the cache at slots[n] (index_dtype I32 or I64, layout axis:
 * rows).  Quantised kinds, with Q = 127 (I8) or 448 (E4M3) and all arithmetic in F32:
 *   a = max |x|, scale = a * (1/Q), code = nearest(x * (Q/a)), ties to even;
 *   a < 2^-100: scale 0 and codes 0; a row with an infinity or a NaN: scale NaN, codes 0,
 *   so that whatever reads the row shows it.
 * 16-bit kinds: x rounded.  A slot outside [0, pages * page_size) drops its row.  Where two
 * rows have the same slot, its contents afterwards are unspecified. */
int t4a_cache_write(void* stream, int dtype, int index_dtype, const t4a_kv_cache* cache, const void* key,
                    const t4a_cuda_layout* key_layout, long long key_len, const void* value,
                    const t4a_cuda_layout* value_layout, long long value_len, const void* slots,
                    const t4a_cuda_layout* slots_layout, long long slots_len);

/* The rows at slots[n] as the values they stand for, code * scale rounded once to dtype
 * (F32, F16 or BF16), into key[n] and value[n].  A slot outside the cache reads zeros. */
int t4a_cache_read(void* stream, int dtype, int index_dtype, const t4a_kv_cache* cache, void* key,
                   const t4a_cuda_layout* key_layout, long long key_len, void* value,
                   const t4a_cuda_layout* value_layout, long long value_len, const void* slots,
                   const t4a_cuda_layout* slots_layout, long long slots_len);

/* Attention of the drafted nodes of each sequence over the paged cache.
 *   q, out: layout axes dim, query heads, nodes, batch; dtype F16 or BF16; unit stride along
 *     dim.  A 16-bit cache has q's type; query head h reads cache head h / (query heads /
 *     cache heads).
 *   table: I32, layout axes pages of a sequence, batch.  A page outside the cache is not seen.
 *   context: I32 [batch], committed tokens; node j's row is at place context + j.  Places
 *     past the table, and from 2^31 - 257 on, are not seen; a negative context counts as 0.
 *   nodes: I32 [batch], live nodes of each sequence, or NULL for all; the others see nothing
 *     and are not seen.
 *   mask: BOOL, layout axes seen node j, node i, batch (any strides, 0 among them): whether
 *     node i sees node j; NULL: j <= i, a chain.
 *   out[b, i, h] = sum_t w_t v_t, w = softmax_t(scale * q . k_t) over the context and the
 *     nodes that i sees; lse (F32, layout axes query heads, nodes, batch, or NULL) is the log
 *     of the softmax's sum.  A node that sees nothing gets zeros and -infinity.
 * Rows that a node does not see do not enter its result, whatever they hold.  Sums and the
 * softmax are in F32; a weight is rounded to the cache's 16-bit type (F16 for the quantised
 * kinds) before its product with V.  Over a quantised cache the scales of the V rows that a node
 * sees, but those of 0, lie within a factor of 2^90 of one another: a row far below that may be
 * missing from the softmax. */
int t4a_tree_attention_workspace_bytes(int dtype, const t4a_kv_cache* cache, const t4a_cuda_layout* q_layout,
                                       const t4a_cuda_layout* table_layout, size_t* bytes);
int t4a_tree_attention(void* stream, int dtype, const t4a_kv_cache* cache, void* out,
                       const t4a_cuda_layout* out_layout, long long out_len, float* lse,
                       const t4a_cuda_layout* lse_layout, long long lse_len, const void* q,
                       const t4a_cuda_layout* q_layout, long long q_len, const int* table,
                       const t4a_cuda_layout* table_layout, long long table_len, const int* context, const int* nodes,
                       const unsigned char* mask, const t4a_cuda_layout* mask_layout, long long mask_len, float scale,
                       void* workspace, size_t workspace_bytes);

/* Walks each sequence's tree of drafted tokens from node 0, the last committed token.
 *   logits: layout axes vocab, nodes, batch, dtype F32, F16 or BF16, unit stride along vocab:
 *     the target after each node.  tokens, parents: I32 [batch][nodes], compact; a parent's
 *     index is below its child's, and node 0's entries are not read.
 *   draft: F32, layout axes vocab, nodes, batch, or NULL: the distribution that a node's
 *     children were drawn from, each independently, so that siblings may be alike.  Children
 *     drawn without replacement, or picked as the likeliest, need draft NULL: the tokens said then
 *     follow the target wherever the children came from; with a draft they would not.  uniforms: F32 [batch][nodes], compact, in [0, 1).
 *   race: F32, layout axes vocab, batch: reciprocals of standard exponential variates.
 * At a node r = softmax(logits / temperature).  Its children are tried in order: child c with
 * token x is taken when uniforms[c] * draft[x] < r[x] (draft[x] = 1 without draft).  Else r
 * becomes max(r - draft, 0), or r without x, divided by its sum (the node's softmax where that
 * sum is 0).  When no child is left the last token is argmax_x r[x] * race[x], lowest index
 * first.  temperature 0: a child is taken when its token is the lowest-index argmax of the
 * logits, which is the last token too; uniforms, race and draft are not read.
 * Logits of -infinity have no probability; NaN counts as -infinity.  At most 1024 nodes, and as
 * many tokens as 8 blocks keep a row of: 376,000, or 753,000 in 16 bits without a draft
 * (T4A_ERR_DOMAIN_TOO_LARGE beyond).
 *   count [batch]: nodes taken.  path, said [batch][nodes], compact I32: the nodes taken, and
 *     their tokens with the last token after them; -1 in the other places.
 *   logs [batch][nodes], compact F32, or NULL: the log-probability of each token said (at
 *     temperature 1 where it is 0); 0 in the other places. */
int t4a_verify_drafts(void* stream, int dtype, const void* logits, const t4a_cuda_layout* logits_layout,
                      long long logits_len, const int* tokens, const int* parents, const float* uniforms,
                      const float* draft, const t4a_cuda_layout* draft_layout, long long draft_len, const float* race,
                      const t4a_cuda_layout* race_layout, long long race_len, float temperature, int* count, int* path,
                      int* said, float* logs);

#ifdef __cplusplus
}
#endif

#endif /* T4A_B200_CACHE_H_ */
