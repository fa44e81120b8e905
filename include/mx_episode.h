/*
 * mx_episode.h -- C ABI of the episode memory in libmx_physics.so: the keys and values of every
 * world's running episode in pages that the worlds of a batch share, for an attention policy that
 * steps with the batch (mx_physics.h).  Conventions are those of mx_physics.h: every pointer is a
 * device pointer owned by the caller, the library never allocates and never synchronizes, the
 * argument structs are read on the host, 0 = success, > 0 = HIP error code, < 0 = MX_ERR_*, found
 * before any launch.  All calls can be captured into a HIP graph; table, length and start are read
 * on the device, so a replay follows their contents.
 *
 * A chunk is the last n_w of each world's length[w] tokens: mx_episode_write stores a chunk's keys and
 * values, mx_episode_read returns them, mx_episode_attend attends from the chunk's queries to the
 * world's tokens.  Rows are packed world by world: with start == null every world has `count` rows;
 * otherwise world w has the rows start[w] .. start[w + 1] of `tokens` rows (start[0] = 0,
 * start[nworld] = tokens, nondecreasing; rows outside `tokens` are never touched).  A chunk longer
 * than its world's length has only its last length[w] tokens; tokens beyond the table's reach, or
 * whose table entry names no page, are neither written nor seen, and read as zeros.  Sizes that would take
 * more than 2^24 - 1 workgroups of 256 threads (2^30 rows of one write) are MX_ERR_DOMAIN.
 */
#ifndef MX_EPISODE_H
#define MX_EPISODE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MX_ERR_WORKSPACE (-5)   /* mx_episode_attend: workspace missing, misaligned or too small */

/* Element types of rows, and of pages (F32 for rows of write and read only, FP8 for pages only). */
#define MX_TYPE_F32  0
#define MX_TYPE_BF16 1
#define MX_TYPE_F16  2
#define MX_TYPE_FP8  3

/* 8-bit pages: OCP e4m3 codes with one E8M0 scale byte b (2^(b - 127)) per MX_SCALE_BLOCK values along
 * head_dim.  mx_episode_write takes the least power of two, 2^-117 at least, at which the block's
 * largest magnitude is within the codes' 448, and rounds to nearest even; a block with an infinity or
 * NaN gets b = 255 and reads back as NaN. */
#define MX_SCALE_BLOCK 32

/* Pages of keys and values: k, v [npage][kv_heads][page_tokens][head_dim], 16-byte aligned; scales (FP8,
 * otherwise null) [npage][kv_heads][page_tokens][head_dim / 32].  Token t of world w is slot
 * t % page_tokens of page table[w * width + t / page_tokens].  page_tokens: a power of two from 16 to
 * 4096; head_dim: 32, 64, 96, 128 or 256; npage * page_tokens below 2^31, width * page_tokens at most 2^30. */
typedef struct MxPages {
  void *k, *v;
  uint8_t *k_scale, *v_scale;
  const int32_t *table, *length;
  int32_t nworld, npage, width, kv_heads, head_dim, page_tokens, type;
} MxPages;

/* The chunk's rows (see above): start, and either count (start null; tokens = nworld * count) or tokens. */
typedef struct MxChunk {
  const int32_t* start;
  int32_t tokens, count;
} MxChunk;

/* Rows of heads: element (token, head, d) at data[token * token_stride + head * head_stride + d]; strides in
 * elements.  Any alignment of the element type; 16-byte aligned rows are the faster ones. */
typedef struct MxRows {
  void* data;
  int64_t token_stride, head_stride;
  int32_t heads, type;
} MxRows;

size_t mx_pages_bytes(void);                 /* sizeof(MxPages)  */
size_t mx_chunk_bytes(void);                 /* sizeof(MxChunk)  */
size_t mx_rows_bytes(void);                  /* sizeof(MxRows)   */
size_t mx_attention_bytes(void);             /* sizeof(MxAttention) */

/* Store the chunk's keys and values (kv_heads heads, any of F32, BF16, F16) into its slots. */
int mx_episode_write(const MxPages* pages, const MxChunk* chunk, const MxRows* k, const MxRows* v, void* stream);

/* The chunk's keys and values as the pages stand for them, rounded once to the rows' type. */
int mx_episode_read(const MxPages* pages, const MxChunk* chunk, const MxRows* k, const MxRows* v, void* stream);

/* Softmax attention of the chunk's queries over their worlds' tokens.  Query head h uses key head
 * h / (heads / kv_heads).  The query at position p = length[w] - n_w + i sees the keys j <= p (causal) or
 * j < length[w], and of those the `window` last up to its own position (j > p - window) when window > 0:
 *     out = sum_j exp(scale * q.k_j - m) v_j / sum_j exp(scale * q.k_j - m),  lse = m + log(sum)
 * A query that sees no key, or none with a score above -infinity, gives out 0 and lse -infinity.
 *
 * Scores, sums, lse and out before its one rounding are in 32 bits.  The probabilities that multiply the values are
 * rounded to the queries' type: in two parts, value and remainder, where few rows (new tokens x query heads) share a key
 * head (16, with 8-bit pages 32), in one where more do.  float16 probabilities below 2^-26 of a row's largest lose bits,
 * those below 2^-37 count in the sum alone.  Sums of weighted values that pass 32 bits (bfloat16 values of 2^116 and more)
 * are infinities.  An infinity or NaN in a value reaches all queries that see its key, whatever its weight, and no others.
 *
 * q and out have one type, BF16 or F16, which is the pages' too unless those are FP8 (whose values are then taken in q's
 * type).  max_count bounds n_w (a longer chunk's rows beyond it are not computed).  longest: the most tokens that a world
 * has, if the caller knows (0: not known); it says how to divide the work, and worlds that are longer all the same only
 * take longer.  lse (tokens x heads floats) may be null.  workspace: mx_episode_workspace bytes, 16-byte aligned, its
 * contents undefined before and after (null when that is 0). */
typedef struct MxAttention {
  MxRows q, out;
  float* lse;
  void* workspace;
  size_t workspace_bytes;
  int32_t max_count, causal, window;
  float scale;
  int32_t longest;
} MxAttention;

int mx_episode_attend(const MxPages* pages, const MxChunk* chunk, const MxAttention* a, void* stream);

/* Bytes of workspace that mx_episode_attend takes for these sizes (which of the pointers are set does not
 * matter); 0 also for arguments that it refuses. */
size_t mx_episode_workspace(const MxPages* pages, const MxChunk* chunk, const MxAttention* a);

#ifdef __cplusplus
}
#endif
#endif /* MX_EPISODE_H */
