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

/* ---------------------------------------------------------------------------------------------- rotary positions
 * A row at position p has the pairs of the first `width` values of each head turned by the angle p * turn[i], and
 * multiplied by amplitude; the other values stay:
 *     y_a = amplitude * (x_a cos - x_b sin),  y_b = amplitude * (x_a sin + x_b cos)
 * Pair i is (i, i + width / 2), or with `interleaved` (2 i, 2 i + 1).  turn: width / 2 angles in radians, 64 bits, on the
 * device.  The angle is reduced in 64 bits (off by 3 * 2^-53 of itself at most; positions beyond 2^53 are rounded to 64-bit
 * floating point first); its sine and cosine, times amplitude, are rounded to 32 bits, and so are each product and their
 * sum, by themselves: none is fused. */
typedef struct MxRotary {
  const double* turn;
  int32_t width, interleaved;
  double amplitude;
} MxRotary;

size_t mx_rotary_bytes(void);                /* sizeof(MxRotary) */

/* Turn rows (F32, BF16 or F16; out of the same type) of head_dim values by positions[token % period], int32, or int64
 * with `wide`; `back` turns by the negative angle, with the same amplitude: this is the gradient.  width is even, from 2 to
 * head_dim, which is at most 1024.  x and out must not share memory. */
int mx_rotate(const MxRotary* rotary, const MxRows* x, const MxRows* out, int32_t head_dim, int32_t tokens,
              const void* positions, int32_t period, int32_t wide, int32_t back, void* stream);

/* Turn the chunk's queries and keys by their rows' positions in their worlds (length[w] - n_w + i), the queries to `out`, the
 * keys on into the pages, with the values beside them as mx_episode_write stores them; keys are rounded once, when they
 * are stored.  All rows have one type.  Rows that belong to no world are left out, their places in `out` as they were. */
int mx_episode_enter(const MxPages* pages, const MxChunk* chunk, const MxRotary* rotary, const MxRows* q, const MxRows* out,
                     const MxRows* k, const MxRows* v, void* stream);

/* ---------------------------------------------------------------------------------------------- room for tokens
 * The worlds' tables and lengths and the pages that none of them has: free[0 .. state[0]) is a stack of page numbers, of
 * npage places.  state[1] collects what was refused (MX_ROOM_*); it is never cleared here.  A world has the pages of its
 * first (length + page_tokens - 1) / page_tokens table entries and holds at most `tokens` tokens. */
typedef struct MxRoom {
  int32_t *table, *length, *free, *state;
  int32_t nworld, width, npage, page_tokens, tokens;
} MxRoom;

#define MX_ROOM_TOKENS 1    /* a world would pass `tokens` (or the table), or fall below no token */
#define MX_ROOM_PAGES  2    /* the free pages do not suffice */
#define MX_ROOM_ROWS   4    /* more new rows than `rows` */

/* A change of all worlds: those of `over` (nworld bytes, null: none) are emptied; then world w gets count[w] new tokens
 * (count null: `each`), or gives back its last -count[w].  Pages come off the stack in the order of the worlds and their
 * tokens, and go onto it in the opposite order, so that tokens taken back leave tables and stack as they were.
 * If any world or the stack refuses, no world gets or gives back tokens, and state[1] says why; `over` is done all the
 * same.  start (nworld + 1, null: not wanted) becomes the sums of the new tokens before each world (of a refused change,
 * and for tokens given back, 0): the chunk to write and attend with.  rows: the most rows that the chunk may have.
 * workspace: mx_room_workspace bytes, 16-byte aligned. */
typedef struct MxRoomChange {
  const int32_t* count;
  const uint8_t* over;
  int32_t* start;
  void* workspace;
  size_t workspace_bytes;
  int32_t each, rows;
} MxRoomChange;

size_t mx_room_bytes(void);                  /* sizeof(MxRoom) */
size_t mx_room_change_bytes(void);           /* sizeof(MxRoomChange) */
size_t mx_room_workspace(const MxRoom* room);
int mx_room_update(const MxRoom* room, const MxRoomChange* change, void* stream);

/* World, position and slot (page * page_tokens + place in it) of each of the chunk's rows; -1, -1, -1 for rows that belong
 * to no world, -1 as position for rows before the world's first token, and as slot for those without a place.  Of the
 * room, table and length are read; free and state may be null. */
int mx_room_places(const MxRoom* room, const MxChunk* chunk, int32_t* world, int32_t* position, int32_t* slot, void* stream);

/* ---------------------------------------------------------------------------------------------- recall
 * Attention of a query to some blocks of block_tokens tokens (a power of two from 16 to page_tokens) of its world: the
 * blocks whose summaries match it best, the latest ones, and the first ones.
 *
 * The summary of a block that is full is the mean m of its keys (in 64 bits): codes c = rint(m / 2^e), |c| <= 127, with
 * the least e from -40 to 40 at which |m| is at most 127 * 2^e (codes beyond are cut off), and the byte e + 127; a block
 * with a key that is not finite has the byte 255.  codes [npage][kv_heads][page_tokens / block_tokens][head_dim], 16-byte
 * aligned, exponent without head_dim. */
typedef struct MxSummaries {
  int8_t* codes;
  uint8_t* exponent;
  int32_t block_tokens;
} MxSummaries;

/* What mx_episode_select chooses for each of the chunk's rows and key heads: of the world's blocks, those that begin at
 * or before the last token that the query sees, the blocks [0, first); from the `near`-th block before the one behind the
 * query's own on, all; and of those between the `top` with the largest scores, of equal ones the earlier.  The score of a block is
 *     max over the query heads h of the key head of  (sum_d q_hd c_d) 2^(e_h + e),
 * with q_h in codes of its own head by the rule above (a NaN counts as 0, an infinity as cut off): exact in 32 bits,
 * the same on any machine.  The byte 255 stands above all scores, a table entry that names no page below.
 * blocks: tokens x kv_heads x width, filled from the left in ascending order, then -1; all of it is written, -1 for rows
 * that see nothing, belong to no world, or lie beyond max_count in it.  width is at least first + near + top, and at most
 * 4096; top at most 1024.  Where queries see tokens behind them (causal 0) it has to be more by (n + block_tokens - 2) /
 * block_tokens for chunks of n tokens, also where max_count is less: a list without that room leaves out its last
 * blocks. */
typedef struct MxSelection {
  int32_t* blocks;
  int32_t width, top, near, first, max_count, causal;
} MxSelection;

size_t mx_summaries_bytes(void);             /* sizeof(MxSummaries) */
size_t mx_selection_bytes(void);             /* sizeof(MxSelection) */

/* The summaries of the blocks that the chunk's tokens complete, from the keys in the pages. */
int mx_episode_summarise(const MxPages* pages, const MxChunk* chunk, const MxSummaries* summaries, void* stream);

int mx_episode_select(const MxPages* pages, const MxChunk* chunk, const MxSummaries* summaries, const MxRows* q,
                      const MxSelection* selection, void* stream);

/* mx_episode_attend over the keys of the listed blocks: s->blocks, s->width and block_tokens are read, the other numbers
 * of s are not.  A block counts as often as it is listed; numbers that are no block of the world's table are left out.
 * The probabilities are in two parts.  a->longest says how to divide the work, as for mx_episode_attend.  a->window must
 * be 0. */
int mx_episode_recall(const MxPages* pages, const MxChunk* chunk, const MxAttention* a, const MxSelection* s,
                      int32_t block_tokens, void* stream);

size_t mx_recall_workspace(const MxPages* pages, const MxChunk* chunk, const MxAttention* a, const MxSelection* s,
                           int32_t block_tokens);

#ifdef __cplusplus
}
#endif
#endif /* MX_EPISODE_H */
