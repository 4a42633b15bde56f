/*
 * tq4 paged key-value cache: what fills it, reads it and trims it when a q4 decoder serves many
 * sequences at once. tq4_decoder.h attends over one contiguous f32 cache at one position; here a
 * pool of pages holds the rows of every sequence, in f32, f16 or bf16.
 *
 * The pool: k_pages and v_pages, each [num_pages][kv_heads][page_size][head_dim], and a page table
 * [max_seqs][max_pages] of int32 page numbers. Slot j of sequence s is row j % page_size of page
 * page_table[s][j / page_size]; entries behind a sequence's last page are never read. Several
 * sequences may list the same page (a shared prefix). A sequence's length and a token's slot count
 * cache rows; positions (the angles of the rotary embedding) are given apart, so that a trimmed
 * sequence keeps counting positions where it was.
 *
 * Pointers are device pointers of the handle's device unless "host" is said; every call enqueues
 * on `stream` and may be captured into a CUDA graph (lengths, slots and tables live on the device).
 * A length, slot, sequence, position or page number out of range never leads out of bounds: what it
 * stands for is skipped and the device status set to 0x200 (tq4_device_status). Where the attention's own waits ran
 * out (0x107, tq4_set_wait_limit), what the call's outputs hold is not defined.
 */
#ifndef TQ4_PAGED_H
#define TQ4_PAGED_H

#include "tq4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The pool's type and sizes. head_dim values of a row take a multiple of 16 bytes and are at most
 * 256; page_size is a power of two. */
typedef struct {
  tq4_dtype dtype; /* of the pages, and of q, k, v and the attention's output */
  int32_t kv_heads;
  int32_t head_dim;
  int32_t page_size;
  int64_t num_pages;
  int32_t max_seqs;  /* rows of the page table */
  int32_t max_pages; /* its columns */
} tq4_paged_desc;

typedef struct tq4_paged tq4_paged;

/* A handle over memory that stays the caller's: 16-byte aligned pages, and the page table, whose
 * entries may change between calls. */
tq4_status tq4_paged_create(const tq4_paged_desc* desc, void* k_pages, void* v_pages,
                            const int32_t* page_table, int device, tq4_paged** out);
tq4_status tq4_paged_destroy(tq4_paged* cache);

/* The rotary embedding and the per-head RMSNorm before it. The first 2 * pairs values of a head
 * are turned: pair i is values (i, i + pairs), or (2i, 2i + 1) with interleaved = 1 (rotate/4,
 * lib/transmuter/ops/transformer.ex:558-590), by the angle whose cosine and sine stand in row
 * positions[axis][token] and column i of the f32 tables [max_pos][pairs]. With several axes (time,
 * height and width of an image's patches) pair i follows axis pair_axis[i]; pair_axis is host
 * memory of `pairs` entries below `axes`, or NULL where every pair follows axis 0. q_w and k_w are
 * f32 [head_dim] norm weights (rms_norm/4, :1056-1069), or NULL for no norm. */
typedef struct {
  const float* cos_table;
  const float* sin_table;
  int64_t max_pos;
  int32_t pairs;
  int32_t axes; /* 1 to 4 */
  const uint8_t* pair_axis;
  int32_t interleaved;
  const float* q_w;
  const float* k_w;
  float eps;
} tq4_rotary;

/* Writes the keys and values of `tokens` new tokens into the cache, and their turned queries to
 * q_out: token t is row slot[t] of sequence seq[t]. q [tokens][heads][head_dim], k and v
 * [tokens][kv_heads][head_dim], each token's heads contiguous and tokens `*_stride` values apart
 * (views of one merged projection); q_out is dense. positions is int32 [axes][tokens]. Norm and
 * rotation are computed in f32 and rounded once. seq[t] < 0 marks a padding token: nothing is
 * written for it, its row of q_out included. rotary may be NULL (no norm, no rotation;
 * positions unused), and q NULL with heads 0 (only the cache is filled). The (seq, slot) of two
 * tokens of a call must differ, and so must the cache rows that they stand for where sequences share
 * pages: which of the two would remain is not defined. q_out may not overlap q, k or v, and no
 * input may lie in the cache rows that the call writes. Where nothing is turned and there is no norm,
 * values are copied bit for bit. */
tq4_status tq4_paged_append(const tq4_paged* cache, const void* q, int64_t q_stride, const void* k,
                            int64_t k_stride, const void* v, int64_t v_stride, int heads,
                            int64_t tokens, const int32_t* seq, const int32_t* slot,
                            const int32_t* positions, const tq4_rotary* rotary, void* q_out,
                            void* stream);

/* Bytes of workspace that tq4_paged_attention needs for these sizes, whatever the lengths and the window: at most 119 MB
 * and batch * (heads + 1) * 8 bytes, and with scores heads * 4 bytes more a slot of the page table's first batch rows,
 * in use or not (64 rows of 131072 slots and 32 heads: 1.07 GB). 0 for few short rows without scores. */
tq4_status tq4_paged_attention_workspace(const tq4_paged* cache, int heads, int64_t batch,
                                         int with_scores, int64_t* bytes);

/* Attention of one new token of each sequence (GroupQueryAttention, transformer.ex:106-175):
 *   out[b][h] = sum_j softmax_j(scale * q[b][h] . K[j]) V[j],  lengths[b] - window <= j < lengths[b]
 * over the rows of KV head h / (heads / kv_heads) of sequence b = row b of the page table, the new
 * token's own row among them (append it first). window = 0 attends to the whole sequence. A
 * sequence of length 0 gives zeros, and so does a head whose every score is -inf; a NaN among a head's scores gives NaN.
 * q is [batch][heads][head_dim], rows q_stride values apart; out is dense and may not overlap q, nor any other buffer of
 * the call. heads is any multiple of kv_heads.
 * With scores and new_scores (f32 [batch][kv_heads][max_pages * page_size], both or neither; they
 * may be the same buffer), the softmax weights that eviction goes by are accumulated: slot j of
 * new_scores is that of scores plus the sum over the KV head's query heads of slot j's weight, and
 * slots at and behind lengths[b] are left as they were.
 * workspace: 16-byte aligned device memory that this call has to itself until it has run (NULL where
 * 0 bytes are needed); what it held before does not matter.
 * Sums, maxima and outputs are accumulated in f32. Over a 16-bit cache each softmax weight is rounded once to the cache's
 * type before it multiplies its value (f16: scaled by 2^15 first); the weights' sum and the scores take it unrounded. The
 * order of the sums depends on the sizes, the page table's shape, the window, whether there are scores, and all lengths
 * of the batch: calls that are equal in these give equal bits, others may differ in the last bits of f32. */
tq4_status tq4_paged_attention(const tq4_paged* cache, const void* q, int64_t q_stride, int heads,
                               const int32_t* lengths, int64_t batch, float scale, int64_t window,
                               const float* scores, float* new_scores, void* out, void* workspace,
                               int64_t workspace_bytes, void* stream);

/* Eviction by accumulated attention weight. Of each sequence b longer than `keep`, and for each of
 * its KV heads apart, the last `recent` slots stay and of those before them the keep - recent with
 * the highest scores (equal scores: the lower slot; NaN counts as lowest). Shorter sequences stay
 * whole. What stays moves, in the order of its slots, to the first rows of the pages of
 * new_table[b] (int32 [batch][new_max_pages]); kept [batch][kv_heads][keep] tells the old slots
 * (-1 behind the last), new_lengths [batch] the new lengths, and new_scores, if not NULL, takes the
 * scores along (rows new_score_stride >= keep values apart; what lies behind is left as it was).
 * The pages of new_table are pages of the same pool, each in one place of it, that no sequence of
 * this call lists in its page table: the old rows are only read, so that pages shared with other
 * sequences stay whole. No output may overlap an input or another output. */
tq4_status tq4_paged_evict(const tq4_paged* cache, const int32_t* lengths, int64_t batch,
                           const float* scores, int64_t keep, int64_t recent,
                           const int32_t* new_table, int32_t new_max_pages, int32_t* new_lengths,
                           int32_t* kept, float* new_scores, int64_t new_score_stride,
                           void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TQ4_PAGED_H */
