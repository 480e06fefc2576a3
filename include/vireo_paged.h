/* Serving many sequences from one paged key-value cache in 16 bits.
 *
 * The KV stores of vireo_kv.h hold one sequence in fp32 and are paged by the
 * host. Here a pool of blocks of block_tokens tokens is shared by many
 * sequences, everything that changes from step to step (block tables, lengths,
 * free blocks, positions) lives in device memory, and every call only reads
 * and writes memory that the caller owns: nothing is allocated, nothing waits
 * for the device, and a whole step can be captured in a HIP graph. One table
 * serves every layer; each layer has a cache of its own over the same blocks.
 *
 * One step of a batch of n sequences:
 *
 *   vireo_paged_extend        blocks, lengths, positions and slots for the new tokens
 *   vireo_paged_plan_update   how the batch's attention is split
 *   per layer:
 *     vireo_paged_append      q and k norms, rotation, k and v into the cache
 *     vireo_paged_select      (optional) the blocks each sequence attends to
 *     vireo_paged_attend      one new token per sequence over its blocks
 *
 * and vireo_paged_truncate when tokens are taken back or a sequence ends.
 * Nothing of it has a counterpart in the reference, whose stores hold one
 * sequence (src/kvstore.h); the attention is its softmax(q . k / sqrt(d)) . v
 * (src/kvstore.h:68-99) and the selection its sinks, window and top blocks by
 * mean key (src/kvstore_ooc.c:163-176, src/select/select_topk.c).
 *
 * Structs and their pointers to structs are read during the call (host
 * memory); every other pointer is a device pointer. Streams and return values
 * are those of vireo_hip.h: with stream NULL a call waits for its work. Calls
 * on different streams are independent as long as they write different
 * memory: two that share a table, a cache being written or a plan's memory
 * need an order between them. */
#ifndef VIREO_PAGED_H
#define VIREO_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types (ggml's numbers) */
enum { VIREO_PAGED_F32 = 0, VIREO_PAGED_F16 = 1, VIREO_PAGED_BF16 = 30 };

/* ---- block tables ----------------------------------------------------------- */

/* Which blocks of the pool hold which tokens. Sequence s's token t lies in
 * block blocks[s * max_blocks + t / block_tokens] at t % block_tokens, its slot
 * being block * block_tokens + t % block_tokens. free_blocks[0 .. n_free) are
 * the unused blocks, a stack with its top at the end. The caller allocates the
 * four arrays and may read them at any time; it may fill them itself instead of
 * calling vireo_paged_reset (a block in two rows, or in a row and in the free
 * list, is the caller's to answer for: e.g. a prompt shared by sequences that
 * never write into its blocks). */
typedef struct {
    int max_seqs;         /* sequences: 1 .. 4096 */
    int max_blocks;       /* blocks a sequence may have: no more than are needed (vireo_paged_select takes
                             longer over wide tables, and vireo_paged_attend a second launch) */
    int n_blocks;         /* blocks of the pool; n_blocks * block_tokens < 2^31 */
    int block_tokens;     /* 16, 32, 64 or 128 */
    int32_t *blocks;      /* [max_seqs x max_blocks] */
    int32_t *len;         /* [max_seqs] tokens of each sequence */
    int32_t *free_blocks; /* [n_blocks] */
    int32_t *n_free;      /* [1] */
} vireo_paged_table;

/* Every sequence empty, every block free (block 0 on top of the stack), the
 * table's entries -1. */
int vireo_paged_reset(const vireo_paged_table *t, void *stream);

/* Room for the next tokens of n sequences: sequence ids[i] (NULL: i) grows by
 * n_new[i] tokens (NULL: 1), i < n <= max_seqs. The step's rows are the new
 * tokens in the batch's order: start [n + 1] receives the rows before each
 * sequence's (start[n]: their number), positions and slots [max_rows] each
 * row's position in its sequence and its slot; a row past the last one, and a
 * row of a sequence that was refused, gets slot -1 (past the last one, or where
 * the entry is not a sequence, -EINVAL, position 0).
 * status [n] says what became of each sequence:
 *   0         extended: its blocks are in the table and len has grown
 *   -EINVAL   ids[i] outside [0, max_seqs), or also an earlier one of the
 *             batch's, or n_new[i] < 0 (counted as 0 rows)
 *   -E2BIG    longer than max_blocks blocks, or its rows do not fit max_rows
 *   -ENOSPC   the free blocks do not last: sequences take them in the batch's
 *             order, and from the first that finds too few none that needs a
 *             block gets one (sequences that need none are extended)
 * A refused sequence keeps its blocks and length. New blocks come from the top
 * of the stack, in the batch's order and in the order of positions. */
int vireo_paged_extend(const vireo_paged_table *t, const int32_t *ids, const int32_t *n_new, int n, int max_rows,
                       int32_t *start, int32_t *positions, int32_t *slots, int32_t *status, void *stream);

/* Sequence ids[i] (NULL: i) is cut back to new_len[i] tokens (NULL: 0, which
 * ends it) if it is longer; blocks that hold none of them go back on the stack,
 * in such an order that the same extension takes them again. An id outside
 * [0, max_seqs) or one that came before in the batch, and a negative length,
 * change nothing. Table entries past a sequence's blocks keep their old values. */
int vireo_paged_truncate(const vireo_paged_table *t, const int32_t *ids, const int32_t *new_len, int n, void *stream);

/* ---- one layer's cache -------------------------------------------------------- */

/* Keys and values of every block, 16 bits each: k [n_blocks x n_kv_heads x
 * block_tokens x head_size], token by token, and v [n_blocks x n_kv_heads x
 * head_size x block_tokens], dimension by dimension (both as the matrix cores
 * take them: a lane's 8 operand values are consecutive). means, if not NULL:
 * [n_blocks x n_kv_heads x head_size], the mean key of each full block, for
 * vireo_paged_select. All 16-byte aligned. */
typedef struct {
    uint32_t type;    /* VIREO_PAGED_F16 or VIREO_PAGED_BF16 */
    int n_blocks, block_tokens, n_kv_heads;
    int head_size;    /* 64, 128 or 256 */
    void *k, *v, *means;
} vireo_paged_cache;

/* The step's rows of one layer: q [rows x n_heads x head_size], k and v [rows x
 * n_kv_heads x head_size] of `type`, a row's heads consecutive and rows
 * `stride` elements apart (so they may be parts of one projection's output). */
typedef struct {
    int rows, n_heads;
    uint32_t type;                          /* F32, F16 or BF16 */
    const void *q, *k, *v;                  /* 16-byte aligned, and so are the rows */
    int64_t q_stride, k_stride, v_stride;   /* elements */
    const float *q_bias, *k_bias, *v_bias;  /* [heads x head_size], NULL: none */
    const float *q_norm, *k_norm;           /* [head_size] RMSNorm weights of every head, NULL: no norm (one over the
                                               row's whole q or k goes before this call: vireo_rmsnorm) */
    float eps;
    const float *rope;                      /* [max_pos x rotary] from vireo_rope_table(base, rotary, max_pos) */
    int rotary;                             /* dimensions rotated, the first ones: a multiple of 16, <= head_size */
    int max_pos;
    const int32_t *positions, *slots;       /* [rows] */
    void *q_out;                            /* [rows x n_heads x head_size], 16-byte aligned rows; may be q, with its
                                               stride and element size */
    uint32_t q_out_type;                    /* F32 or the cache's */
    int64_t q_out_stride;
} vireo_paged_rows;

/* Per row: q and k heads get their bias, their RMSNorm over the head and the
 * NEOX rotation at the row's position (src/gguf_run.c:166-179; a position
 * outside [0, max_pos) rotates nothing), v heads their bias; computed in fp32
 * and rounded once: q into q_out, k and v into the cache at the row's slot. A row
 * whose slot lies outside the pool (padding, a refused sequence) is left out:
 * neither the cache nor q_out changes. Two rows of one call must not have the
 * same slot. With c->means, a row in the last slot of a block also sets that
 * block's mean key, from the keys as stored; those of the block's other slots
 * have to be there by the end of the call. -E2BIG for more heads of rows than one
 * launch takes (2^28 queries and keys of 256, 2^30 of 64, or somewhat fewer beside the values). */
int vireo_paged_append(const vireo_paged_cache *c, const vireo_paged_rows *r, void *stream);

/* ---- attention of one new token per sequence ------------------------------------ */

/* A batch and the split of its attention over the device, made once per step
 * (lengths change) and used by every layer. The fields describe the batch;
 * mem is device memory of vireo_paged_plan_bytes bytes, 256-byte aligned: the
 * split and the attention's partial results. Calls that may run at the same
 * time (other streams, graphs replayed at once) need plans of their own. The
 * memory says which shape it was split for (the fields but ids, and the table's
 * max_seqs, max_blocks and block_tokens): where that is another, or there was no update
 * yet, vireo_paged_attend and vireo_paged_select return 0 and leave out and lists as
 * they were, since only the device knows. */
typedef struct {
    const vireo_paged_table *table;
    const int32_t *ids;      /* [n] rows of the table, NULL: 0 .. n - 1; an id outside it is an empty sequence */
    int n;                   /* 1 .. 4096 */
    int n_heads, n_kv_heads; /* head h reads kv head h / (n_heads / n_kv_heads) */
    int head_size;
    int list_blocks;         /* 0: every block is attended; else the width of the lists of blocks */
    void *mem;
} vireo_paged_plan;

/* Bytes of plan memory, or -EINVAL. */
int64_t vireo_paged_plan_bytes(const vireo_paged_plan *p);
/* Split the batch by the lengths that the table has now. Before the first
 * attend or select of a step, after vireo_paged_extend. */
int vireo_paged_plan_update(const vireo_paged_plan *p, void *stream);

/* out_i = softmax(scale q_i . K) V over sequence i's tokens, its newest among
 * them (extend and append come first): q, out [n x n_heads x head_size], rows
 * q_stride / out_stride elements apart, of `type` (F32 or the cache's), 16-byte
 * aligned. out may be q, with its stride. scale > 0. An empty sequence gives zeros.
 * Products, sums and the softmax are in fp32 or exact: fp32 queries and the weights
 * are split into three 16-bit parts (over fp16 what lies below 2^-38 of a head's
 * largest query value or of the largest weight is cut off). There is one query per
 * sequence, its newest token's: the tokens of a prompt, or of drafts, that need
 * attention of their own go through extend, append and attend one by one (an id
 * named twice attends to the same tokens twice).
 * lists (NULL unless p->list_blocks > 0): [n x n_kv_heads x list_blocks], for
 * each kv head the blocks of the sequence that its heads attend to, by their
 * number in the sequence; only a sequence's first min(its blocks, list_blocks)
 * entries are read, and entries outside it (-1) are skipped. A table entry
 * outside the pool is skipped too; where nothing is left the output is zeros. */
int vireo_paged_attend(const vireo_paged_cache *c, const vireo_paged_plan *p, const void *q, uint32_t type,
                       int64_t q_stride, float scale, const int32_t *lists, void *out, int64_t out_stride,
                       void *stream);

/* The blocks worth attending to: for every sequence and kv head, lists [n x
 * n_kv_heads x p->list_blocks] receives in ascending order the first `sinks`
 * blocks, the last `window` (>= 1: the block being written has no mean key yet)
 * and, of those between, the list_blocks - sinks - window whose score is
 * highest: the largest, over the kv head's query heads, of q . mean key, summed
 * in fp64 and rounded to fp32 (a NaN counts as -inf); of equal ones the lower
 * block first. A sequence of at most list_blocks blocks gets all of them, then
 * -1. c->means is required. -E2BIG for a table of more than 65536 blocks a sequence
 * beside sinks and window. Lengths are those at the plan's update. q as in
 * vireo_paged_attend. Its time goes by the table's width too, not by the lengths alone,
 * most of all beyond 8192 blocks a sequence. */
int vireo_paged_select(const vireo_paged_cache *c, const vireo_paged_plan *p, const void *q, uint32_t type,
                       int64_t q_stride, int sinks, int window, int32_t *lists, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* VIREO_PAGED_H */
