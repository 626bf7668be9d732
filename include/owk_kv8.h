/*
 * owk_kv8.h -- keys and values held in 8 bits: filling the cache, attending over it, reading it back.
 *
 * A sequence's tokens are held in blocks of OWK_KV8_BLOCK. A complete block holds, for each key/value
 * head and for keys and values apart, 64 * head_dim signed codes and one scale s = max|x| / 127 (f32):
 * a code c = rint(x / s) stands for c * s. The last, incomplete block of a sequence (its tail) stays in
 * the 16-bit type it came in until its 64 tokens are there, so what a token is rounded to depends on
 * the data alone and never on how many tokens a call brought. (What is attended does depend on it: tokens are
 * seen as the cache holds them when the call runs, so the tokens of a chunk that completes a block see
 * codes where tokens that came one by one saw 16 bits.) A block with a value that is not finite
 * reads as NaN throughout (keys or values of that head).
 *
 * All pointers are device memory of `device`; every call is queued on `stream` (a hipStream_t, NULL =
 * the default stream) and returns without waiting. Nothing is allocated, kept or read back, so calls
 * can be captured into a graph; lengths are read on the device and may change between replays.
 * Calls on different sequences or caches may overlap. Two entries of one append must not name the same
 * sequence, and two calls in flight must not share a workspace.
 *
 * Return value: 0, OWK_KV8_INVALID (arguments; nothing was queued) or OWK_KV8_HIP (the launch failed);
 * owk_kv8_error() says what was wrong. What only the device can see is bounded there: an entry with a
 * sequence outside [0, n_seqs) has no keys and stores nothing, a table entry outside [0, n_blocks) hides
 * its block (no store, no keys, read as zeros), lengths are cut to the capacity of max_blocks blocks,
 * rows to `rows`.
 */
#ifndef OWK_KV8_H
#define OWK_KV8_H

#include <stddef.h>
#include <stdint.h>

#include "whisper.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OWK_KV8_BLOCK 64

enum owk_kv8_type { OWK_KV8_F16 = 0, OWK_KV8_BF16 = 1, OWK_KV8_F32 = 2 /* outputs of owk_kv8_attend only */ };
enum { OWK_KV8_INVALID = -1, OWK_KV8_HIP = -2 };

struct owk_kv8_cache {
    int device;
    int dtype;      /* type of the tails and of what is appended and read back: OWK_KV8_F16 or OWK_KV8_BF16 */
    int head_dim;   /* 64 or 128 */
    int n_heads;    /* key/value heads */
    int n_seqs;     /* sequences (tails) */
    int n_blocks;   /* blocks in the pool */
    int max_blocks; /* blocks a sequence can have: its capacity is 64 * max_blocks tokens */
    int8_t * k;       /* [n_blocks][n_heads][64][head_dim]  16-byte aligned, as all six */
    int8_t * v;       /* [n_blocks][n_heads][head_dim][64] */
    float * k_scale;  /* [n_blocks][n_heads] */
    float * v_scale;
    void * k_tail;    /* [n_seqs][n_heads][64][head_dim] */
    void * v_tail;    /* [n_seqs][n_heads][head_dim][64] */
    const int32_t * table; /* [n_seqs][max_blocks] block of the pool; NULL: sequence s owns s * max_blocks + i */
};

/* The entries of a call. Entry b works on sequence seq[b] (NULL: b), which holds lens[b] tokens before
 * the call's own, and brings count[b] tokens / query rows (NULL: max_new):
 *   off == NULL  they are rows 0 .. count-1 of entry b of a padded tensor (entry strides below)
 *   off != NULL  they are rows off[b] .. off[b+1]-1 of a joined tensor of `rows` rows (count is unused)
 * More than max_new are cut off. */
struct owk_kv8_batch {
    int n;
    int max_new;
    int64_t rows;         /* rows of the joined tensors; unused without off */
    const int32_t * lens; /* [n] */
    const int32_t * seq;  /* [n] or NULL */
    const int32_t * off;  /* [n+1] or NULL */
    const int32_t * count;/* [n] or NULL */
};

/* A tensor of rows: element strides of an entry (unused with off), a row and a head; head_dim elements
 * of a head lie together. Any strides and alignment of whole elements; 16-byte aligned rows and heads
 * are loaded and stored as vectors. */
struct owk_kv8_rows {
    void * data;
    int64_t entry, row, head;
};

/* Store the entries' tokens at positions lens[b] .. of their sequences. lens[b] has to be the number of
 * tokens stored so far, or a multiple of 64 below it (the tokens from there on are dropped). */
WHISPER_API int owk_kv8_append(const struct owk_kv8_cache * cache, const struct owk_kv8_batch * batch,
                               const struct owk_kv8_rows * k, const struct owk_kv8_rows * v, void * stream);

struct owk_kv8_attend_params {
    int n_q_heads;  /* a multiple of n_heads; query head h reads key/value head h / (n_q_heads / n_heads) */
    int causal;     /* 0: every row sees tokens [0, lens[b]), which are what the sequence holds (or a multiple of 64 below);
                       1: row i sees [0, lens[b] + i], the call's own tokens were appended before */
    int out_type;   /* type of out: the cache's, or OWK_KV8_F32 */
    int max_len;    /* no sequence holds more tokens than this (decides how the work is split; 0: the capacity) */
    float scale;    /* of the products of queries and keys; finite */
};

/* out = softmax(scale * q . k) . v for each row and query head; zeros for a row that sees nothing. Rows
 * behind an entry's own are left as they were. out may lie where q lies (the same type and strides); other
 * overlaps are not allowed.
 *
 * Scores, sums, maxima and the accumulators are f32, and a weight is divided by the sum of the weights as they
 * were rounded. What is multiplied has fewer bits, also where out is f32:
 *   calls of few rows   each query element to 2^-16 of its row's largest, each weight to 2^-16 of the largest of its
 *                       block of 64 tokens
 *   calls of many rows  weights to half precision (2^-11 of each, or 2^-15 of its block's largest if that is more); bf16
 *                       query elements below 2^-14 of their row's largest to 2^-25 of it
 *   tails, in both      queries, keys and values as they are; weights to half precision (f16), 2^-16 of each (bf16)
 * Which form a call takes follows from its sizes (rows, heads, entries, length), not from its data.
 *
 * A row whose query is not finite is NaN if it sees anything; so is a row that sees any of a block that is not finite, or
 * a tail token with a value that is not finite (a tail key that is not finite counts by its score). Hidden tokens and
 * blocks add nothing, whatever they hold. A row whose weighted values add up beyond the range of f32 may be infinite. */
WHISPER_API int owk_kv8_attend(const struct owk_kv8_cache * cache, const struct owk_kv8_batch * batch,
                               const struct owk_kv8_attend_params * params, const struct owk_kv8_rows * q,
                               const struct owk_kv8_rows * out, void * workspace, size_t workspace_bytes, void * stream);
/* bytes of workspace such a call needs (0: none; its contents do not matter); 0 for invalid arguments */
WHISPER_API size_t owk_kv8_attend_workspace(const struct owk_kv8_cache * cache, const struct owk_kv8_batch * batch,
                                            const struct owk_kv8_attend_params * params);

/* Tokens first[b] .. first[b] + max_tokens - 1 (first NULL: 0) of n sequences that hold lens[b] tokens, as
 * the cache's 16-bit type, [entry][token][head] with the given strides; zeros from lens[b] on. */
WHISPER_API int owk_kv8_read(const struct owk_kv8_cache * cache, int n, int max_tokens, const int32_t * lens,
                             const int32_t * seq, const int32_t * first, const struct owk_kv8_rows * k,
                             const struct owk_kv8_rows * v, void * stream);

/* test hook (host only: every pointer is host memory): what the kernels make of entry b -- out receives its
 * sequence or -1, the tokens held before, its own tokens, its first row -- and of block i of sequence seq:
 * the block of the pool, or -1 */
WHISPER_API void owk_debug_kv8_entry(const struct owk_kv8_cache * cache, const struct owk_kv8_batch * batch, int b,
                                     int64_t out[4]);
WHISPER_API int64_t owk_debug_kv8_page(const struct owk_kv8_cache * cache, int seq, int i);
/* test hook: owk_kv8_attend takes its many-row form for calls of more than `rows` rows a key/value head (0: by its own rule).
 * For the calling thread alone; workspaces that were asked for before are of the other form's size. */
WHISPER_API void owk_debug_kv8_set_many_rows(int rows);

/* what the calling thread's last failed call found wrong ("" if none failed) */
WHISPER_API const char * owk_kv8_error(void);

#ifdef __cplusplus
}
#endif

#endif /* OWK_KV8_H */
