/*
 * aero_cuda_pages — a paged key/value cache on one B200, the attention that reads
 * it, and the adjustment of a batch's logits, plain C ABI (same library as
 * aero_cuda_moe.h).
 *
 * A cache holds n_page pages of page_size positions for every layer: K and V as
 * (n_layer, n_page, n_head_kv, page_size, head_dim) f16 or bf16. Its books are
 * three int32 device arrays:
 *   table  (n_seq, max_pages)  table[s][i] = the page of positions
 *                              [i * page_size, (i + 1) * page_size) of sequence s, or -1
 *   length (n_seq)             positions that sequence s holds
 *   refs   (n_page)            sequences that hold the page; 0: free
 * The pages a call takes are the lowest-numbered free ones, in the order of its
 * list. Sequences share full pages only (a fork copies the last page when it is
 * partly filled), so room taken by an extend is a sequence's own; an append to an earlier
 * position, in a page that a fork shares, is refused.
 *
 * All arrays are device memory; every call enqueues its work on the handle's stream
 * and returns (0, or -1 with the reason in aero_cuda_pages_last_error), does not
 * allocate and does not synchronise, so calls can be captured in a CUDA graph. What
 * the host cannot see (sequence numbers, lengths, free pages) is checked on the
 * device: a call that fails there changes nothing (append and copy skip the rows and
 * pages at fault, free the places of a sequence's row that hold no page) and records a
 * code for aero_cuda_pages_status. There is no CPU path.
 *
 * The calls of a cache share its books and its workspace, so their work runs one call after
 * another: set_stream orders calls on different streams; replays of graphs that hold calls
 * of the cache are ordered by their caller, among one another and with calls. A handle is not
 * for two threads at once.
 */
#ifndef AERO_CUDA_PAGES_H
#define AERO_CUDA_PAGES_H

#include <stdint.h>

#include "aero_cuda_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types (ggml numbering) */
#define AERO_CUDA_TYPE_F32 0
#define AERO_CUDA_TYPE_F16 1
#define AERO_CUDA_TYPE_BF16 30

/* aero_cuda_pages_status codes */
#define AERO_CUDA_PAGES_BAD_SEQ 1    /* a sequence number outside [0, n_seq), or listed twice */
#define AERO_CUDA_PAGES_NO_PAGES 2   /* more pages asked for than are free */
#define AERO_CUDA_PAGES_ROW_FULL 3   /* a sequence would pass max_pages, or a negative count */
#define AERO_CUDA_PAGES_NOT_EMPTY 4  /* a fork into a sequence that holds positions */
#define AERO_CUDA_PAGES_BAD_PAGE 5   /* a page number outside [0, n_page), or a position without a page */
#define AERO_CUDA_PAGES_BAD_ROWS 6   /* q_start does not ascend from 0 to T within the sequences' lengths */
#define AERO_CUDA_PAGES_WAIT 7       /* a bounded device wait gave up */
#define AERO_CUDA_PAGES_SHARED 8     /* an append into a page that several sequences hold */

typedef struct aero_cuda_pages_desc {
    int32_t n_layer, n_page;
    int32_t page_size; /* a power of two, 8 to 256 */
    int32_t n_head_kv;
    int32_t head_dim;  /* 64, 128, 192 or 256 */
    int32_t n_seq, max_pages;
    int32_t dtype;     /* AERO_CUDA_TYPE_F16 or AERO_CUDA_TYPE_BF16 */
    int32_t device, reserved;
} aero_cuda_pages_desc;

/* Allocate the pool (zeroed), the books (no pages held) and the workspace, charged
 * to the library's memory guard. NULL with the reason in err. */
void* aero_cuda_pages_open(const aero_cuda_pages_desc* desc, char* err, int errlen);
/* Device bytes that open allocates: the total, and by_class[0] pool / by_class[1]
 * books and workspace when by_class is not NULL. -1 for an invalid description. */
int64_t aero_cuda_pages_plan_bytes(const aero_cuda_pages_desc* desc, int64_t* by_class);
void aero_cuda_pages_close(void* cache);

/* Run on a cudaStream_t (NULL: the handle's own); work enqueued from now on waits
 * for what the handle has enqueued before, unless one of the two streams is being
 * captured (synchronise before the capture). A stream given here must exist until
 * another one is set or the cache is closed. 0 / -1. */
int aero_cuda_pages_set_stream(void* cache, void* stream);
/* Device addresses of the pool and the books (the books to be read: they are changed
 * by the calls below); any of them may be NULL. 0 / -1. */
int aero_cuda_pages_buffers(void* cache, void** k, void** v, int32_t** table, int32_t** length, int32_t** refs);
/* The first code recorded since the last status read (0: none), after
 * synchronising the handle's stream. */
int aero_cuda_pages_status(void* cache);
const char* aero_cuda_pages_last_error(void* cache);

/* Adopt books kept elsewhere (arrays of the same shapes). */
int aero_cuda_pages_set_tables(void* cache, const int32_t* table, const int32_t* length, const int32_t* refs);
/* Room for counts[i] more positions at the end of sequence seqs[i] (each listed
 * once): its length grows, pages are taken where it passes its last one. */
int aero_cuda_pages_extend(void* cache, const int32_t* seqs, const int32_t* counts, int n);
/* K and V rows of T tokens into `layer`: token t's head h at k + t * k_token + h *
 * k_head elements (head_dim contiguous values of the cache's type), to position
 * positions[t] < length of sequence seqs[t], in a page that no other sequence holds. */
int aero_cuda_pages_append(void* cache, int layer, const void* k, int64_t k_token, int64_t k_head, const void* v,
                           int64_t v_token, int64_t v_head, const int32_t* seqs, const int32_t* positions, int T);
/* Sequence children[i] (empty, listed once) becomes a copy of parents[i]: full
 * pages are shared, a partly filled last page is copied in every layer. */
int aero_cuda_pages_fork(void* cache, const int32_t* parents, const int32_t* children, int n);
/* The sequences (each listed once) give up their pages and become empty; pages that no
 * sequence holds any more are free. */
int aero_cuda_pages_free(void* cache, const int32_t* seqs, int n);
/* Pages dst[i] = src[i] in every layer (whole pages; no dst among the src or twice). */
int aero_cuda_pages_copy(void* cache, const int32_t* src, const int32_t* dst, int n);
/* Moves the live pages to the pool's front: with L live pages, the i-th free page
 * below L takes the contents of the i-th live page from L on, and the books follow. */
int aero_cuda_pages_compact(void* cache);

/* Attention over the pages of `layer`. q and out: T tokens of n_head heads, token t's
 * head h at t * q_token + h * q_head elements (head_dim contiguous values of the
 * cache's type); n_head a multiple of n_head_kv, at most 16 query heads per kv head.
 * q_start NULL: T == n, one new token of each of the n sequences seqs[i], its last
 * position. Else q_start (n + 1, ascending from 0 to T): tokens [q_start[i],
 * q_start[i + 1]) are the last positions of sequence seqs[i]. A sequence may be
 * listed more than once. A token at position p sees position j when j <= p and
 * (window == 0 or j > p - window or j < sinks); where none is visible (an empty
 * sequence) its output is 0. scores = scale * q . k with a positive, finite scale; softmax statistics and sums
 * are f32. The probabilities meet V as two values of the cache's type where tokens go one
 * by one (q_start NULL, at most 32 tokens, or fewer than two a sequence), so the output is as
 * exact as its own rounding; else as one value, which leaves it up to 1.4 times as far from
 * the exact one. A column of V that is not finite where a token sees it leaves that column
 * of the token's output not finite (infinite or no number), and nothing else. Values of
 * positions past a sequence's length are never used; a visible position without a page is recorded and
 * counts as a key and a value of zeros. */
int aero_cuda_pages_attend(void* cache, int layer, const void* q, int64_t q_token, int64_t q_head, int T, int n_head,
                           const int32_t* seqs, const int32_t* q_start, int n, float scale, int window, int sinks,
                           void* out, int64_t o_token, int64_t o_head);

/* Adjusts `rows` rows of `vocab` logits (type dtype, row stride ld elements) into out
 * (same type, row stride ld_out; may be logits itself), on `stream`. Per row r, with
 * its history's first n_history[r] token ids (row stride ld_history; at most ld_history count) of which the
 * first n_prompt[r] are the prompt:
 *   x = a token of the history? (x > 0 ? x / repetition[r] : x * repetition[r]) : x
 *   x -= frequency[r] * c + presence[r], c > 0 times in the history after the prompt
 *   x += the sum, in the list's order, of bias_value[i] for the entries i in
 *        [bias_start[r], bias_start[r + 1]) that name the token (bias_token[i])
 *   x = -infinity where bit (token % 32) of mask[r * ld_mask + token / 32] is 0
 * computed in f32. history, n_prompt (none), repetition (1), frequency (0), presence
 * (0), bias_start and mask may be NULL. ld_mask 0: one row of the mask for all rows.
 * Token ids outside [0, vocab) are passed over. bias_start ascends from 0 and its last entry is
 * the number of entries of bias_token and bias_value: this form cannot check it.
 * 0, or -1 with the reason in aero_cuda_moe_last_error(NULL). */
int aero_cuda_logits_adjust(const void* logits, int64_t ld, int dtype, int rows, int vocab, const int32_t* history,
                            int64_t ld_history, const int32_t* n_history, const int32_t* n_prompt,
                            const float* repetition, const float* frequency, const float* presence,
                            const int32_t* bias_start, const int32_t* bias_token, const float* bias_value,
                            const int32_t* mask, int64_t ld_mask, void* out, int64_t ld_out, void* stream);
/* The same for views: a history's rows hold history_width tokens each, of which at most that
 * many count, and lie ld_history apart, which may be less (rows that overlap) or 0 (one
 * history for all rows); bias_token and bias_value hold n_bias entries, and what bias_start
 * names outside them is passed over. */
int aero_cuda_logits_adjust_views(const void* logits, int64_t ld, int dtype, int rows, int vocab, const int32_t* history,
                                  int64_t ld_history, int history_width, const int32_t* n_history,
                                  const int32_t* n_prompt, const float* repetition, const float* frequency,
                                  const float* presence, const int32_t* bias_start, const int32_t* bias_token,
                                  const float* bias_value, int n_bias, const int32_t* mask, int64_t ld_mask,
                                  void* out, int64_t ld_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AERO_CUDA_PAGES_H */
