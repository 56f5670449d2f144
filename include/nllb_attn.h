/*  nllb_attn.h -- C ABI of the B200 attention path for the MetalNLLB engine.
 *
 *  libnllb_attn.so replaces the three attention loops of the reference's C11
 *  engine with sm_100a kernels:
 *
 *    encoder self-attention prefill     encoder.c:166-205 (multi_head_self_attn_flash),
 *                                       and the declared single-head API
 *                                       attention_head / attention_head_flash
 *                                       (pico.h:85-92, tensor.c:255-332)
 *    decoder self-attention, KV cache   decoder.c:48-99   (decoder_self_attn_cached)
 *    cross-attention, encoder memory    decoder.c:103-152 (decoder_cross_attn_cached)
 *
 *  plus the beam reorder of the per-beam KV caches (main.c:462-488), which is
 *  an index permutation here instead of a copy of every cache.
 *
 *  Conventions
 *  - Every int-returning call returns an NLLB_ATTN_* status (0 = success).
 *  - Plain calls take DEVICE pointers (cudaMalloc'd) and only enqueue work on
 *    the context's stream; they return before the GPU finishes.  Call
 *    nllb_attn_sync() (or synchronise the stream) before reading outputs.
 *  - *_host calls take HOST pointers (pageable or pinned), copy inputs in,
 *    run, copy outputs back and return once the outputs are written, the way
 *    the reference's call sites use their stack and heap buffers.
 *  - fp32 in, fp32 out.  head_dim must be 64 (NLLB-200: 16 heads x 64).
 *    (nllb_attn_paged, _window, _cross_rows and _append also take 16-bit types
 *    and heads of 128; their rows lie at the strides of their arguments.)
 *  - Rows of q/k/v/out hold all heads, head h at columns [64h, 64h+64), as the
 *    reference's projections produce them (decoder.c:57-59, encoder.c:159-163).
 *  - One context belongs to one device and is used by one host thread at a
 *    time.  The reference calls decoder attention from one thread per beam
 *    (main.c:124-150); here one call covers all beams of all sentences.
 *  - No call falls back to a CPU implementation.  Without a usable sm_100
 *    device nllb_attn_create() fails with NLLB_ATTN_ENODEV.
 */
#ifndef NLLB_ATTN_H
#define NLLB_ATTN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define NLLB_ATTN_API __attribute__((visibility("default")))
#else
#define NLLB_ATTN_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes -------------------------------------------------------- */
#define NLLB_ATTN_OK        0
#define NLLB_ATTN_EINVAL    1  /* bad argument: NULL pointer, size < 1, head_dim != 64, misaligned */
#define NLLB_ATTN_ECAPACITY 2  /* size beyond the capacity the context was created with */
#define NLLB_ATTN_ECUDA     3  /* a CUDA runtime call failed (see nllb_attn_last_error) */
#define NLLB_ATTN_ETIMEOUT  4  /* a bounded device-side wait gave up; the call's outputs are invalid */
#define NLLB_ATTN_ENODEV    5  /* no CUDA device, or the device is not compute capability 10.x */
#define NLLB_ATTN_ESTATE    6  /* call order violated (e.g. cross-attention before its memory is set) */

typedef struct nllb_attn_ctx nllb_attn_ctx;

/* Capacities fixed at creation; device buffers are sized from them.
 * The reference fixes the same quantities at compile time (pico.h:11-22). */
typedef struct {
    int n_layers;       /* decoder layers with a KV cache and a memory (12) */
    int n_heads;        /* attention heads (16) */
    int head_dim;       /* must be 64 */
    int max_sentences;  /* sentence slots resident on the device (0: prefill only) */
    int n_beams;        /* beams per sentence: 1, 2, 4 or 8 (BEAM_SIZE, pico.h:97) */
    int max_tgt;        /* KV-cache positions per beam (MAX_GEN_LEN, pico.h:19) */
    int max_src;        /* encoder-memory rows per sentence (MAX_SEQ_LEN, pico.h:18) */
} nllb_attn_dims;

/* Create a context on `device` (CUDA ordinal).  Allocates the KV caches
 * [n_layers][max_sentences][n_heads][max_tgt][n_beams][64] (K and V), the
 * encoder memory [n_layers][max_sentences][n_heads][max_src][64] (K and V),
 * the beam history and a small split-K workspace, all zeroed.
 * Replaces the calloc of per-beam caches in main.c:297-302. */
NLLB_ATTN_API int  nllb_attn_create(int device, const nllb_attn_dims* dims, nllb_attn_ctx** out_ctx);
NLLB_ATTN_API void nllb_attn_destroy(nllb_attn_ctx* ctx);

/* Device bytes nllb_attn_create would allocate for `dims`. */
NLLB_ATTN_API size_t nllb_attn_device_bytes(const nllb_attn_dims* dims);

/* Use `stream` (a cudaStream_t) for all later work; NULL restores the
 * context's own stream. */
NLLB_ATTN_API int   nllb_attn_set_stream(nllb_attn_ctx* ctx, void* stream);
NLLB_ATTN_API void* nllb_attn_get_stream(nllb_attn_ctx* ctx);

/* Wait for all enqueued work, then read and clear the device error word
 * (set by a kernel whose bounded wait gave up).  Returns NLLB_ATTN_ETIMEOUT
 * in that case. */
NLLB_ATTN_API int nllb_attn_sync(nllb_attn_ctx* ctx);

/* Forget all sentences: beam histories reset to the identity. */
NLLB_ATTN_API int nllb_attn_reset(nllb_attn_ctx* ctx);

NLLB_ATTN_API const char* nllb_attn_strerror(int status);
/* Text of the last failure seen on the calling thread ("" if none). */
NLLB_ATTN_API const char* nllb_attn_last_error(void);

/* ---- encoder self-attention prefill -------------------------------------
 * Replaces encoder.c:166-205 and attention_head_flash (tensor.c:286-332):
 * for every (batch b, head h, query row i)
 *    s_j  = (q_i . k_j) * scale + mask_ij        (j < seq_len)
 *    out_i = sum_j softmax(s)_j v_j
 * Element (b,h,row,d) of q/k/v/out is at b*stride_batch + h*stride_head +
 * row*stride_row + d (elements).  Both the engine's head-interleaved rows
 * (stride_head = 64, stride_row = n_heads*64) and [B,H,S,64] tensors fit.
 * Keys j >= valid_len[b] are excluded (the reference expresses the same
 * padding as an additive -1e9 mask, tensor.c:309); valid_len may be NULL,
 * entries lie in [0, seq_len], and 0 gives the plain mean of V over all
 * seq_len keys, which is what the -1e9 mask yields when every key is
 * masked.  mask (may be NULL) is an additive
 * fp32 mask, row i of (b,h) at mask + b*mask_stride_batch +
 * h*mask_stride_head + i*seq_len.  Pointers and strides must keep every row
 * 16-byte aligned. */
typedef struct {
    const float* q;
    const float* k;
    const float* v;
    float*       out;
    int batch, n_heads, seq_len, head_dim;
    int64_t stride_batch, stride_head, stride_row;
    const int*   valid_len;
    const float* mask;
    int64_t mask_stride_batch, mask_stride_head;
    float scale;            /* the reference uses 1/sqrt(head_dim) = 0.125 */
} nllb_attn_prefill_args;

NLLB_ATTN_API int nllb_attn_prefill(nllb_attn_ctx* ctx, const nllb_attn_prefill_args* args);
/* Same, with every pointer in args a host pointer. */
NLLB_ATTN_API int nllb_attn_prefill_host(nllb_attn_ctx* ctx, const nllb_attn_prefill_args* args);

/* ---- decoder self-attention over the per-beam KV cache ------------------
 * Replaces decoder.c:64-96 for every beam of sentences [0, n_sentences):
 * writes k_new/v_new at position `step` of each beam's cache (decoder.c:64-69)
 * and attends q over positions 0..step of that beam's history
 * (decoder.c:71-96: scores * 1/sqrt(64), softmax, P.V).
 * q, k_new, v_new, out: [n_sentences][n_beams][n_heads*64].
 * step must be < max_tgt; all sentences advance together. */
NLLB_ATTN_API int nllb_attn_decode_self(nllb_attn_ctx* ctx, int layer, int step, int n_sentences,
                          const float* q, const float* k_new, const float* v_new,
                          float* out);
NLLB_ATTN_API int nllb_attn_decode_self_host(nllb_attn_ctx* ctx, int layer, int step, int n_sentences,
                               const float* q, const float* k_new, const float* v_new,
                               float* out);

/* Beam reorder, replacing the cache copies of main.c:462-488 (and the
 * bootstrap copies main.c:335-340, 384-392): new beam b of sentence s
 * continues the history of old beam parent[s*n_beams + b], for every layer.
 * Applies to positions already written; costs O(n_sentences*max_tgt) bytes,
 * independent of the cache size.  parent: [n_sentences][n_beams] int32.
 * The reorder takes effect for every later call on the context.  It is
 * applied lazily: when the next nllb_attn_decode_self covers exactly these
 * n_sentences and they are all of the context's max_sentences, that launch
 * reads each beam's rows through its parent and writes the composed history
 * itself (one launch per step instead of two); otherwise a reorder kernel
 * runs first.  So nllb_attn_reorder's device buffer `parent` must stay valid
 * and unchanged until the next nllb_attn_decode_self, nllb_attn_reorder,
 * nllb_attn_sync or nllb_attn_reset call on the context.
 * nllb_attn_reorder_host checks the parents on the host and returns once
 * they are copied (the caller may reuse its buffer at once). */
NLLB_ATTN_API int nllb_attn_reorder(nllb_attn_ctx* ctx, int n_sentences, const int* parent);
NLLB_ATTN_API int nllb_attn_reorder_host(nllb_attn_ctx* ctx, int n_sentences, const int* parent);

/* Test of the bounded device waits: the next self-attention launch on this
 * context (nllb_attn_decode_self or _host, 4 beams) waits for a cache chunk
 * that it never requests, with a budget of about 1 ms, so that the wait runs
 * out.  That launch writes no output and sets the device error word, which
 * the call (_host) or the next nllb_attn_sync reports as NLLB_ATTN_ETIMEOUT;
 * the context stays usable.  No counterpart in the reference. */
NLLB_ATTN_API int nllb_attn_test_expire_next_wait(nllb_attn_ctx* ctx);
/* The same for the next cross-attention launch (nllb_attn_cross or _host,
 * 4 beams): it waits ~1 ms for a memory chunk that it never requests, writes
 * no output, and the error is reported as above. */
NLLB_ATTN_API int nllb_attn_test_expire_next_cross_wait(nllb_attn_ctx* ctx);

/* ---- cross-attention over the shared encoder memory ---------------------
 * Stores one sentence's projected encoder keys/values for one layer
 * (what decoder.c:118-125 writes into the shared cache at step 0).
 * Row r, head h of k/v is at k + r*stride_row + h*stride_head (elements):
 * stride_head 64 / stride_row n_heads*64 for the engine's rows,
 * stride_head n_src*64 / stride_row 64 for [H][n_src][64] tensors. */
NLLB_ATTN_API int nllb_attn_set_memory(nllb_attn_ctx* ctx, int layer, int sentence, int n_src,
                         const float* k, const float* v,
                         int64_t stride_head, int64_t stride_row);
NLLB_ATTN_API int nllb_attn_set_memory_host(nllb_attn_ctx* ctx, int layer, int sentence, int n_src,
                              const float* k, const float* v,
                              int64_t stride_head, int64_t stride_row);

/* decoder.c:128-149 for every beam of sentences [0, n_sentences): each
 * beam's query attends all n_src memory rows of its sentence.  The memory
 * is read once per call for all beams.  q, out: [n_sentences][n_beams][n_heads*64]. */
NLLB_ATTN_API int nllb_attn_cross(nllb_attn_ctx* ctx, int layer, int n_sentences,
                    const float* q, float* out);
NLLB_ATTN_API int nllb_attn_cross_host(nllb_attn_ctx* ctx, int layer, int n_sentences,
                         const float* q, float* out);

/* ---- many query rows against keys of another length ----------------------
 * Calls for a decoder that draws its tokens (nllb_sample) or scores given
 * target rows (nllb_logprobs): a chunk of new tokens over a paged cache, over
 * all of it or through a sliding window, target rows over encoder states, and
 * new rows into the cache, turned by their positions.  No counterpart in the
 * reference, whose decoder moves one token at a time (decoder.c:48-152).
 *
 * Types: q, k, v and out are all fp32, all fp16 or all bf16.  Scores, softmax
 * sums and outputs are accumulated in fp32 and an output is rounded once.
 * The weights of 16-bit calls of several rows are rounded to the type before
 * their product with V, and their sums over n keys may come out up to n 2^-27
 * short (relative), over more than 32768 no more than over 32768: 2^-12, where
 * half a step of fp16 is 2^-11.  fp32 calls of many rows split q, k and v into
 * two fp16 parts, after a division by a power of two where sizes ask for it:
 * 22 bits down to 2^-17 of the largest value of a row of q or k, or of 128 rows
 * of v (a chunk's later tokens among them); below that an absolute 2^-39 of the
 * largest, or 2^-25 where the largest of 16 rows of q or k, or of the 128 of v,
 * lies in [2^-3, 65504).  Finite values below 2^100 are meant; scores have to
 * be finite in fp32.  At most 8 rows of a key head (max_q times the query heads
 * that share it; 16-bit types: 16) count as few.
 * All pointers are of the context's device.
 * n_heads is a multiple of n_kv_heads: query head h reads key head
 * h / (n_heads / n_kv_heads).  head_dim is 64 or 128.
 * Sequence s has q_len[s] query rows from row q_start[s] of q and out
 * (device arrays; q_len NULL: max_q rows each, q_start NULL: s * max_q).
 * Rows of q and out that belong to no sequence are neither read nor written.
 * Strides count elements; every row must start on 16 bytes (out may not
 * overlap an input, nor rows that the call writes one another).  max_q and max_kv bound the lengths: they size the
 * launch, larger lengths on the device are refused there.  A length, start
 * or page number outside its bound or buffer sets the device error word
 * (nllb_attn_sync then returns NLLB_ATTN_EINVAL): a sequence with a bad
 * length or start is left out, a key on a bad page is left out of the
 * attention.  The calls allocate nothing and may be captured into a graph. */
#define NLLB_F32  0
#define NLLB_F16  1
#define NLLB_BF16 2

/* A chunk of new tokens over a paged cache.  Slot r of page p, key head g is
 * at k_pages + p*k_stride_page + r*k_stride_slot + g*k_stride_head; key j of
 * sequence s lies in slot j % page_size of page
 * page_table[s*page_table_stride + j / page_size].  kv_len[s] counts the keys
 * with the chunk: new token i stands at position kv_len[s] - q_len[s] + i and
 *    out_i = sum_{j <= its position} softmax_j(scale * q_i . k_j) v_j.
 * With k_new and v_new (both or neither; rows as q's) the call also writes
 * the chunk's keys and values into their slots; without, they are there
 * already.  The slots written belong to one sequence each: a page that two
 * sequences of a call share may only hold keys from before both chunks.
 * Entries of page_table past a sequence's last page are not read.  A value
 * that is not finite in a chunk's keys or values may also reach the rows of
 * earlier tokens of the same chunk (a weight of 0 times it is no number). */
typedef struct {
    const void* q;
    const void* k_new;
    const void* v_new;
    void*       k_pages;
    void*       v_pages;
    void*       out;
    const int*  q_start;
    const int*  q_len;
    const int*  kv_len;
    const int*  page_table;
    int dtype, head_dim, n_heads, n_kv_heads;
    int n_seq, q_rows, max_q, max_kv;
    int n_pages, page_size, page_table_stride;
    float scale;
    int64_t q_stride_row, q_stride_head;
    int64_t out_stride_row, out_stride_head;
    int64_t k_new_stride_row, k_new_stride_head;
    int64_t v_new_stride_row, v_new_stride_head;
    int64_t k_stride_page, k_stride_slot, k_stride_head;
    int64_t v_stride_page, v_stride_slot, v_stride_head;
} nllb_attn_paged_args;

NLLB_ATTN_API int nllb_attn_paged(nllb_attn_ctx* ctx, const nllb_attn_paged_args* args);

/* The same where a token sees the last `window` positions, its own among them,
 * and the first `sinks` ones (of a running translation: the tokens that name the
 * languages), so that a cache need not grow with what was said:
 *    out_i = softmax over the keys j <= its position p with j > p - window or
 *    j < sinks.
 * Keys that no token of the call sees are not read, nor are the entries of
 * page_table that hold nothing else and no new token: their pages may be given
 * back, or be the same as later entries' (a ring), as long as no slot that the
 * call writes holds a key that a token of the call sees.  max_kv bounds kv_len,
 * the whole length.  What nllb_attn_paged says holds for the rest; a value that
 * is not finite, in a key or value that one token of the call sees, may also
 * reach the call's other tokens of its sequence. */
typedef struct {
    nllb_attn_paged_args cache;
    int window, sinks;      /* window >= 1, sinks >= 0 */
} nllb_attn_window_args;

NLLB_ATTN_API int nllb_attn_window(nllb_attn_ctx* ctx, const nllb_attn_window_args* args);

/* Target rows over encoder states of another length: every query row of
 * sequence s attends to its kv_len[s] key rows from row kv_start[s] of k and v
 * (kv_start NULL: s * max_kv), except those whose byte of key_mask (indexed
 * like the rows of k; NULL: none) is 0.  Hidden rows, and rows past the
 * lengths, are never read.  A sequence without a visible key gives zeros. */
typedef struct {
    const void* q;
    const void* k;
    const void* v;
    void*       out;
    const int*  q_start;
    const int*  q_len;
    const int*  kv_start;
    const int*  kv_len;
    const uint8_t* key_mask;
    int dtype, head_dim, n_heads, n_kv_heads;
    int n_seq, q_rows, kv_rows, max_q, max_kv;
    float scale;
    int64_t q_stride_row, q_stride_head;
    int64_t k_stride_row, k_stride_head;
    int64_t v_stride_row, v_stride_head;
    int64_t out_stride_row, out_stride_head;
} nllb_attn_cross_rows_args;

NLLB_ATTN_API int nllb_attn_cross_rows(nllb_attn_ctx* ctx, const nllb_attn_cross_rows_args* args);

/* New tokens into a paged cache without attention, queries and keys turned by
 * their positions on the way: what a decoder with rotary positions makes of its
 * projections before nllb_attn_paged or nllb_attn_window (called without k_new)
 * reads the cache.  Sequences, rows, lengths, pages, types and errors are those of
 * nllb_attn_paged: token i of sequence s, row q_start[s] + i, goes to position
 * kv_len[s] - q_len[s] + i.  A head's first rot_dim values (a multiple of 16;
 * 0: nothing is turned) are rot_dim / 2 pairs: value i with value
 * i + rot_dim / 2 (NLLB_ROT_HALVES), or 2i with 2i + 1 (NLLB_ROT_NEIGHBOURS).
 * Pair i of every query and key head becomes
 *    (a cos x - b sin x, b cos x + a sin x),  x = p * inv_freq[i],
 * with p the token's position, or position[row] where that is given; x is
 * taken in 64 bits.  Values are left as they are.  q and q_out (both or
 * neither) may be one buffer, turned in its place; otherwise outputs may not
 * overlap inputs, nor one another (refused where rows and pages have no gaps).  Rows that belong to no sequence are
 * neither read nor written, of page_table only the entries of written slots
 * are read; a token whose page number is bad is turned but not stored (nor are
 * its neighbours hurt), and the error word is set.  Nothing is allocated; the
 * call may be captured into a graph. */
#define NLLB_ROT_HALVES 0
#define NLLB_ROT_NEIGHBOURS 1
typedef struct {
    const void* q;
    void*       q_out;
    const void* k_new;
    const void* v_new;
    void*       k_pages;
    void*       v_pages;
    const int*  q_start;
    const int*  q_len;
    const int*  kv_len;
    const int*  page_table;
    const int*  position;
    const float* inv_freq;
    int dtype, head_dim, n_heads, n_kv_heads;
    int n_seq, q_rows, max_q, max_kv;
    int n_pages, page_size, page_table_stride;
    int rot_dim, rot_pairs;
    int64_t q_stride_row, q_stride_head;
    int64_t q_out_stride_row, q_out_stride_head;
    int64_t k_new_stride_row, k_new_stride_head;
    int64_t v_new_stride_row, v_new_stride_head;
    int64_t k_stride_page, k_stride_slot, k_stride_head;
    int64_t v_stride_page, v_stride_slot, v_stride_head;
} nllb_attn_append_args;

NLLB_ATTN_API int nllb_attn_append(nllb_attn_ctx* ctx, const nllb_attn_append_args* args);

/* Test of the bounded device waits: if the next nllb_attn_paged, _window or
 * _cross_rows of this context counts as many rows, a wait of its
 * launch runs out after about 1 ms; it writes no output (paged: the chunk's
 * keys and values may be written) and the next nllb_attn_sync returns
 * NLLB_ATTN_ETIMEOUT.  The context stays usable, and calls behind that next one
 * are as ever, also where it was refused, had no rows or counts few. */
NLLB_ATTN_API int nllb_attn_test_expire_next_rows_wait(nllb_attn_ctx* ctx);

/* ---- drop-ins for the declared single-head API (pico.h:85-92) -----------
 * Same signatures and meaning as the reference's attention_head
 * (tensor.c:255-282) and attention_head_flash (tensor.c:286-332): host
 * pointers, Q/K/V/out [seq_len][head_dim], optional additive mask
 * [seq_len][seq_len].  They run on the calling thread's own context (device
 * from $NLLB_ATTN_DEVICE, default 0), created on first use.  head_dim must be
 * 64.  attention_head also leaves the softmaxed score matrix [seq_len][seq_len]
 * in scores_buf, as the reference does (tensor.c:258-277).
 * They return void like the originals; a failure is printed to stderr and
 * reported by nllb_attn_last_status(). */
NLLB_ATTN_API void nllb_attention_head(const float* Q, const float* K, const float* V,
                         const float* mask, float* out, float* scores_buf,
                         int seq_len, int head_dim);
NLLB_ATTN_API void nllb_attention_head_flash(const float* Q, const float* K, const float* V,
                               const float* mask, float* out,
                               int seq_len, int head_dim);
NLLB_ATTN_API int  nllb_attn_last_status(void);

#ifdef __cplusplus
}
#endif
#endif /* NLLB_ATTN_H */
