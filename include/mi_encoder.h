/*
 * mi_encoder.h -- C ABI of the MI355X-native text encoder (encode hot path).
 *
 * Replaces what runs underneath `SentenceTransformer(model).encode(batch)` in
 * the reference: `sidecar-search build -b 32` (reference Makefile:65,
 * README.md:60) and the query-time app (reference README.md:28) -- the Qwen2
 * decoder stack of stella_en_1.5B_v5, mean pooling, the Dense 1536->1024 module
 * and L2 normalisation.  Tokenisation stays on the host (the `tokenizers`
 * library); this ABI starts at token ids.  The Python mirror of the
 * sentence-transformers surface is abstracts-search_amd/sentence_transformers.py.
 *
 * Conventions: as in mi_ivfpq.h (int status, mi_enc_last_error(), opaque
 * handle, plain pointers, hipStream_t as void*).  Threading: mi_encoder_encode /
 * mi_encoder_hidden are safe to call from several host threads on one handle --
 * activations live in one workspace set per stream, leased for the duration of a
 * call (threads on distinct streams overlap on the GPU, threads sharing a stream
 * take turns); create / load_tensor / destroy are exclusive.  Token ids arrive PACKED:
 * ids[T] with cu_seqlens[nseq+1] (sequence i is ids[cu[i] .. cu[i+1])), host or
 * device pointers.  Weights are stored and multiplied in bf16 with f32
 * accumulation (MFMA); norms, softmax, pooling, Dense and the final
 * normalisation are f32.  Output is float32 [nseq][out_dim].
 */
#ifndef MI_ENCODER_H
#define MI_ENCODER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mi_encoder mi_encoder;

typedef struct mi_encoder_cfg {
    int32_t vocab_size;
    int32_t hidden;        /* 1536 */
    int32_t n_layers;      /* 28 */
    int32_t n_heads;       /* 12 */
    int32_t n_kv_heads;    /* 2 */
    int32_t head_dim;      /* 128 (64 also supported) */
    int32_t intermediate;  /* 8960 */
    float rms_eps;         /* 1e-6 */
    float rope_theta;      /* 1e6 */
    int32_t causal;        /* 0 = bidirectional (stella), 1 = causal (plain Qwen2) */
    int32_t dense_out;     /* 1024; 0 = no Dense module */
    int32_t dense_bias;    /* 1 */
    int32_t max_seq_len;   /* 512 */
} mi_encoder_cfg;

#define MI_DTYPE_F32 0
#define MI_DTYPE_BF16 1
#define MI_DTYPE_F16 2

const char *mi_enc_last_error(void);

/* SentenceTransformer(model_name_or_path, device=...) : allocate the model. */
int mi_encoder_create(const mi_encoder_cfg *cfg, int device, mi_encoder **out);
int mi_encoder_destroy(mi_encoder *h);

/* Load one parameter by its HF name without the "model." prefix, e.g.
 * "embed_tokens.weight", "layers.3.self_attn.q_proj.weight", "norm.weight",
 * "dense.weight", "dense.bias".  `data` is a host or device pointer to a dense
 * row-major tensor of `dtype`; it is converted to the internal layout. */
int mi_encoder_load_tensor(mi_encoder *h, const char *name, const void *data, int dtype,
                           const int64_t *shape, int ndim);
/* Number of parameters still missing (0 = ready to encode). */
int mi_encoder_missing(mi_encoder *h, int *count);
int mi_encoder_out_dim(mi_encoder *h, int *out);

/* SentenceTransformer.encode on token ids: Transformer -> mean Pooling ->
 * Dense -> optional L2 normalisation.  out: float32 [nseq][out_dim], host or
 * device.  total tokens = cu_seqlens[nseq]; each sequence 1..max_seq_len tokens. */
int mi_encoder_encode(mi_encoder *h, int nseq, const int32_t *ids, const int32_t *cu_seqlens,
                      int normalize, float *out, void *stream);

/* The same with the caller's un-sort folded in: embedding i is written to row out_rows[i] of `out` (a device pointer;
 * out_rows a host int32 [nseq]).  sentence-transformers sorts its inputs by length and restores the input order
 * afterwards; here the last kernel of the call does that.  With host `ids` / `cu_seqlens` both encode calls only ENQUEUE
 * work on `stream` and return (token ids travel through pinned staging slots): the host prepares the next pass while the
 * GPU runs this one. */
int mi_encoder_encode_rows(mi_encoder *h, int nseq, const int32_t *ids, const int32_t *cu_seqlens,
                           int normalize, float *out, const int32_t *out_rows, void *stream);

/* Prompts computed once (causal models: cfg.causal).  Texts are encoded behind an instruction prompt (reference README.md:28,
 * PROMPT_NAME); in a causal model the prompt's keys, values and hidden states do not depend on the text behind it.
 * mi_encoder_cache_prompt runs the n tokens of a prompt once and keeps their keys and values (in pages of the prompt cache
 * below: a prompt that begins as a cached one shares its full pages and runs only the tokens behind it) and what they add to
 * the mean pooling; it returns when the prompt is ready, on any stream.  mi_encoder_encode_prompted encodes texts behind it --
 * `ids` hold each text's own tokens alone, at least one, prompt and text together at most max_seq_len -- and gives what
 * mi_encoder_encode gives for prompt + text, to bf16 rounding.  out_rows as for mi_encoder_encode_rows, or NULL.  Loading a
 * weight drops all cached prompts. */
int mi_encoder_cache_prompt(mi_encoder *h, int n, const int32_t *ids, int32_t *prompt, void *stream);
int mi_encoder_drop_prompt(mi_encoder *h, int32_t prompt);
int mi_encoder_encode_prompted(mi_encoder *h, int32_t prompt, int nseq, const int32_t *ids, const int32_t *cu_seqlens,
                               int normalize, float *out, const int32_t *out_rows, void *stream);

/* Parity hook: the stack's last hidden state after the final norm,
 * float32 [T][hidden] (host or device), packed like ids. */
int mi_encoder_hidden(mi_encoder *h, int nseq, const int32_t *ids, const int32_t *cu_seqlens,
                      float *out, void *stream);

/* Timing of the dominant kernel family for the roofline: with profiling on, mi_encoder_encode() records the arguments of
 * its bf16 MFMA GEMM launches; mi_encoder_profile_read() re-issues exactly those launches back to back on the same
 * stream between two HIP events (one warm pass, three timed) and returns the device time of one pass (ms) and the FLOPs
 * the launches perform.  (The residual GEMMs add into the activations again: call it after the embeddings were read.) */
int mi_encoder_profile_enable(mi_encoder *h, int on);
int mi_encoder_profile_read(mi_encoder *h, double *gemm_ms, double *gemm_flops);

/* Test hook: process-wide counters of code paths the dispatcher takes on its own.  "tail_split_launches" = GEMM
 * launches whose last (partial) round of 256x256 tiles was split along K with f32 atomics into the residual stream;
 * "splitk_launches" = residual GEMMs whose every tile was split along K through the workspace (a few hundred to ~5 000
 * tokens); "reduce_norm_launches" = those whose reduction pass also wrote the next RMSNorm; "n192_launches" = residual
 * GEMMs run on 256 x 192 tiles; "prompted_passes" = forward passes behind a cached prompt (and those that cached one). */
int mi_enc_debug_counter(const char *name, int64_t *value);

/* The library reads its MI_* environment knobs (README.md lists them; each overrides a measured dispatch rule) ONCE, at the
 * first call that needs one, into a process-wide struct: no encode call path calls getenv.  This re-reads them -- for tests
 * and tools that switch a knob inside one process; not to be called while another thread is inside the library. */
int mi_encoder_reload_env(void);

/* Building block exposed for numerics tests: C[M][N] = A[M][K] . W[N][K]^T in
 * bf16 with f32 accumulation (device pointers; C bf16 row-major). */
int mi_enc_gemm_bf16(int device, int M, int N, int K, const void *A, const void *W, void *C,
                     void *stream);

/* ---------------------------------------------------------------------------------------------------------------------
 * Prompt cache: the keys and values of prompts, in pages, and the attention of texts that all stand behind one of them.
 *
 * In a causal model what a prompt's tokens compute does not depend on the text behind them, so a batch of prompted texts
 * needs the prompt's keys and values once.  A cache is a pool of n_pages pages of MI_PROMPT_PAGE tokens:
 *     pages [n_pages][n_layers][n_kv_heads][2: keys, values][MI_PROMPT_PAGE][head_dim]      (bf16 or f16)
 * An ENTRY is one prompt: a length and a page table.  Entries made by mi_prompt_cache_fork share their full pages (counted);
 * a page that is not full belongs to one entry alone, so extending an entry never changes another one.  Pages are handed out
 * lowest number first.
 *
 * Streams and threads: calls are safe from several host threads.  An entry belongs to the stream it was made on; work on
 * it from that stream is in order.  It may be read (attention, fork, copy) on other streams too, once the caller has ordered
 * them behind its writes (as with any device buffer); pages of entries that other streams read, or that a captured graph
 * reads, are given out again only after the device has been waited for.  mi_prompt_attention and mi_prompt_cache_write may be
 * captured into a graph (a replay uses the entry's length as it was at the capture; the entry must live, page moves by
 * mi_prompt_cache_compact are followed by replays that the caller orders behind them, a resize ends its use); the other calls
 * are refused on a stream that is being captured.  A stream that entries were made or freed on must have finished its work when
 * it is destroyed; on the per-thread handle, which is another stream in every thread, whatever is handed on is waited for.
 * A capture that another thread has open is left alone: no call here fails because of it or ends it, also where it waits (work on
 * the null stream excepted while a blocking stream is captured: HIP refuses it).
 * ------------------------------------------------------------------------------------------------------------------- */
#define MI_PROMPT_PAGE 64

typedef struct mi_prompt_cache mi_prompt_cache;

typedef struct mi_prompt_cache_cfg {
    int32_t n_layers;
    int32_t n_kv_heads;
    int32_t head_dim;      /* 64 or 128 */
    int32_t dtype;         /* MI_DTYPE_BF16 or MI_DTYPE_F16 */
    int32_t n_pages;
    int32_t max_entries;   /* entries alive at a time */
    int32_t max_tokens;    /* of one entry (0: all the pages hold) */
} mi_prompt_cache_cfg;

/* pages: device memory of the caller for the pool, 16-byte aligned, kept until destroy or resize; NULL: the cache allocates it. */
int mi_prompt_cache_create(const mi_prompt_cache_cfg *cfg, int device, void *pages, mi_prompt_cache **out);
int mi_prompt_cache_destroy(mi_prompt_cache *c);

int mi_prompt_cache_new(mi_prompt_cache *c, void *stream, int32_t *entry);
/* n more tokens at the end of an entry; their keys and values are undefined until mi_prompt_cache_write. */
int mi_prompt_cache_reserve(mi_prompt_cache *c, int32_t entry, int32_t n, void *stream);
/* keys and values of tokens start .. start + n - 1 of an entry, layers layer .. layer + n_layers - 1.  k and v: device, the
 * cache's dtype, element (l, t, h, d) at l * layer_stride + t * token_stride + h * head_stride + d (strides in elements,
 * multiples of 8; pointers 16-byte aligned).  Pages that other entries share are refused; reading by entries that shared one and are
 * freed is waited for.  (Reading of this entry on other streams is the caller's to order, as with any device buffer.) */
int mi_prompt_cache_write(mi_prompt_cache *c, int32_t entry, int32_t layer, int32_t n_layers, int32_t start, int32_t n,
                          const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3], void *stream);
/* n more tokens and their keys and values, all layers, in one launch: reserve and write. */
int mi_prompt_cache_extend(mi_prompt_cache *c, int32_t entry, int32_t n, const void *k, const int64_t k_strides[3], const void *v,
                           const int64_t v_strides[3], void *stream);
/* count new entries that begin as `entry` does: full pages are shared, the used rows of the last page are copied.  (Pages that a captured
 * mi_prompt_cache_write reaches, and all behind them, are copied too: a replay changes this entry alone.)  pages (may be NULL): the
 * number of each one's own last page, -1 where all pages are shared, -2 where several are its own. */
int mi_prompt_cache_fork(mi_prompt_cache *c, int32_t entry, int32_t count, int32_t *entries, int32_t *pages, void *stream);
/* one new entry with pages of its own throughout. */
int mi_prompt_cache_copy(mi_prompt_cache *c, int32_t entry, int32_t *copy, void *stream);
int mi_prompt_cache_free(mi_prompt_cache *c, int32_t n, const int32_t *entries, void *stream);
/* moves pages down until the used ones are 0 .. used - 1 (each page above goes to the lowest free place, lowest first). */
int mi_prompt_cache_compact(mi_prompt_cache *c, void *stream, int32_t *moved);
/* compacts into another pool of n_pages pages (`pages` as for create), which replaces the old one: larger or smaller.
 * Waits for the device. */
int mi_prompt_cache_resize(mi_prompt_cache *c, void *pages, int32_t n_pages, void *stream);
/* length in tokens, and the page numbers (up to `cap` of them into `table`, which may be NULL). */
int mi_prompt_cache_entry(mi_prompt_cache *c, int32_t entry, int32_t *length, int32_t *table, int32_t cap);
int mi_prompt_cache_used(mi_prompt_cache *c, int32_t *used_pages, int32_t *entries);

/* Attention of packed texts behind the prompt `entry`: token t of a text attends to every token of the prompt and to its
 * own text's keys,
 *     out[t] = sum_j softmax_j(scale * q[t] . key_j) value_j,
 * text i holding the query tokens cu_q[i] .. cu_q[i + 1] and the keys cu_k[i] .. cu_k[i + 1] (its newest; with more keys
 * than queries the first ones are the text's past: one query per text is the single-token form).  causal: query number a of
 * a text sees its keys 0 .. a + keys - queries; otherwise all of them.  A query that sees nothing (empty prompt, no key)
 * gets zeros.  n_heads is a multiple of the cache's n_kv_heads: head h reads key head h / (n_heads / n_kv_heads).
 * Masked keys and values may hold anything, infinities and NaN too.  Sums are f32; where a key head's rows (tokens x heads of its group)
 * are more than 256, a probability is rounded to the tensors' type before its product with V, up to there it is kept in two parts. */
typedef struct mi_prompt_attn {
    int32_t entry, layer;
    int32_t n_heads;
    int32_t n_tokens, n_keys, n_texts;
    const void *q;                   /* [n_tokens][n_heads][head_dim], the cache's dtype, device (as k, v, out) */
    const void *k, *v;               /* [n_keys][n_kv_heads][head_dim]; may be NULL with n_keys = 0 */
    void *out;                       /* [n_tokens][n_heads][head_dim] */
    int64_t q_token, q_head;         /* strides in elements, multiples of 8; head_dim is contiguous */
    int64_t k_token, k_head, v_token, v_head, o_token, o_head;   /* k_token, v_token: 0 .. 2^23 - 1; o_token, o_head: not 0 */
    const int32_t *cu_q, *cu_k;      /* device, [n_texts + 1], not decreasing; both NULL: one text */
    int32_t causal;
    float scale;                     /* 1 / sqrt(head_dim) as a rule */
    int32_t zero_rest;               /* tokens of no text, in front of the first and behind the last: 0 left as they are, 1 zeros */
    int32_t reserved;                /* 0 */
    void *workspace;                 /* device, 16-byte aligned, mi_prompt_attention_workspace bytes; not shared by calls that can overlap */
    int64_t workspace_bytes;
} mi_prompt_attn;
int mi_prompt_attention_workspace(mi_prompt_cache *c, const mi_prompt_attn *a, int64_t *bytes);
int mi_prompt_attention(mi_prompt_cache *c, const mi_prompt_attn *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MI_ENCODER_H */
