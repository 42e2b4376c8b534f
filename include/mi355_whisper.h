/*
 * mi355_whisper.h — entry points of libmi355_whisper.so beyond the whisper.h-compatible set.
 *
 * These have no counterpart in whisper.h; they exist for (a) choosing the arithmetic mode at load
 * time, (b) the stage-level parity tests (each stage of the path that whisper_full runs as one call at
 * /root/reference/src/whisper-utils/whisper-processing.cpp:218-219 can be run and read back on its own)
 * and (c) measurement.  All pointers are plain host pointers unless a name says `_device`.
 * Every function returns 0 on success and a negative code on failure; none throws.
 */
#ifndef MI355_WHISPER_H
#define MI355_WHISPER_H

#include "whisper.h"

#ifdef __cplusplus
extern "C" {
#endif

enum mw_precision {
    MW_PRECISION_BF16 = 0, /* bf16 weights / MFMA operands / KV caches, fp32 accumulate + residual stream */
    MW_PRECISION_FP32 = 1, /* exact fp32 everywhere (f32 MFMA): the bit-exact-token mode for tiny/base */
    MW_PRECISION_FP8 = 2,  /* MW_PRECISION_BF16 with the decoder's projection matrices and the logits matrix quantised to OCP
                              e4m3 at load (one power-of-two scale per output row) and streamed as bytes by the decode-step
                              kernels (bf16 activations, fp32 accumulate); the encoder keeps bf16 weights */
    MW_PRECISION_FP8_MX = 3 /* MW_PRECISION_FP8 and, in the encoder, the Q|K|V, attention-output, fc1 and fc2 products of every block and the cross K / V projections in MX-fp8 on
                              the fp8 matrix cores: weights AND activations as e4m3 with one power-of-two scale per block of
                              32 along k (OCP microscaling; scale = the smallest power of two that brings the block under
                              448, round to nearest even).  Needs n_audio_state % 256 == 0 (base, small, medium, large) */
};

/* Same as whisper_init_from_file_with_params (whisper-processing.cpp:112) with the arithmetic mode made
   explicit.  whisper_init_* use MW_PRECISION_BF16 unless the environment variable
   MI355_WHISPER_PRECISION is "fp32", "fp8" or "fp8mx". */
struct whisper_context *mw_init_from_file(const char *path_model, int gpu_device, int precision);
struct whisper_context *mw_init_from_buffer(const void *buffer, size_t size, int gpu_device, int precision);
/* A further context (one more audio stream / OBS source) on src's GPU that SHARES src's HBM-resident weights: nothing is
   parsed or uploaded again; KV caches, workspace, HIP stream and whisper_full state are its own, so the two contexts run
   concurrently from different threads.  The weights are freed with the last context that uses them (either may be freed
   first).  whisper_init_from_file_with_params (whisper-processing.cpp:112) does this by itself when the same file
   (path, size, mtime) is already resident on the same device in the same precision — one upload per GPU however many
   filter instances load the model — unless MI355_WHISPER_NO_SHARED_WEIGHTS is set.  whisper.cpp's counterpart is
   whisper_init_state, which LocalVocal does not call (one whisper_context per filter, whisper-utils.cpp:27-51). */
struct whisper_context *mw_init_shared(struct whisper_context *src);

/* model facts: n_vocab,n_audio_ctx,n_audio_state,n_audio_head,n_audio_layer,n_text_ctx,n_text_state,
   n_text_head,n_text_layer,n_mels,ftype */
int mw_hparams(struct whisper_context *ctx, int32_t out[11]);

/* ---- stage-level entry points (same stages whisper_full chains) ---- */
/* log-mel of host PCM; result stays in HBM */
int mw_pcm_to_mel(struct whisper_context *ctx, const float *samples, int n_samples);
/* same, PCM already resident in HBM (the timed region of bench.py starts here) */
int mw_pcm_to_mel_device(struct whisper_context *ctx, const float *samples_device, int n_samples);
/* The same log-mel for callers that cannot allocate (tight serving loops, harnesses that forbid hipMalloc, code that
   must not disturb an allocator while another thread captures a HIP graph).  The call itself cannot be captured: it
   launches on the context's own stream and synchronises that stream before it returns.  No counterpart in the reference.  Calls no hipMalloc / hipFree / allocating routine: the
   intermediate rows and the global-maximum word live in a static __device__ array of the library (1.54 MB per GPU, held
   until the process ends).  Input and output are the caller's device buffers: samples_device[n_samples] ->
   mel_out_device[n_len][n_mel] fp32, frame-major (the engine's HBM layout, the transpose of mw_get_mel's),
   n_len = (n_samples + 480000) / 160 written to *n_len_out.  Limits: n_samples <= 480640 (one 30 s window plus
   LocalVocal's margins), mel_out_floats >= n_len * n_mel; beyond them the call fails (-100, mw_last_error says why).
   The context's own mel state is left untouched.  Every call on one GPU shares that GPU's array: calls that overlap on
   one GPU race (the call synchronises the context's stream before it returns). */
int mw_pcm_to_mel_noalloc(struct whisper_context *ctx, const float *samples_device, int n_samples, float *mel_out_device,
                          size_t mel_out_floats, int *n_len_out);
int mw_mel_n_len(struct whisper_context *ctx);
/* MX-fp8 stages of MW_PRECISION_FP8_MX on host arrays (parity entry points; the encoder chains the same kernels inside
   whisper_full, whisper-processing.cpp:218-219).  epilogue: 0 = bf16 rows (+ bias), 1 = fp32 rows + bias + residual R,
   2 = GELU(+ bias) re-quantised to MX-fp8 (returned decoded).  A [M][K] and W [N][K] are quantised by the library's kernels
   (W from its bf16 rounding, as the loader does) and handed back decoded when the pointers are given; C_out is [M][N]
   fp32.  K % 128 == 0, N % 256 == 0. */
int mw_mx_gemm(int device, const float *A, int M, int K, const float *W, int N, const float *bias, const float *R, int epilogue,
               float *C_out, float *A_decoded, float *W_decoded);
/* LayerNorm (ggml_norm + weight, bias) whose rows leave as MX-fp8 (returned decoded) and, optionally, as bf16; d % 256 == 0 */
int mw_mx_layernorm(int device, const float *x, const float *w, const float *b, int rows, int d, float *out_decoded, float *out_bf16);
/* whisper_full (whisper-processing.cpp:218-219) with the PCM already resident in HBM on the context's device */
int mw_full_device(struct whisper_context *ctx, struct whisper_full_params params, const float *samples_device,
                   int n_samples);
/* out[n_mel][n_len] (whisper.cpp layout) */
int mw_get_mel(struct whisper_context *ctx, float *out);
/* encoder + cross-K/V for the 30 s window starting at mel frame `seek` */
int mw_encode(struct whisper_context *ctx, int seek, int audio_ctx);
/* out[n_ctx][n_audio_state] fp32 */
int mw_get_encoder_out(struct whisper_context *ctx, float *out);
/* out[n_ctx][n_text_state] fp32: cross-attention keys (pre-scaled by dh^-1/4) or values of one layer */
int mw_get_cross_kv(struct whisper_context *ctx, int layer, int is_v, float *out);
/* decode n tokens of sequence `seq` at positions n_past..n_past+n-1; keeps logits of the last
   min(n, 32) tokens */
int mw_decode(struct whisper_context *ctx, const whisper_token *tokens, int n, int n_past, int seq);
/* ONE decode step over n rows of different sequences (the shape of a beam step: n <= 32 rows, row i = token tokens[i] of
   sequence seq[i] at position pos[i]); keeps the logits of every row.  For teacher-forced parity tests. */
int mw_decode_rows(struct whisper_context *ctx, const whisper_token *tokens, const int *pos, const int *seq, int n);
/* out[rows][n_vocab]; rows = min(n, 32) of the last mw_decode / mw_decode_rows */
int mw_get_logits(struct whisper_context *ctx, float *out);
/* forget every cached key/value (start of a new prompt) */
int mw_kv_clear(struct whisper_context *ctx);
/* logits rules + sampler on one caller-supplied logits row (whisper_process_logits + samplers).
   history: tokens sampled so far.  n_draws = 0: greedy arg-max, else inverse-CDF draws with u[].
   Any of the three [n_vocab] outputs may be null.  tok_out gets max(1, n_draws) records. */
int mw_process_logits(struct whisper_context *ctx, const struct whisper_full_params *params, float temperature,
                      const float *logits_in, const whisper_token *history, int n_history, int has_ts, int seek_delta,
                      int n_draws, const double *u, float *logits_out, float *logprobs_out, float *probs_out,
                      whisper_token_data *tok_out);

/* ---- decoder operators on device memory ----
   A key / value cache in pages that any number of sequences share, the attention that reads it and a sampler, for callers
   that drive a decoder of their own beside Whisper's.  Unlike the entry points above these take DEVICE pointers and a HIP
   stream, launch on that stream of GPU `device` and return without waiting; the caller's current device is restored.  They
   allocate nothing, keep nothing between calls (the workspace is the caller's, its contents need no initialisation; two
   calls that may overlap need two) and may be captured into a graph; what a captured call reads from device memory (lengths,
   block tables, sampler settings) may change between replays.  The structures themselves are host memory, read before the
   call returns.  0: launched; -1: a null or inconsistent argument, -100: refused or failed, mw_last_error says why.

   The cache.  Row `offset` of page `page` of head `h` is the head_dim consecutive elements at
   page * page_stride + h * head_stride + offset * row_stride of k and v, its scales the floats at the same place of
   k_scale and v_scale with the scale strides.  Any order of pages, heads and rows is allowed; rows and scales that are written,
   here and in the results below, may not overlap (strides smaller than a row are refused).  head_dim is 64 or 128,
   page_size a power of two up to 32768, strides multiples of 16 bytes and bases 16-byte aligned.  Element types:
     MW_ELEM_BF16  no scales
     MW_ELEM_E4M3  OCP e4m3 codes; scale = the smallest power of two >= 2^-126 with max|x| <= 448 scale
     MW_ELEM_INT8  codes -127 .. 127; scale = max|x| * (1 / 127 rounded to fp32), at least 2^-126
   one fp32 scale per row and head, code = round to nearest even (x / scale).  A row of an 8-bit cache that holds an
   infinity or a NaN is kept as scale NaN and codes 0: it reads back as NaN. */
enum mw_elem { MW_ELEM_F32 = 0, MW_ELEM_BF16 = 1, MW_ELEM_E4M3 = 2, MW_ELEM_INT8 = 3 };
struct mw_kv_cache {
    void *k, *v;
    float *k_scale, *v_scale; /* null for MW_ELEM_BF16 */
    int32_t dtype;            /* enum mw_elem */
    int32_t n_pages, page_size, n_kv_heads, head_dim;
    int64_t page_stride, head_stride, row_stride;                   /* elements */
    int64_t scale_page_stride, scale_head_stride, scale_row_stride; /* floats */
};
/* One row per token of n_seqs sequences, back to back: sequence b owns rows cu_rows[b] .. cu_rows[b + 1] - 1 and its last row
   is the token at position kv_len[b] - 1.  Position p of sequence b lives in page block_table[b * table_stride + p / page_size],
   row p % page_size.  An entry outside 0 .. n_pages - 1 (a page not there yet, or given back) and positions behind
   table_cols pages hold nothing: they are not written, read back as zeros and are invisible to the attention, as are
   positions below zero (a sequence with more rows than kv_len).  Rows behind the last sequence are left as they are.
   Sequences may be empty, and may share pages; a slot that two rows of one write name holds undefined values afterwards. */
struct mw_kv_batch {
    int32_t n_seqs, n_rows;
    const int32_t *cu_rows;     /* [n_seqs + 1], not decreasing */
    const int32_t *kv_len;      /* [n_seqs] tokens of the sequence, the batch's rows included */
    const int32_t *block_table; /* [n_seqs][table_cols] */
    int64_t table_stride;
    int32_t table_cols;
    int32_t max_rows, max_kv;   /* what cu_rows and kv_len are expected to reach: used to shape the launch, never for what is computed */
};
/* rows of keys and values (dtype MW_ELEM_F32 or MW_ELEM_BF16; head h of row t at t * row_stride + h * head_stride elements, strides
   and bases 16-byte aligned) -> the pages */
int mw_kv_write_device(int device, void *stream, const struct mw_kv_cache *cache, const struct mw_kv_batch *batch, int dtype,
                       const void *k, const void *v, int64_t row_stride, int64_t head_stride);
/* the pages' contents at the batch's rows -> k, v (layout as above): the fp32 product code * scale, rounded to dtype (the bits of
   tensor operations; of an int8 row in bf16 one element in 10^5 is a last place beside the exact product's rounding) */
int mw_kv_read_device(int device, void *stream, const struct mw_kv_cache *cache, const struct mw_kv_batch *batch, int dtype,
                      void *k, void *v, int64_t row_stride, int64_t head_stride);
/* out[t][h] = sum_j softmax_j(scale q[t][h] . k_j) v_j over the keys j of the row's sequence that its token sees: those at its
   position p and before it; with window > 0 only j > p - window and the first `sinks` positions.  Query head h reads key /
   value head h / (n_heads / n_kv_heads).  q and out: bf16, head h of row t at t * stride + h * head_stride, 16-byte aligned.
   Scores, softmax and sums in fp32; the probabilities are rounded to bf16 for the product with v, in calls of few rows a sequence
   (single tokens, drafts) and over int8 caches with the rounding's residue.  A row that sees nothing, or only scores of -infinity,
   is zero.  Invisible keys and values are never used, whatever they hold.  scale > 0, finite.  workspace: at least
   mw_kv_attend_workspace bytes for the same device, cache, batch, n_heads, window and sinks (may be 0 bytes), 16-byte aligned. */
size_t mw_kv_attend_workspace(int device, const struct mw_kv_cache *cache, const struct mw_kv_batch *batch, int n_heads, int window,
                              int sinks);
int mw_kv_attend_device(int device, void *stream, const struct mw_kv_cache *cache, const struct mw_kv_batch *batch, int n_heads,
                        const void *q, int64_t q_row_stride, int64_t q_head_stride, void *out, int64_t out_row_stride,
                        int64_t out_head_stride, float scale, int window, int sinks, void *workspace, size_t workspace_bytes);
/* One token per row of logits (MW_ELEM_F32 or MW_ELEM_BF16, [n_rows] rows row_stride elements apart).  x = logit / temperature[row];
   the tokens in the order (x falling, index rising); top_k keeps that many of them; top_p, of those, the fewest that hold
   at least top_p of their probability (counted in 2^-43 of the likeliest token's); min_p, of those, the ones at least min_p times
   as likely as the likeliest; the token is the first in the order of the index whose cumulated probability reaches u[row]
   (0 <= u < 1) of what is kept.
   temperature <= 0: the first largest logit.  top_k <= 0, top_p >= 1 and min_p <= 0 keep all; the likeliest token is always
   kept.  The settings are device arrays [n_rows], each may be null (temperature 1, nothing dropped).  logprobs (may be null)
   gets log softmax(x) at the token over ALL tokens (as whisper_token_data.plog; temperature <= 0: x = logit).
   -infinity marks a suppressed token.  A row with a NaN, a +infinity or nothing but -infinity, or whose temperature, u, top_p or
   min_p is not a number, gives token -1 and logprob NaN.  Results do not depend on n_rows or on the other rows.
   n_vocab <= 1048576. */
int mw_sample_device(int device, void *stream, const void *logits, int dtype, int n_rows, int n_vocab, int64_t row_stride,
                     const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p, const double *u,
                     int32_t *ids, float *logprobs);

/* ---- measurement ---- */
struct mw_timings {
    double mel_ms, encode_ms, decode_ms, sample_ms, total_ms; /* host wall clock, cumulative */
    int n_encode, n_decode, n_sample;
};
int mw_get_timings(struct whisper_context *ctx, struct mw_timings *out);
int mw_reset_timings(struct whisper_context *ctx);
/* the HIP stream every kernel of this context is launched on (for HIP-event timing by the caller) */
void *mw_stream(struct whisper_context *ctx);
int mw_synchronize(struct whisper_context *ctx);
/* Benchmark-only: with n > 0, EOT is suppressed and no decoder may complete before n sampled tokens
   (synthetic random weights otherwise end a window after a handful of tokens).  0 restores normal
   behaviour.  See DESIGN.md "forced decode length". */
int mw_set_force_decode_steps(struct whisper_context *ctx, int n);
/* Counters of the batcher that runs the decode steps of every context sharing ctx's weights on its GPU:
   out = {batched steps run, activation rows in them, decode requests served, encoder passes run, 30 s windows in them}.
   rows / steps > rows per request means rows of different streams really shared weight passes; windows / passes > 1 the
   same for the encoder.  Returns 1 (and zeros) when ctx does not use the batcher
   (fp32 mode, widths without tile kernels).  No counterpart in the reference. */
int mw_hub_stats(struct whisper_context *ctx, unsigned long long out[5]);
/* Measurement-only: every launch of kernel class `step_class` (MW_STEP_*, -1: off) inside the replayed decode step is
   issued twice (the second writes a scratch output where the kernel updates in place), so that
   (time with - time without) / launches is the class's cost INSIDE graph replay; results are unchanged.  No
   counterpart in the reference. */
int mw_set_duplicate_class(struct whisper_context *ctx, int step_class);
/* micro-benchmarks of single kernels on device-resident synthetic operands (bench.py roofline legs):
   run `iters` launches of the decode step's weight-streaming projections for `rows` activation rows and
   return the average milliseconds per launch measured with HIP events on the context's stream. */
int mw_bench_decode_step(struct whisper_context *ctx, int rows, int n_past, int iters, float *ms_per_step);
int mw_bench_mel(struct whisper_context *ctx, int n_samples, int iters, float *ms_per_call);
int mw_bench_encode(struct whisper_context *ctx, int iters, float *ms_per_call);

/* Live timing of ONE kernel class of the decode step (the projections of dec.hip / mega.hip and the two
   attention kernels): between begin and end every launch of that class on the context's stream is bracketed
   by HIP events (the step then runs launch by launch, not as a captured graph); end returns the launch count
   and the summed elapsed time.  Classes: */
enum mw_gemv_class {
    MW_GEMV_QKV = 0, MW_GEMV_ATTN_OUT = 1, MW_GEMV_CROSS_Q = 2, MW_GEMV_FC1 = 3, MW_GEMV_FC2 = 4, MW_GEMV_LOGITS = 5,
    MW_STEP_SELF_ATTN = 6, MW_STEP_CROSS_ATTN = 7
};
int mw_profile_begin(struct whisper_context *ctx, int gemv_class, int max_launches);
int mw_profile_end(struct whisper_context *ctx, int *n_launches, float *total_ms);

const char *mw_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
