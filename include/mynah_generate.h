/* mynah_generate.h — the generation loop over the resident decoder: the GPU
 * twin of the reference's mynah_slm_generate (src/generate.c:13-86), which
 * the CLI `run` command (cli/main.c:225-315) and the server's completion
 * handler (server/main.c:175-300) both drive.
 *
 * The loop is the reference's, step for step:
 *   - every prompt token but the last only fills the cache (the batched
 *     prefill, which leaves the same cache bits as one step per token), and
 *     each is shown to the sampler's accept hook;
 *   - then up to max_new steps: forward the current token, pick the next id,
 *     accept it, stop on any of the EOS ids (the EOS id counts as generated
 *     but is not passed to on_token), else pass it to on_token (non-zero
 *     stops), and feed it back;
 *   - a full context ends the loop (the ids so far stand).
 * The return value is the number of ids generated, or -1.
 *
 * Picking the next id:
 *   - sample == NULL: greedy on the device (src/sampler.c:122-129, first
 *     index of the largest logit), with the logits never leaving HBM; steps
 *     run as captured graphs, up to `chunk` per host round trip (0: 8), the
 *     first step alone so TTFT is one step. This is the reference's sampler
 *     at temp <= 0 with every penalty off; with penalties on, pass a
 *     device sampler or the reference's sampler as below.
 *   - sample != NULL: every step's logits are copied to a host buffer and
 *     sample(sampler, logits) picks (the reference's mynah_slm_sample, which
 *     may modify the logits in place, fits as is); accept(sampler, id), when
 *     set, is called where the reference calls mynah_slm_sampler_accept.
 *   - device_sampler != NULL (sample, accept and sampler are then unused):
 *     the reference's sampler on the device (below), inside the captured
 *     steps like greedy, so the logits never leave HBM; the prompt tokens
 *     and every generated id enter its window, and its rng advances once
 *     per sampled id, exactly as the reference's sampler object would.
 *
 * Detokenisation and the thinking channel (src/generate.c:38-77) stay with
 * the caller: on_token receives the id, and the reference's binding feeds
 * its own detokenizer and routes the think markers inside that callback.
 *
 * Timing follows src/timing.c:30-62 (CLOCK_MONOTONIC, host side): prefill_s
 * from the call to the end of the prompt, decode_s from there to the end,
 * ttft_s stamped at the first generated id (prefill plus that step).
 *
 * SPDX-License-Identifier: MIT */
#ifndef MYNAH_GENERATE_H
#define MYNAH_GENERATE_H

#include <stddef.h>
#include <stdint.h>

#include "mynah_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* src/generate.h:13-15 (mynah_slm_token_cb), without the text: non-zero
 * stops generation after this id. */
typedef int (*mynah_hip_token_fn)(void *ctx, uint32_t id);
/* src/sampler.h:40-43 (mynah_slm_sample, mynah_slm_sampler_accept). */
typedef uint32_t (*mynah_hip_sample_fn)(void *sampler, float *logits);
typedef void (*mynah_hip_accept_fn)(void *sampler, uint32_t id);

/* src/generate.h:18-45 (mynah_slm_gen_params) */
typedef struct {
    const uint32_t *prompt;
    size_t n_prompt;
    uint32_t max_new;
    const uint32_t *eos;            /* stop on any of these */
    size_t n_eos;
    mynah_hip_token_fn on_token;
    void *token_ctx;
    mynah_hip_sample_fn sample;     /* NULL: greedy on the device */
    mynah_hip_accept_fn accept;     /* optional */
    void *sampler;
    uint32_t chunk;                 /* device steps per round trip, 0 = 8 */
    struct mynah_hip_sampler *device_sampler; /* NULL: as above */
} mynah_hip_gen_params;

/* src/timing.h:14-28 (mynah_slm_timing), the fields the loop fills. */
typedef struct {
    double prefill_s, decode_s, ttft_s;
    uint32_t n_prompt, n_gen;
    int ttft_done;
} mynah_hip_timing;

/* ── the reference's sampler on the device ─────────────────────────────────
 * src/sampler.h:16-30 (mynah_slm_sampler_params), field for field. */
typedef struct {
    float temp;                     /* <= 0: greedy */
    uint32_t top_k;                 /* 0 = off (host sampler only when temp > 0) */
    float top_p, min_p;
    float repeat_penalty, freq_penalty, presence_penalty;
    uint32_t penalty_window;
    uint64_t seed;
} mynah_hip_sampler_params;

/* A sampler object like the reference's (src/sampler.c:16-25): parameters,
 * splitmix64 state and penalty window, kept in device memory. Every id it
 * returns is the one mynah_slm_sample returns for the same logits and
 * history (the same penalties, f32 exponentials, double sum, f32
 * probabilities, candidate order, draw and walk). It takes what the
 * reference's defaults use: with temp > 0, 1 <= top_k <= 128 (and below the
 * vocabulary; the reference's top_k = 0 sorts the whole vocabulary, which
 * this sampler does not), a penalty window of at most 4096; otherwise
 * mynah_hip_sampler_new returns NULL (mynah_hip_last_error says why) and
 * the caller keeps the reference's sampler on the host. */
typedef struct mynah_hip_sampler mynah_hip_sampler;

/* src/sampler.c:48-64 (mynah_slm_sampler_new); seed 0 takes the same
 * fixed default state. */
mynah_hip_sampler *mynah_hip_sampler_new(const mynah_hip_sampler_params *p, uint32_t vocab);
/* src/sampler.c:66-71 (mynah_slm_sampler_free). */
void mynah_hip_sampler_free(mynah_hip_sampler *s);
/* src/sampler.c:73-78 (mynah_slm_sampler_accept). 0, or -1. */
int mynah_hip_sampler_accept(mynah_hip_sampler *s, uint32_t token);
/* src/sampler.c:116-187 (mynah_slm_sample) over host logits, modified in
 * place like the reference's (the penalties): *id is the picked token. The
 * generation loop samples on the device without this host copy. 0, or -1. */
int mynah_hip_sample(mynah_hip_sampler *s, float *logits, uint32_t *id);

/* ── rules on a batch's logits, ahead of any choice ───────────────────────────
 * No reference counterpart for a batch (its sampler penalises one sequence's logits,
 * src/sampler.c:72-94). For every row r and token i, in 32 bits, in this order:
 *   penalties  where i occurs c > 0 times in the row's history hist[hist_start[r]] ..
 *              hist[hist_start[r + 1] - 1]:
 *                l = l > 0 ? l / repeat[r] : l * repeat[r]
 *                l = l - freq[r] * c
 *                l = l - presence[r]
 *              one history for all three (where only some of them shall count a token,
 *              two calls, the first to f32, the second in place there);
 *              MYNAH_PENALTY_ONCE: once for the token; MYNAH_PENALTY_EACH: c times over,
 *              as the sampler above does for its window (the same bits); NULL arrays
 *              stand for 1, 0 and 0
 *   biases     l = l + bias[k] where bias_id[k] = i, bias_start[r] <= k <
 *              bias_start[r + 1]; of several such k the last
 *   grammars   -inf unless bit i % 32 of allowed[m][i / 32] is set, m = mask_row[r]
 *              (NULL: r); a row with m outside [0, n_masks) has none
 * rounded to out_type once. Ids outside [0, vocab) count for nothing. hist, bias_id and
 * allowed may be NULL: no such rule. All pointers are device pointers and everything
 * but the sizes is read there, so a captured call follows it; calls are asynchronous
 * on `stream` and allocate nothing. Starts rise and are 64-bit counts, each row's own
 * lists shorter than 2^32 - 1. Types are ggml's ids F32 = 0, F16 = 1, BF16 = 30;
 * strides count elements; y may be x with the same type and stride, otherwise they do
 * not overlap. mask_words >= ceil(vocab / 32); vocab < 2^31; elements on their own
 * size. 0, or -1 with the reason in
 * mynah_hip_last_error(). */
enum { MYNAH_PENALTY_ONCE = 0, MYNAH_PENALTY_EACH = 1 };
typedef struct {
    int type, out_type;
    uint32_t n_rows, vocab;
    const void *x;
    size_t x_stride;
    void *y;
    size_t y_stride;
    const int32_t *hist;
    const int64_t *hist_start;                  /* [n_rows + 1] */
    const float *repeat, *freq, *presence;      /* [n_rows] */
    int penalty;
    const int32_t *bias_id;
    const float *bias;
    const int64_t *bias_start;                  /* [n_rows + 1] */
    const uint32_t *allowed;                    /* [n_masks][mask_words] */
    const int32_t *mask_row;                    /* [n_rows] */
    uint32_t mask_words, n_masks;
} mynah_logits;

int mynah_hip_logits_dev(const mynah_logits *a, void *stream);

/* src/generate.h:47-52 (mynah_slm_generate). t may be NULL. */
long mynah_hip_qwen3_generate_tokens(mynah_qwen3 *s, const mynah_hip_gen_params *p,
                                     mynah_hip_timing *t);

#ifdef __cplusplus
}
#endif
#endif
