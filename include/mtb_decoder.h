/*
 * B200 strict speculative decoder: C ABI of the generate layer.
 *
 * This is the boundary the reference's generation layer would call instead of
 * its CPU path.  Each entry replaces one reference interface (paths relative
 * to the moss-transcribe.cpp project root):
 *
 *   mtb_model_load / mtb_model_free      ModelLoader::load (src/model_loader.cpp:21)
 *                                        + Qwen3Decoder::load weight part
 *                                        (src/qwen3_decoder.cpp:20-57)
 *   mtb_decoder_create / _free           Qwen3Decoder::load KV part
 *                                        (src/qwen3_decoder.cpp:59-85)
 *   mtb_decoder_run                      Qwen3Decoder::run / prefill / decode_one
 *                                        (src/qwen3_decoder.cpp:91-172)
 *   mtb_decoder_logits                   Qwen3Decoder::logits_from_hidden (:174-206)
 *   mtb_decoder_rewind / _past_len       CpuSpeculativeDecoder::rewind (src/cpu_speculative.cpp:22-24),
 *                                        Qwen3Decoder::past_len (src/qwen3_decoder.hpp:55)
 *   mtb_greedy_generate                  greedy_generate serial path (src/generate.cpp:235-326)
 *   mtb_spec_generate                    cpu_speculative_generate (src/cpu_speculative.cpp:68-147)
 *                                        with CpuSpeculativeHooks draft/committed
 *                                        (src/cpu_speculative.hpp:9-15)
 *   mtb_ngram_draft                      cpu_ngram_draft (src/cpu_speculative.cpp:27-38),
 *                                        evaluated by the device draft kernel
 *   mtb_greedy_choice                    cpu_greedy_choice (src/cpu_speculative.cpp:39-50),
 *                                        evaluated by the device choice kernel
 *   mtb_spec_step / _async, mtb_resume,  one verify step of the loop body
 *   mtb_spec_prime, mtb_spec_step_group_async, mtb_spec_run_group
 *                                        the same loop for several recordings at once
 *                                        (one launch per step; no reference counterpart:
 *                                        the reference decodes one recording at a time)
 *   mtb_snapshot_save / _restore         (src/cpu_speculative.cpp:100-137)
 *   mtb_audio_load / _encode / _free     AudioEncoder (src/audio_encoder.cpp:16-75): WhisperMel,
 *                                        WhisperEncoder, AudioAdaptor on the device
 *   mtb_rope_append, mtb_paged_attention, mtb_attention_weights, mtb_cache_evict,
 *   mtb_logits_process                   operators on a caller's own device memory
 *
 * Conventions: every function returns 0 on success or a negative code and
 * sets a per-object error string; no C++ exception crosses the boundary.  One
 * decoder is one CUDA device and one stream; decoders on different devices
 * may be driven from different host threads.  There is no CPU fallback: on a
 * host without a usable GPU, mtb_model_load fails with an error.
 */
#ifndef MTB_DECODER_H
#define MTB_DECODER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mtb_model mtb_model;
typedef struct mtb_decoder mtb_decoder;

/* KV cache element type; MTB_KV_DEFAULT reads MTB_KV_DTYPE ("f16" or "f32",
 * unset: f32, the reference's cache type, src/qwen3_decoder.cpp:67-75). */
enum { MTB_KV_DEFAULT = -1, MTB_KV_F32 = 0, MTB_KV_F16 = 1 };
enum { MTB_STOP_NONE = 0, MTB_STOP_EOS = 1, MTB_STOP_LIMIT = 2, MTB_STOP_ERROR = 3 };

/* Draft policy.  The reference policy is k_max 4, n-gram sizes 16..2
 * (src/cpu_speculative.cpp:29,104); penalty clamped to [1, 1.5] (:85-86).  A
 * NULL params pointer selects mtb_spec_params_from_env: that policy with the
 * penalty read from MTD_REPETITION_PENALTY, as the reference does, and k_max /
 * n_min / n_max overridable by MTB_SPEC_K / MTB_NGRAM_MIN / MTB_NGRAM_MAX. */
typedef struct mtb_spec_params {
    int32_t k_max;   /* proposals per step, 0..15 */
    int32_t n_min;   /* smallest n-gram size, >= 1 */
    int32_t n_max;   /* largest n-gram size */
    float penalty;   /* repetition penalty over the last 100 ids */
} mtb_spec_params;

/* Counters of the CPU_SPECULATIVE log line (src/cpu_speculative.cpp:140). */
typedef struct mtb_counters {
    int64_t target_calls, drafted_calls, proposed, accepted, target_input_tokens, rewinds;
    int32_t stop_reason; /* MTB_STOP_* */
    int32_t past_len;
} mtb_counters;

/* Mirrors CpuSpeculativeHooks::draft: write at most `budget` ids, return count. */
typedef int (*mtb_draft_fn)(void* user, const int32_t* ids, int n_ids, int budget, int32_t* out);
/* Mirrors CpuSpeculativeHooks::committed: after every commit. */
typedef void (*mtb_commit_fn)(void* user, const int32_t* ids, int n_ids, int past_len, int stopped);

int mtb_abi_version(void);
/* Whether moss_transcribe_capi_transcribe_pcm / _path can return a
 * transcript from this build: 0 (WAV decoding and the tokenizer are not part
 * of it; those calls return NULL with an error).  No counterpart in the
 * reference. */
int mtb_capi_can_transcribe(void);
/* The generate entries (mtb_spec_generate, mtb_spec_generate_ids,
 * mtb_greedy_generate) end by printing the reference's lines
 * (src/cpu_speculative.cpp:138-145) to stderr as "[mt I] <line>":
 * BENCH_GENERATION, CPU_PROFILE, CPU_SPECULATIVE and, with
 * MTD_TRACE_TOKENS=1 in the environment, BENCH_TOKEN_TRACE in chunks of 128
 * ids.  level 0 silences them, 1 (the default) prints them. */
void mtb_set_log_level(int level);
/* The same lines as text (no prefix, '\n' after each) for given results;
 * needs no GPU.  Returns the full length; out gets at most out_size - 1 bytes
 * and a terminating 0. */
int mtb_format_generation_log(const int32_t* ids, int n_ids, int eos, const mtb_counters* counters, int k_max,
                              double prefill_seconds, double decoder_seconds, int trace, char* out, int out_size);
/* The policy a NULL params pointer selects (see mtb_spec_params); needs no
 * GPU.  Unparsable or out-of-range variables are reported here (-1, with
 * mtb_global_error) rather than clamped. */
int mtb_spec_params_from_env(mtb_spec_params* out);
/* MTB_KV_F32 or MTB_KV_F16 as MTB_KV_DTYPE selects (unset: MTB_KV_F32), -1 for
 * an unknown value; needs no GPU. */
int mtb_kv_type_from_env(void);
/* 256-K slices per block the F16 GEMV uses for an n x k projection on the
 * device configured last (1, 2 or 4; -1 for an invalid shape), so tests can
 * check which block shapes a model's projections reach. */
int mtb_f16_slices_per_block(int n, int k);
/* Test hook (host-side fault injection): the n-th device allocation made by
 * this library from now on fails as if cudaMalloc had (n = 0: off).  The
 * failing call returns its error and leaves no allocation behind. */
void mtb_debug_fail_alloc(int n);
/* Bounds-check build (libmoss_transcribe_b200_bc.so, -DMTB_BOUNDS_CHECK):
 * the kernels check cache positions, page-table entries, the attention
 * partial buffers and step row counts, record the first violated check on the
 * device and skip or redirect that access (no trap).  _enabled: 1 in that
 * build, 0 otherwise.  _status: the recorded site on `device` (0 none, 1 a
 * cache position outside the decoder's pages, 2 a page-table entry outside
 * the pool, 3 attention chunks beyond the partial buffers, 4 a step beyond 16
 * rows), then cleared; always 0 in a normal build; -1 if the device cannot be
 * selected.  Restores the caller's current device. */
int mtb_bounds_check_enabled(void);
int mtb_bounds_check_status(int device);
/* Returns the error of the last failed call on this thread that had no object. */
const char* mtb_global_error(void);

/* ---- model: decoder weights resident on one device ---- */
int mtb_model_load(const char* gguf_path, int device, mtb_model** out);
void mtb_model_free(mtb_model* m);
const char* mtb_model_error(const mtb_model* m);
/* hidden, n_layers, n_heads, n_kv_heads, head_dim, ffn, vocab, eos */
int mtb_model_dims(const mtb_model* m, int32_t* out8);
/* CTAs of the persistent verify-step kernel (one per SM), or 0 when verify
 * steps run as a graph of separate kernels (unsupported shape, repetition
 * penalty > 1, or MTB_NO_PERSISTENT set at load). */
int mtb_model_persistent_grid(const mtb_model* m);

/* ---- decoder: KV cache (paged, 64 positions per page) and step state ---- */
int mtb_decoder_create(mtb_model* m, int max_seq, int kv_type, int max_new, mtb_decoder** out);
void mtb_decoder_free(mtb_decoder* d);
const char* mtb_decoder_error(const mtb_decoder* d);
int mtb_decoder_past_len(const mtb_decoder* d);
int mtb_decoder_reset(mtb_decoder* d);
int mtb_decoder_rewind(mtb_decoder* d, int position);
/* Append T host rows [T][hidden] at past..past+T-1 (any T; chunks of 16),
 * writing the final-RMSNorm'd hidden rows to hidden_out [T][hidden] (may be NULL). */
int mtb_decoder_run(mtb_decoder* d, const float* embeds, int T, float* hidden_out);
/* Tied LM head on one host hidden row -> logits[vocab]. */
int mtb_decoder_logits(mtb_decoder* d, const float* hidden_row, float* logits);
/* KV rows of one layer (which 0 = K, 1 = V) as f32 [n_pos][n_kv][128]. */
int mtb_decoder_kv_read(mtb_decoder* d, int layer, int which, int pos0, int n_pos, float* out);
/* Synthetic fp16-valued KV at positions [0, n_pos) of every layer; sets past_len. */
int mtb_decoder_fill_synthetic_kv(mtb_decoder* d, int n_pos, uint32_t seed);

/* ---- generation ---- */
int mtb_greedy_generate(mtb_decoder* d, const float* fused, int seq, int max_new, int eos, float penalty,
                        int32_t* out_ids, int* n_out);
int mtb_spec_generate(mtb_decoder* d, const float* fused, int seq, int max_new, int eos,
                      const mtb_spec_params* params, int32_t* out_ids, int* n_out, mtb_counters* counters,
                      mtb_draft_fn draft, mtb_commit_fn commit, void* user);

/* fuse_embeds (src/generate.cpp:113-177) on the device: row p of out
 * [seq][hidden] (host) is the dequantised token_embd row of ids[p], except that
 * the k-th position holding audio_token_id takes audio row k (masked scatter).
 * Errors as the reference: an id outside [0, vocab), or more audio positions
 * than audio rows; fewer positions than rows is accepted. */
int mtb_fuse_embeds(mtb_decoder* d, const int32_t* ids, int seq, const float* audio, int n_audio, int audio_token_id,
                    float* out);
/* mtb_spec_generate from token ids + audio rows: the fused prompt is built on
 * the device (mtb_fuse_embeds) and prefilled from device memory, so it never
 * round-trips the host (generate.cpp:229-241 fuse_embeds + greedy_generate). */
int mtb_spec_generate_ids(mtb_decoder* d, const int32_t* ids, int seq, const float* audio, int n_audio,
                          int audio_token_id, int max_new, int eos, const mtb_spec_params* params, int32_t* out_ids,
                          int* n_out, mtb_counters* counters);

/* Continue from an existing cache: ids[0:n_ids] are the generated ids (the
 * last is the pending seed, not yet in the cache), past the cache length. */
int mtb_resume(mtb_decoder* d, const int32_t* ids, int n_ids, int past, int max_new, int eos,
               const mtb_spec_params* params);
/* One verify step.  draft == NULL -> on-device n-gram draft; otherwise the
 * n_draft host ids are the proposal.  Synchronous; new ids via mtb_read_ids. */
int mtb_spec_step(mtb_decoder* d, const int32_t* draft, int n_draft, mtb_counters* counters);
/* Same, asynchronous on the decoder's stream, proposal from DEVICE memory
 * (NULL -> on-device draft).  Nothing is copied to or from the host. */
int mtb_spec_step_async(mtb_decoder* d, const int32_t* draft_device, int n_draft);
/* Set the decode parameters and prefill the fused rows (the first id is
 * emitted), without decoding: the start of mtb_spec_generate
 * (src/cpu_speculative.cpp:68-99), for decoders stepped as a group.  Returns
 * once the prefill is queued on the decoder's stream (the rows have been
 * copied out of `fused`), so the members of a group prefill side by side; a
 * prefill that fails on the device is reported by the next call that reads
 * the decoder's state back (mtb_spec_run_group, mtb_read_ids, ...). */
int mtb_spec_prime(mtb_decoder* d, const float* fused, int seq, int max_new, int eos, const mtb_spec_params* params);
/* One verify step of n decoders (1..8) created from the same model, as ONE
 * persistent launch: each decoder drafts on the device; their rows (seed +
 * proposals, at most 16 together) are verified against their own KV caches;
 * each accepts and rolls back on its own.  Proposals beyond the 16 rows are
 * cut in group order (the accepted ids do not change: verification is strict
 * greedy; only the proposal counters do).  ds[0] needs the largest max_seq;
 * no repetition penalty.  Asynchronous: ordered after the work queued on every
 * member's stream and before the work queued on it later. */
int mtb_spec_step_group_async(mtb_decoder* const* ds, int n);
/* Group steps until every member has stopped (max_steps <= 0: no limit),
 * then synchronous; steps_out = steps launched.  New ids via mtb_read_ids. */
int mtb_spec_run_group(mtb_decoder* const* ds, int n, int max_steps, int* steps_out);
/* Device-side copy of the step state and ids (save) and back (restore),
 * asynchronous on the decoder's stream. */
int mtb_snapshot_save(mtb_decoder* d);
int mtb_snapshot_restore_async(mtb_decoder* d);
int mtb_read_ids(mtb_decoder* d, int32_t* out, int max_out, int* n_out, mtb_counters* counters);

/* ---- timing on the decoder's stream ---- */
int mtb_sync(mtb_decoder* d);
int mtb_event_record(mtb_decoder* d, int slot);          /* slot 0..15 */
int mtb_event_elapsed_ms(mtb_decoder* d, int a, int b, float* ms);
/* Kernel launches per verify step (counted when the step graph is built). */
int mtb_step_kernel_launches(mtb_decoder* d);
/* Timeline of the last persistent verify step (decoder created with
 * MTB_PROFILE=1 in the environment): out[2b], out[2b+1] = CTA 0's arrival and
 * release at grid barrier b, out[2*512], out[2*512+1] = kernel start and end,
 * out[2*512 + 2 + 4b + k] = sub-phase mark k of phase b (0 when unused),
 * out[6*512 + 2 + 512 c + b] = CTA c's arrival at barrier b,
 * out[6*512 + 2 + 256*512 + 16 (512 c + b) + k] = CTA c's sub-phase mark k of
 * phase b (c < 256, k < 16), all in ns of the
 * GPU global timer; the profile counterpart of the
 * reference's MTD_PROFILE phase timers (src/cpu_profile.cpp:23-68). */
int mtb_step_timeline(mtb_decoder* d, int64_t* out, int max_out, int* n_out);
/* Test read-back of the last persistent verify step's own outputs (decoder
 * created with MTB_STEP_CAPTURE=1 in the environment; for a group step, the
 * group's first decoder): the step's T rows (all streams, stream order) as
 * final-RMSNorm'd hidden rows hidden_out [T][hidden], each row's LM-head
 * maximum max_val[T] and its first index max_idx[T], and per stream
 * (rows, first row) in stream_rows[8][2].  Any output may be NULL. */
int mtb_step_capture(mtb_decoder* d, float* hidden_out, float* max_val, int32_t* max_idx, int32_t* stream_rows,
                     int* T_out);
/* Test hook: NaN into KV positions [pos0, pos0 + n_pos) of every layer (K and
 * V), to show that a step never reads a cache slot it has not written. */
int mtb_debug_poison_kv(mtb_decoder* d, int pos0, int n_pos);
/* Host<->device bytes this decoder has copied so far (both cumulative). */
int mtb_transfer_bytes(mtb_decoder* d, int64_t* h2d, int64_t* d2h);

/* ---- controller pieces, run by the same device kernels the loop uses ---- */
/* history: n host ids (n <= the decoder's max_new); out: up to `maximum` ids. */
int mtb_ngram_draft(mtb_decoder* d, const int32_t* history, int n, int maximum, int n_min, int n_max,
                    int32_t* out, int* n_out);
/* raw: n_raw host logits (n_raw <= vocab); history: n host ids. */
int mtb_greedy_choice(mtb_decoder* d, const float* raw, int n_raw, const int32_t* history, int n, float penalty,
                      int32_t* choice);

/* ---- LM head without device allocation ----
 * No counterpart in the reference (its LM head, Qwen3Decoder::logits_from_hidden,
 * allocates a ggml graph per call).  For callers that cannot allocate device
 * memory: serving processes that give all free device memory to their own pool
 * allocator at start-up and forbid later cudaMalloc, because a late cudaMalloc
 * can fail for lack of room and cudaMalloc/cudaFree synchronise the device.
 *
 * hidden_rows: DEVICE pointer to T final-normed hidden rows [T][hidden];
 * choices: DEVICE pointer to T int32, receives each row's first-max token id
 * (mtb_greedy_choice without penalty).  stream: a cudaStream_t, NULL for the
 * default stream; the call is asynchronous on it.  Limits: T in [1, 16],
 * hidden <= 4096; larger sizes return -2 with mtb_noalloc_error() set.
 * Intermediates live in one static device array of about 148 KB that every
 * device loading this library holds until exit; the first call on a device
 * looks its address up (call it once before any stream capture).  Calls share
 * that array: calls that overlap on the GPU race.  Nothing is allocated: no
 * cudaMalloc, cudaFree or allocating library routine is called.  The call runs
 * on the model's device and leaves the caller's current device as it found it. */
int mtb_lm_head_argmax_noalloc(const mtb_model* m, const float* hidden_rows, int T, int32_t* choices, void* stream);
const char* mtb_noalloc_error(void);

/* ---- Audio front end: 16 kHz samples -> the decoder's audio embedding rows ----
 * Replaces mt::AudioEncoder (src/audio_encoder.hpp:23-34, src/audio_encoder.cpp:16-75):
 * WhisperMel::compute (src/mel.cpp:153-224), WhisperEncoder::encode
 * (src/whisper_encoder.cpp:98-207) and AudioAdaptor::apply
 * (src/audio_adaptor.cpp:39-96), all on the device.  The GGUF is the one the
 * decoder loads (mtd.audio.*, mtd.feat.*, mel_filters, enc.*, adaptor.*);
 * the encoder and adaptor linear weights must be q8_0. */
typedef struct mtb_audio mtb_audio;
int mtb_audio_load(const char* gguf_path, int device, mtb_audio** out);
void mtb_audio_free(mtb_audio* a);
/* The object's last error, or the last load error of this thread for NULL. */
const char* mtb_audio_error(const mtb_audio* a);
/* dims[10]: hidden, d_model, n_layers, n_heads, ffn, n_mels, mel frames per
 * chunk, samples per chunk, encoder frames per chunk, merge size. */
int mtb_audio_dims(const mtb_audio* a, int32_t* dims);
/* Sum over 30 s chunks of token_len = (unpadded - 1) / (hop * 2 * merge) + 1:
 * the rows mtb_audio_encode returns for n_samples samples. */
int mtb_audio_tokens(const mtb_audio* a, int n_samples);
/* AudioEncoder::encode: host samples -> host rows out[n_tokens][hidden]
 * (max_tokens rows available).  Empty input and a too-small output are
 * errors, as in the reference. */
int mtb_audio_encode(mtb_audio* a, const float* samples16k, int n_samples, float* out, int max_tokens,
                     int* n_tokens);
/* Device time of the last mtb_audio_encode (host copies included), ms. */
float mtb_audio_last_ms(const mtb_audio* a);
/* Test read-back of one chunk: mel [n_mels][frames] (after the chunk
 * normalisation) and the encoder output [encoder frames][d_model] (after the
 * final LayerNorm, before the trim); n_samples <= samples per chunk (the rest
 * is zero-padded as in encode); either output may be NULL. */
int mtb_audio_debug_chunk(mtb_audio* a, const float* samples, int n_samples, float* mel_out, float* enc_out);

/* ---- Operators on a caller's own device memory ----
 * For programs that keep their own projections, cache pool or logits and want
 * this library's kernels for what lies between: rotary positions with the
 * append to a paged cache, attention over it, eviction from it, and the logits
 * that steer the next token.  No counterpart in the reference (its cache is
 * one contiguous tensor per layer, its logits leave the device).
 *
 * Conventions, beside those above.  Every pointer is DEVICE memory unless it
 * says host; nothing is allocated, no host copy is made and no call waits for
 * the device.  `stream` is a cudaStream_t (NULL: the default stream); a call
 * is asynchronous on it, may be captured into a graph, runs on the device that
 * owns the memory and leaves the caller's current device as it found it.
 * 0 on success; -1 for a CUDA error, a null pointer, or the cache's k (or the
 * logits) not in device memory, -2 for an argument outside its limits, with
 * mtb_global_error() set and nothing launched.  Pointers are aligned to their
 * elements, and further where it says so; the others are taken as memory of the
 * same device.  Calls may run at once on any streams as long as no memory that
 * one writes is used by another.  Sizes that live on the device (lengths, page-table entries) are
 * checked by the kernels: a violated check sets its bit in *status (never
 * cleared by the library) and the access is skipped, never made. */
enum { MTB_T_F32 = 0, MTB_T_F16 = 1, MTB_T_BF16 = 2 };
enum {
    MTB_BAD_PAGE = 1,   /* a page-table entry outside [0, n_pages): its positions count as masked, are not written,
                           and a sequence that has one is not evicted from */
    MTB_BAD_LEN = 2,    /* kv_len outside [0, 64 table_stride] (clamped to it), or smaller than the new tokens */
    MTB_BAD_TOKENS = 4, /* cu_tokens not ascending inside [0, n_tokens]: the sequence counts as one without tokens */
    MTB_BAD_WAIT = 8    /* a wait inside the attention or its weights ran out (two seconds; none lasts longer than a CTA's
                           share of one tile of rows, which takes that long from some 10^8 slots on): that call's
                           results are void, its workspace must be zeroed again */
};

/* A view of one layer's paged cache in the caller's pool: 64 positions per
 * page, position `slot` of a sequence in page page_table[seq][slot / 64], row
 * slot % 64.  Dim d of KV head h is at k[page * page_stride + h * head_stride
 * + row * head_dim + d] (strides in elements, the same for v), so a view of
 * one layer of [page][layer][K/V][kv_head][64][head_dim] needs no copy.  k and
 * v are 16-byte aligned and the strides multiples of 8 elements.  position and
 * weight are the book-keeping of eviction, one value per cached position and
 * KV head, [page][kv_head][64] without gaps; NULL where not wanted.  Sequences
 * may share pages that a call only reads. */
typedef struct mtb_paged_cache {
    void* k;
    void* v;
    int32_t type;             /* MTB_T_F16 or MTB_T_BF16 */
    int32_t head_dim;         /* 64 or 128 */
    int32_t n_kv_heads;
    int32_t n_pages;          /* pages in the pool */
    int64_t page_stride, head_stride;
    const int32_t* page_table; /* [n_seq][table_stride] */
    int32_t table_stride;
    int32_t n_seq;
    const int32_t* kv_len;    /* [n_seq] positions held, the call's new tokens included */
    int32_t* position;        /* or NULL */
    float* weight;            /* or NULL */
    int32_t* status;          /* one word of MTB_BAD_* bits, or NULL */
} mtb_paged_cache;

/* Scaling of rotary frequencies for contexts beyond the trained length.
 * LINEAR: all frequencies / factor.  NTK: base * factor^(R / (R - 2)).  YARN:
 * pairs that turn more than `fast` times over original_len keep their frequency,
 * those below `slow` turns are divided, a ramp over the pair index between, and
 * cos and sin are scaled by 0.1 ln(factor) + 1.  BANDS: the same blend with the
 * ramp over the number of turns, unscaled. */
enum { MTB_ROPE_PLAIN = 0, MTB_ROPE_LINEAR = 1, MTB_ROPE_NTK = 2, MTB_ROPE_YARN = 3, MTB_ROPE_BANDS = 4 };
/* inv_freq [rotary_dim / 2] and *factor (both HOST memory) for
 * mtb_rope_append; computed once by the caller, needs no GPU. */
int mtb_rope_frequencies(int rotary_dim, double base, int kind, double factor, double original_len, double fast,
                         double slow, double* inv_freq, float* out_factor);
/* Rotary positions of q and k, and the append of k and v to the cache, in one
 * pass.  Tokens cu_tokens[s] .. cu_tokens[s + 1] - 1 (cu_tokens [n_seq + 1])
 * are the newest of sequence s: token i of n goes to slot kv_len[s] - n + i.
 * q [n_tokens][n_heads][head_dim], k and v [n_tokens][n_kv_heads][head_dim], rows
 * of a token contiguous, tokens `stride` elements apart, all of `in_type`;
 * q_out has the cache's type (it may be q itself when in_type is that type and
 * the strides are equal).  The first rotary_dim dims are rotated by
 * positions[token] * inv_freq[pair] (64-bit, reduced before the sine), pairs
 * (j, j + rotary_dim / 2) or, interleaved, (2j, 2j + 1); cos and sin times
 * factor; the others pass.  Each result is rounded once.  Where the cache has
 * them, position gets the token's position and weight 0.  Rows behind the last
 * sequence are left as they are. */
int mtb_rope_append(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, const int32_t* positions,
                    int in_type, const void* q, int64_t q_stride, int n_heads, const void* k, int64_t k_stride,
                    const void* v, int64_t v_stride, const double* inv_freq, int rotary_dim, int interleaved,
                    float factor, void* q_out, int64_t q_out_stride, void* stream);

/* Device bytes of mtb_paged_attention's workspace (any sizes).  Zeroed once
 * before its first use; every call leaves it ready for the next.  Calls (and
 * replays of captured graphs) that share one must not overlap. */
enum { MTB_ATTENTION_WORKSPACE = 64 << 20 };
/* Attention of the new tokens over the paged cache, causal: token i of a
 * sequence's n sees the slots <= kv_len - n + i, so its own (appended before).
 * q and out [n_tokens][n_heads][head_dim] of the cache's type (16-byte aligned,
 * strides multiples of 8 elements); n_heads a multiple of n_kv_heads, at most
 * 64 for each, n_tokens * n_heads / n_kv_heads at most 2^30; head h reads KV head
 * h / (n_heads / n_kv_heads).  Scores are scale times q.k (1 / sqrt(head_dim) usually).
 * lse [n_tokens][n_heads] f32 (or NULL) gets log sum exp of the row's scores.
 * A row that sees nothing gets out 0 and lse -inf; rows behind the last
 * sequence are left as they are.  Slots a row does not see may hold anything
 * in K; in V, slots at or behind kv_len may too, and a new token's V must be finite
 * where earlier tokens of the same call matter.  max_tokens: the most new tokens
 * of one sequence, if known (it only picks the kernel; <= 0: n_tokens). */
int mtb_paged_attention(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, int max_tokens,
                        const void* q, int64_t q_stride, int n_heads, float scale, void* out, int64_t out_stride,
                        float* lse, void* workspace, size_t workspace_bytes, void* stream);
/* The softmax weight each cached position received in that attention:
 * cache->weight[slot] = decay * cache->weight[slot] + sum of exp(score - lse) over the
 * new tokens that see the slot and the query heads of its KV head (decay 0
 * ignores the old value; a row whose lse is -inf adds nothing).  A page whose weights are written belongs to one
 * sequence.  Slots at or behind kv_len are left as they are;
 * sequences without new tokens too.  Arguments as above. */
int mtb_attention_weights(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, int max_tokens,
                          const void* q, int64_t q_stride, int n_heads, float scale, const float* lse, float decay,
                          void* stream);
/* Test hook: the kernels of the next n calls of the two hand out none of their work,
 * so that their waits run out and MTB_BAD_WAIT is set (0 clears).  Process-wide. */
void mtb_debug_stall_attention(int n);

/* Device bytes of mtb_cache_evict's workspace (needs no GPU); -2 for sizes that
 * a cache cannot have (n_seq and n_kv_heads at most 65535, their product and table_stride
 * at most 2^24).  Needs no zeroing; calls that share one must not overlap. */
int64_t mtb_cache_evict_workspace(int n_seq, int n_kv_heads, int table_stride);
/* Eviction by accumulated weight, in place, each KV head on its own: of a
 * sequence with kv_len > keep the `keep` slots stay that rank highest, others go.
 * Rank: first slots whose position is < sinks or among the `recent` highest
 * (> newest - recent), then larger weight (NaN below all), then lower slot.
 * Kept slots below `keep` stay where they are; the kept ones at or above it move
 * into the gaps, both in ascending order (K, V, position and weight), so the cache
 * is then slots [0, keep) in no particular order of positions: attention of later
 * tokens does not depend on it, since rotary positions are in K.
 * new_len[s] = min(kv_len, keep); it may be kv_len itself.  Needs position
 * and weight, sinks + recent <= keep, n_pages <= 2^25, and each page in the table once. */
int mtb_cache_evict(const mtb_paged_cache* cache, int keep, int sinks, int recent, int32_t* new_len, void* workspace,
                    size_t workspace_bytes, void* stream);

/* What mtb_logits_process applies; any pointer may be NULL (left out). */
typedef struct mtb_logits_params {
    const int32_t* history;     /* [history_len] ids; row r's are [history_begin[r], history_end[r]) (ranges may overlap) */
    int64_t history_len;        /* the kernels cut ranges to it */
    const int32_t *history_begin, *history_end; /* [rows] */
    const float *repetition, *presence, *frequency; /* [rows] */
    const int32_t* bias_ids;    /* [bias_len]; row r's entries are [bias_begin[r], bias_end[r]) */
    const float* bias_values;   /* [bias_len] */
    int64_t bias_len;
    const int32_t *bias_begin, *bias_end; /* [rows] */
    const uint32_t* mask;       /* bit i % 32 of word i / 32 of a mask row: id i is allowed */
    int64_t mask_stride;        /* words between mask rows */
    int32_t mask_rows;
    const int32_t* mask_row;    /* [rows] the mask row of each logits row, NULL: its own index; a row outside
                                   [0, mask_rows) is not masked */
} mtb_logits_params;
/* logits [rows][vocab] of `type`, rows `stride` elements apart; out the same type
 * (it may be logits itself, or NULL), choice [rows] (or NULL).  For an id that
 * occurs c > 0 times in its row's history: x > 0 ? x / repetition : x * repetition,
 * then - frequency * c, then - presence (src/cpu_speculative.cpp:39-50 has the first);
 * then + the bias of the id's last entry; then -inf where the mask forbids it.
 * Evaluated in f32 in this order, each step rounded; out is rounded once more.
 * choice: the lowest id of the largest f32 value; NaN never wins; -1 when no
 * value is above -inf.  Ids outside [0, vocab) in history or biases are skipped.
 * vocab, history_len and bias_len are at most 2^30, rows at most 2^26. */
int mtb_logits_process(const void* logits, int type, int rows, int vocab, int64_t stride,
                       const mtb_logits_params* params, void* out, int64_t out_stride, int32_t* choice, void* stream);

#ifdef __cplusplus
}
#endif
#endif
