/* q3h.h - C ABI of libq3h, the MI355X (gfx950) engine of the Qwen3-TTS frame
 * step: the talker (Qwen3, 28 layers) and the code predictor (Qwen3, 5 layers,
 * 15 forwards per frame), with device-resident weights and K/V caches.
 *
 * Every entry point is extern "C", cdecl, takes plain pointers and sizes, and
 * returns an int status: 0 on success, a negative Q3H_E* code on failure, with
 * the message in q3h_last_error() (thread-local, valid until the next call on
 * the same thread). Ownership follows mormot.ai.tts.qwen.lm.pas:364-368
 * (TQwenLm.Destroy): contexts and frames before their stacks, stacks before
 * their device. A stack may serve contexts used from several threads at once;
 * one context (or frame) is used by one thread at a time
 * (mormot.ai.tts.qwen.talker.pas:77). Each entry point makes its device
 * current, so calls may arrive on any thread (mormot.ai.tts.qwen.pas:281-291).
 *
 * Each declaration names the reference interface it replaces (paths relative
 * to the reference checkout). The mormot2-ai engine those Pascal call sites
 * reach (TQwen3Model, TQwen3Vulkan, TDecoderContext) is an un-vendored
 * submodule; only its call sites in the reference tree are cited.
 */
#ifndef Q3H_H
#define Q3H_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* weight formats: the host side of q3h_stack_create / q3h_stack_add_head,
   and the storage of a stack (TInferDType idtF32 / idtQ8_0) */
#define Q3H_F32 0
#define Q3H_Q8_0 1 /* ggml block_q8_0 on the host: fp16 scale + 32 int8, 34 B */
#define Q3H_BF16 2 /* bfloat16 (the text embedding table) */

/* status codes */
#define Q3H_OK 0
#define Q3H_E_ARG (-1)      /* invalid argument or shape */
#define Q3H_E_HIP (-2)      /* a HIP runtime call failed */
#define Q3H_E_CAPACITY (-3) /* a context would exceed its positions */
#define Q3H_E_STATE (-4)    /* call out of order (e.g. step before start) */
#define Q3H_E_NODEV (-5)    /* no usable gfx950 device */

typedef struct q3h_device q3h_device;
typedef struct q3h_stack q3h_stack;
typedef struct q3h_context q3h_context;
typedef struct q3h_frame q3h_frame;
typedef struct q3h_text_proj q3h_text_proj;
typedef struct q3h_codec q3h_codec;

/* TDecoderConfig (mormot.ai.tts.qwen.lm.pas:184-191) + TQwen3Vulkan.KvF16
   (lm.pas:353) + the numerics of the Q8_0 products */
typedef struct {
  int32_t layers, hidden, heads, kv_heads, head_dim, intermediate;
  float rms_eps, rope_theta;
  int32_t dtype;         /* storage: Q3H_F32 or Q3H_Q8_0 (weights and heads) */
  int32_t kv_f16;        /* K/V cache in half floats (lm.pas:128-130): 0 or 1; or
                            Q3H_KV_Q8 (2; no reference counterpart): a byte per
                            element and a scale per position and head, or
                            Q3H_KV_Q4 (4): four bits per element with steps and
                            a scale, both f32 activations only. Other values are refused; before
                            there were int8 caches any value but 0, such as a
                            truth value of -1, chose half floats */
  int32_t act_q8;        /* Q8_0 only: 1 = activations quantized per 32-block
                            (int8 products, ggml vec_dot_q8_0_q8_0); 0 = f32
                            activations times dequantized weights */
  int32_t max_positions; /* the largest context of this stack (RoPE table) */
} q3h_stack_config;

/* one layer, host memory, matrices [out][in] row-major in src_dtype */
typedef struct {
  const void *wq, *wk, *wv, *wo, *wgate, *wup, *wdown;
  const float *input_norm, *post_norm; /* [hidden] */
  const float *q_norm, *k_norm;        /* [head_dim] */
} q3h_layer_weights;

typedef struct {
  int32_t src_dtype;               /* Q3H_F32, Q3H_Q8_0 (ggml blocks) or Q3H_BF16 (the
                                      safetensors rows as stored: widened and, for a
                                      Q8_0 stack, quantized on the device, the
                                      conversion of lm.pas:244-308) */
  const q3h_layer_weights *layers; /* [layers] */
  const float *final_norm;         /* [hidden] */
} q3h_weights;

/* ---- device: replaces TQwenVulkan (lm.pas:44-62, 202-222) ---- */

/* 1 when a gfx950 device is present (TQwenVulkan.Available, lm.pas:202-205) */
int q3h_device_available(void);
/* TQwenVulkan.Create (lm.pas:207-211) */
int q3h_device_open(int ordinal, q3h_device **out);
/* TQwenVulkan.DeviceName (lm.pas:219-222); NULL on a NULL device */
const char *q3h_device_name(const q3h_device *dev);
/* TQwenVulkan.DeviceBytes (lm.pas:57-59): the weight bytes of its stacks */
int64_t q3h_device_bytes(const q3h_device *dev);
/* TQwenVulkan.Destroy (lm.pas:213-217) */
int q3h_device_close(q3h_device *dev);
/* the message of the last failure on this thread ("" if none) */
const char *q3h_last_error(void);

/* ---- stack: replaces TQwen3Model.CreateStack (lm.pas:174-179) followed by
   TQwen3Vulkan.Create(model, backend) (lm.pas:351); the library copies (and
   quantizes or repacks) the host weights, so they may be freed on return ---- */
int q3h_stack_create(q3h_device *dev, const q3h_stack_config *cfg,
                     const q3h_weights *w, q3h_stack **out);
/* TQwenLmHeads.Add (lm.pas:277-308): a head [rows][hidden] in src_dtype
   (Q3H_F32, Q3H_Q8_0 or Q3H_BF16), stored in the stack's dtype; *index
   receives its number (0, 1, ...) */
int q3h_stack_add_head(q3h_stack *s, const void *w, int rows, int src_dtype,
                       int *index);
/* StackBytes (lm.pas:182-197) of the layers on the device, heads excluded */
int64_t q3h_stack_bytes(const q3h_stack *s);
/* TQwen3Vulkan.Free (lm.pas:366) */
int q3h_stack_destroy(q3h_stack *s);

/* ---- context: replaces TQwen3Vulkan.NewContext / TDecoderContext ---- */

/* lm.pas:354 (NewContext); max_positions <= the stack's max_positions */
int q3h_context_create(q3h_stack *s, int max_positions, q3h_context **out);
/* TQwenLm.Reset (lm.pas:374-378): the next row is at position 0 */
int q3h_context_reset(q3h_context *c);
/* TQwenLm.Length (lm.pas:136-138); negative on error */
int q3h_context_length(const q3h_context *c);
/* lm.pas:365 (fCtx.Free) */
int q3h_context_destroy(q3h_context *c);
/* no reference counterpart (long-context setups and tests): write the K/V of
   positions [0, len) from host f32 [layers][kv_heads][len][head_dim] (rounded
   to half floats when kv_f16) and set the length to len */
int q3h_context_fill_kv(q3h_context *c, const float *k, const float *v, int len);
/* no reference counterpart (tests): read the K/V cache of one layer for
   positions [0, length) as f32 [kv_heads][length][head_dim] */
int q3h_context_read_kv(q3h_context *c, int layer, float *k, float *v);
/* no reference counterpart (measurement): the decode attention of every
   layer for one new row at position length (the attention kernels of
   q3h_forward_embeds with rows = 1, fused QK-norm / RoPE / K/V append),
   launched directly iters times over the layers on one stream.
   us_per_launch: the time between two events around those launches per
   layer (with the merge of the splits on long contexts: both kernels and the
   gaps between launches); bytes_per_launch: algorithmic bytes
   (the cache of length positions read, the new key and value written, the
   q / k / v row read, the outputs written). The row's q / k / v are zeros;
   the key and value written at position length are scratch (the length does
   not change). Stacks with f32 activations (act_q8 = 0). */
int q3h_context_time_attention(q3h_context *c, int iters, float *us_per_launch,
                               int64_t *bytes_per_launch);

/* ---- the forward: TQwenLm.Forward (lm.pas:391-408), i.e.
   TQwen3Vulkan.ForwardEmbeds(ctx, x, rows, nil, false, fLast) (lm.pas:397)
   followed by fCpu.Linear(fLast, 1, hidden, head, rows) (lm.pas:404-406),
   with the head on the device. x [rows][hidden] host f32 at positions
   length..length+rows-1; normed_last [hidden] (nullable) receives the
   final-normed state of the last row; head: an index of q3h_stack_add_head,
   or -1 for none; logits [head rows] (nullable). Blocks until the outputs
   are in host memory. rows <= 0 does nothing (lm.pas:394-395). One row
   replays a HIP graph the context captures per (head, position cover)
   (covers of 64 positions up to 256, of 256 beyond; at most 32 graphs per
   context, the one unused longest gives way, all dropped when its work buffers
   grow) and copies its row, logits and state through a pinned host buffer of
   the context (several rows: the logits and state); the results are those of
   the same launches made directly (q3h_forward_embeds_noalloc). ---- */
int q3h_forward_embeds(q3h_context *c, const float *x, int rows, int head,
                       float *logits, float *normed_last);

/* No counterpart in the reference. For callers that cannot allocate device
   memory (tight serving loops, harnesses that forbid hipMalloc); it is called
   outside any stream capture, like q3h_forward_embeds: it launches on the
   context's own stream, copies pageable host memory and blocks until the
   outputs are in host memory. q3h_forward_embeds with the same arguments and results,
   but its work buffers are carved from one static device array of
   Q3H_NOALLOC_SCRATCH_BYTES per GPU (set up by q3h_device_open) instead of
   the context's own buffers, which q3h_forward_embeds grows with hipMalloc.
   Calls no allocating routine. rows <= Q3H_NOALLOC_MAX_ROWS, and the
   buffers of the call (they grow with rows and, for fewer than 16 rows of
   an f32-activation stack over more than 256 positions, with the decode
   attention's splits) must fit the array: otherwise
   Q3H_E_CAPACITY and nothing is computed. With an int8 or 4-bit cache or rotary
   positions of q3h_stack_set_rope they grow with rows alone: the attention's
   partial sums take what the others leave, and where that is less than
   q3h_forward_embeds uses (16 heads over 8, an f32 cache: 33 to 64 rows over
   more than 130 to 310 positions, 17 to 32 over 1480 to 1730; an int8 or
   4-bit one: over twice as many or more), the positions are cut into fewer pieces: the
   results differ in the order of those sums. Every call on one GPU shares that
   GPU's array, which keeps the last call's contents (no kernel reads a
   buffer before writing it); calls on one device are serialized by a lock
   of the device, since overlapping calls would race on the array. */
#define Q3H_NOALLOC_MAX_ROWS 64
#define Q3H_NOALLOC_SCRATCH_BYTES (16 << 20)
int q3h_forward_embeds_noalloc(q3h_context *c, const float *x, int rows, int head,
                               float *logits, float *normed_last);

/* TQwenLm.Forward with TQwenLm.Probe set (lm.pas:139-142, 380-389: the
   probe receives the output of every layer, "name.layerN", then the normed
   state of every row, "name.out"): q3h_forward_embeds, plus layer_out
   [layers][rows][hidden] (host f32, nullable) receiving the raw output of
   each layer for every row (the residual stream after the layer's down
   projection), so that a difference against another implementation can be
   located at a layer, and normed_rows [rows][hidden] (host f32, nullable)
   receiving the final RMSNorm of every row (normed_last is its last row).
   The outputs are those of q3h_forward_embeds; the copies add one
   device-to-device copy per layer. */
int q3h_forward_embeds_probe(q3h_context *c, const float *x, int rows, int head,
                             float *logits, float *normed_last, float *layer_out,
                             float *normed_rows);

/* no reference counterpart (the reference is single-stream): one row per
   context, n contexts of the same stack at their own positions;
   x [n][hidden]; heads [n] (or NULL: no logits); logits [n][head rows of
   heads[0]] (all heads of one call must have the same rows); normed [n][hidden]
   (nullable). Up to 256 contexts of one max_positions with one head: from the
   second use of a (n, head, position cover of the longest context) on replayed
   from a HIP graph that ctxs[0] captures then (at most 64, the one unused
   longest gives way), the contexts read on the device, so any contexts of the
   same n may follow. */
int q3h_forward_embeds_batch(q3h_context *const *ctxs, int n, const float *x,
                             const int *heads, float *logits, float *normed);

/* ---- the frame step: a device-resident, greedy restatement of
   TQwenTalker.NextFrame (talker.pas:640-681) with ChooseCode0 (talker.pas:
   595-630), ChooseCode (talker.pas:632-638) and AddRow (talker.pas:423-429),
   for n_streams independent sentences, replayed as one hipGraph per step ---- */
typedef struct {
  int32_t n_streams;          /* 1..64 */
  int32_t talker_head;        /* head index in the talker stack */
  int32_t cp_heads[15];       /* head indices in the code-predictor stack */
  int32_t vocab, cp_vocab;    /* 3072, 2048 */
  int32_t groups;             /* 16 */
  int32_t eos;                /* codec_eos_token_id, -1: none */
  float repetition_penalty;   /* 1.05 (talker.pas:215) */
  int32_t max_frames;         /* frames per sentence (history capacity) */
  int32_t max_positions;      /* talker positions per stream */
  int32_t use_graph;          /* 1: capture the step once, replay it */
} q3h_frame_config;

/* TQwenTalker.Create's tables (talker.pas:300-311): codec_emb [vocab][hidden],
   pred_emb[g] [cp_vocab][hidden] (g = 0..groups-2), tts_pad [hidden];
   copied to the device */
int q3h_frame_create(q3h_stack *talker, q3h_stack *cp, const q3h_frame_config *cfg,
                     const float *codec_emb, const float *const *pred_emb,
                     const float *tts_pad, q3h_frame **out);
/* the talker part of TQwenTalker.Start (talker.pas:586-593): reset stream s,
   prefill its rows, keep the logits and the last normed state; trailing
   [trailing_rows][hidden] (talker.pas:578-580) follows the frames */
int q3h_frame_start(q3h_frame *f, int stream, const float *prefill, int rows,
                    const float *trailing, int trailing_rows);
/* no reference counterpart (batched serving; the reference starts one
   sentence at a time): q3h_frame_start for n distinct streams at once. The
   prompts of an int8 stack, and those over 64 rows of the others, run as the
   rows of one pass (of at most 8192 rows, each taking the prompts left that
   still fit; its work buffers, at most 0.54 GB, stay with the frame); the rest
   each on its stream's own talker context and HIP stream, so that they overlap
   on the device; blocks until all are done. streams [n];
   prefill[i] [rows[i]][hidden]; trailing (nullable) and trailing_rows
   (nullable: none) as q3h_frame_start's per stream. The results equal n
   calls of q3h_frame_start. Every argument is checked before any prefill is
   enqueued (a bad or repeated stream: Q3H_E_ARG, nothing started). */
int q3h_frame_start_batch(q3h_frame *f, int n, const int *streams,
                          const float *const *prefill, const int *rows,
                          const float *const *trailing, const int *trailing_rows);
/* one NextFrame for every started stream: codes [n_streams][groups] (-1 for a
   stream that has ended); alive [n_streams] (nullable) 1 while a stream runs,
   0 once its code 0 was eos. */
int q3h_frame_step(q3h_frame *f, int32_t *codes, int32_t *alive);
/* the talker logits [vocab] and normed state [hidden] of stream s (nullable
   outputs), as fLogits / fPastHidden after the last Start or step */
int q3h_frame_state(q3h_frame *f, int stream, float *logits, float *past_hidden);
int q3h_frame_destroy(q3h_frame *f);

/* TQwenSampling (talker.pas:60-70) without the repetition penalty (a frame
   setting): the choosers of code 0 (talker) and of codes 1..15 (code
   predictor, the sub-sampler). do_sample 0: argmax, as QwenGreedy. Else the
   scores (code 0: after ChooseCode0's processors) / temperature, top-k (0:
   off; ties at the k-th value kept), top-p (1: off; < 1 needs 1 <= top_k <=
   64), then one uniform through the inverse distribution (the logits warpers
   of Hugging Face generate(), which NewSampler, talker.pas:455-469,
   configures). Uniforms: Philox4x64-10 of counter (frame, group, 0, 0) under
   key (seed, 0) for code 0 (group 0), (seed xor 0x5DEECE66D, 0) for code g
   (group g), frame = frames of the sentence before this one. seed: the
   sentence seed of every q3h_frame_start* (0: a fresh random one per start,
   as talker.pas:582-584). At most 3072 codes per chooser. */
typedef struct {
  int32_t do_sample;
  float temperature;
  int32_t top_k;
  float top_p;
  int32_t sub_do_sample;
  float sub_temperature;
  int32_t sub_top_k;
  float sub_top_p;
  uint64_t seed;
} q3h_sampling;

/* property TQwenTalker.Sampling (talker.pas:150-151) for every stream of the
   frame; takes effect at the next step (its seed at the next start) */
int q3h_frame_set_sampling(q3h_frame *f, const q3h_sampling *s);

/* ---- the text projection and the device-side prefill ---- */
typedef struct {
  int32_t text_vocab;  /* rows of the text embedding (talker text_vocab_size, 151936) */
  int32_t text_hidden; /* text_hidden_size, 2048 (1024, 2048 or 3072) */
  int32_t hidden;      /* the talker's hidden_size, 1024 (a multiple of 16) */
  int32_t emb_dtype;   /* Q3H_BF16 (as in the safetensors file) or Q3H_F32 */
} q3h_text_config;

/* TQwenTalker's text projection weights (talker.pas:302-307): emb
   [text_vocab][text_hidden] (talker.model.text_embedding), fc1 [text_hidden]
   [text_hidden] + b1 [text_hidden], fc2 [hidden][text_hidden] + b2 [hidden]
   (talker.text_projection.linear_fc1 / fc2, widened to f32); copied to the
   device as given (the products stay in f32) */
int q3h_text_create(q3h_device *dev, const q3h_text_config *cfg, const void *emb,
                    const float *fc1_w, const float *fc1_b, const float *fc2_w,
                    const float *fc2_b, q3h_text_proj **out);
/* TQwenTalker.TextProject (talker.pas:390-421): y [n][hidden] =
   fc2 . SiLU(fc1 . emb[ids[r]] + b1) + b2, SiLU 0 below -80. n == 0 does
   nothing; an id outside [0, text_vocab) is Q3H_E_ARG ("text token out of
   range", nothing computed) */
int q3h_text_project(q3h_text_proj *t, const int32_t *ids, int n, float *y);
int q3h_text_destroy(q3h_text_proj *t);

/* the special ids TQwenTalker.Start uses (talker.pas:256-261): text ids
   tts_bos / tts_eos / tts_pad (config tts_*_token_id), codec ids codec_pad /
   codec_bos (talker_config codec_pad_id / codec_bos_id) */
typedef struct {
  int32_t tts_bos, tts_eos, tts_pad;
  int32_t codec_pad, codec_bos;
} q3h_start_ids;

/* TQwenTalker.Start (talker.pas:471-593) from its token ids, on the device:
   ids [n_ids] = PromptIds (im_start, assistant, \n, the text, im_end, \n,
   im_start, assistant, \n; n_ids >= 9), codec [n_codec] = the think /
   language / speaker ids then codec_pad, codec_bos (n_codec >= 2). The
   prefill rows (the role, tts_pad / tts_bos over the codec ids, then the text
   over codec_pad and tts_eos, tts_pad over codec_bos when non_streaming, else
   the first text token over codec_bos) and the trailing rows are built on the
   device from t's projection and the frame's codec_emb, then stream s starts
   as q3h_frame_start does with them. tts_bos / tts_eos / tts_pad are
   projected with the text. Errors: an id out of range (Q3H_E_ARG), more
   rows than max_positions (Q3H_E_CAPACITY) or trailing rows than max_frames
   (Q3H_E_ARG). */
int q3h_frame_start_text(q3h_frame *f, int stream, q3h_text_proj *t, const q3h_start_ids *sp,
                         const int32_t *ids, int n_ids, const int32_t *codec, int n_codec,
                         int non_streaming);

/* ---- the 12 Hz decoder's back part: replaces TQwenCodecVulkan's GPU pass
   (src/tts/mormot.ai.tts.qwen.codec.vulkan.pas:568-652) ---- */

/* the tensors of the back part (TQwenCodec.Create, codec.pas:644-751), f32,
   host memory, in their safetensors layouts (decoder.* of the speech
   tokenizer); the library repacks and copies them */
typedef struct {
  const float *a1_alpha, *a1_beta; /* block.{2+r}.act1.alpha / beta [dim] */
  const float *c1_w, *c1_b;        /* block.{2+r}.conv1.conv [dim][dim][7], [dim] */
  const float *a2_alpha, *a2_beta; /* block.{2+r}.act2 */
  const float *c2_w, *c2_b;        /* block.{2+r}.conv2.conv [dim][dim][1], [dim] */
} q3h_codec_res;

typedef struct {
  const float *act_alpha, *act_beta; /* decoder.{i+1}.block.0 [in] */
  const float *up_w, *up_b;          /* block.1.conv [in][out][2 rate], [out] */
  q3h_codec_res res[3];              /* dilations 1, 3, 9 */
} q3h_codec_block;

typedef struct {
  const float *up_w[2], *up_b[2];     /* upsample.i.0.conv [1024][1024][2], [1024] */
  const float *dw_w[2], *dw_b[2];     /* upsample.i.1.dwconv.conv [1024][1][7], [1024] */
  const float *norm_w[2], *norm_b[2]; /* upsample.i.1.norm [1024] */
  const float *pw1_w[2], *pw1_b[2];   /* upsample.i.1.pwconv1 [4096][1024], [4096] */
  const float *pw2_w[2], *pw2_b[2];   /* upsample.i.1.pwconv2 [1024][4096], [1024] */
  const float *gamma[2];              /* upsample.i.1.gamma [1024] */
  const float *conv0_w, *conv0_b;     /* decoder.0.conv [1536][1024][7], [1536] */
  q3h_codec_block block[4];           /* decoder.1 .. 4 (rates 8, 5, 4, 3) */
  const float *out_alpha, *out_beta;  /* decoder.5 [96] */
  const float *out_w, *out_b;         /* decoder.6.conv [1][96][7], [1] */
} q3h_codec_weights;

/* TQwenCodecVulkan.CreateVulkan's upload (codec.vulkan.pas:166-237):
   max_frames frames per device pass (1..64; longer inputs run in passes, as
   CHUNK_FRAMES does) */
int q3h_codec_create(q3h_device *dev, const q3h_codec_weights *w, int max_frames,
                     q3h_codec **out);
/* TQwenCodecVulkan.Reset (codec.vulkan.pas:455-488): every history to zeros */
int q3h_codec_reset(q3h_codec *c);
/* TQwenCodecVulkan.Back (codec.vulkan.pas:633-652): x [frames][1024] (the
   transformer output) -> pcm [frames * 1920] in [-1, 1]. Causal: each
   convolution keeps the last rows of its input for the next call, and every
   output sums its terms in one order whatever the frames per call, so
   decoding 1 + 3 frames or 4 at once gives the same samples. */
int q3h_codec_back(q3h_codec *c, const float *x, int frames, float *pcm);
int64_t q3h_codec_bytes(const q3h_codec *c);
int q3h_codec_destroy(q3h_codec *c);

/* ---- drafted continuations: a cache of its own, the rotary forms, attention
   over a tree of drafted rows, scores of given tokens (no reference
   counterpart; the reference decodes one token at a time over an f32 or f16
   cache) ----

   These four operators work on device memory of the caller, of the GPU of
   their handle, in the order of a stream of the caller (hipStream_t as void *;
   NULL: the default stream). They only enqueue kernels: no allocation, no
   copy, no wait, so they can be captured into a graph (a captured call's
   kernels hold the pointers it was given). The caller's current device is as
   it was when they return. Arguments that the host can see are checked
   (Q3H_E_ARG, Q3H_E_CAPACITY, nothing enqueued); what only the device holds
   (lengths, counts, parents, tokens) is checked there, and what is out of range
   never reads or writes outside the tensors: the rows concerned come out as
   NaN. Calls on one cache may run at once where none writes rows that another
   reads or writes.

   A call covers the first `sequences` sequences of a cache, each with `rows`
   drafted rows: tensors are [sequences][rows][...], row r of sequence b at row
   b * rows + r, rows ld* floats apart. lens [sequences]: the positions each
   sequence held before the draft; its row r goes to (is) position lens[b] + r
   of the cache. counts [sequences] (nullable: all rows): how many of the rows
   there are, taken into [0, rows]; the others are neither read nor written.
   parents [sequences][rows] (nullable): the row that row r continues, below r,
   or -1 for one that continues the sequence itself; for at most
   Q3H_TREE_MAX_ROWS rows. A row sees the positions before the draft, the rows on
   its path and itself, and its rotary position is lens[b] plus its depth.
   NULL: a chain, row r after row r - 1, of any length (a prompt, or one new
   token). */
#define Q3H_KV_F32 0
#define Q3H_KV_F16 1
/* a byte per element and one f32 scale per position and kv head: scale =
   max |x| / 127 rounded to f32, byte = x / scale rounded to even, both from 64
   bits. A row with an infinity or NaN reads as NaN. */
#define Q3H_KV_Q8 2
/* four bits per element, a step (a byte) per 32 of them and one f32 scale per position
   and kv head: scale = max |x| / 1785 rounded to f32 (1785 = 7 * 255), step = max |x| of
   the 32 / (7 scale) rounded up (255 at most), element = x / (step * scale) rounded to
   even within -7 .. 7, from 64 bits; it stands for element * step * scale. An element is
   off by at most 1/14 of the largest of its 32 plus 1/3570 of the row's largest, and by
   f32's roundings of the scale and the product beside that: 2^-23 of the row's largest, or
   2.6e-42 where that is more (a row under 1.2e-42 reads as zeros). A row, the key or the
   value of a position and kv head, takes head_dim / 2 + 8 bytes. A row with an infinity
   or NaN reads as NaN. */
#define Q3H_KV_Q4 4
#define Q3H_TREE_MAX_ROWS 64
#define Q3H_TOP_MAX 64

typedef struct q3h_rope q3h_rope;
typedef struct q3h_cache q3h_cache;

/* rotary positions: the first rot_dim elements of a head turn in pairs i by
   position * f(i), in 64 bits; f(i) = theta ^ (-2 i / rot_dim), then
   - Q3H_ROPE_PLAIN: as it is;
   - Q3H_ROPE_LINEAR: / factor;
   - Q3H_ROPE_YARN: / factor where a pair turns less than beta_slow times over
     original_positions, as it is where more than beta_fast times, in between a
     ramp over the pair number (its ends rounded outwards to whole pairs);
   - Q3H_ROPE_BANDS: / factor where a pair turns less than low_turns times over
     original_positions, as it is where more than high_turns times, in between
     mixed by its turns. */
#define Q3H_ROPE_PLAIN 0
#define Q3H_ROPE_LINEAR 1
#define Q3H_ROPE_YARN 2
#define Q3H_ROPE_BANDS 3
typedef struct {
  int32_t head_dim;      /* 64 or 128 */
  int32_t rot_dim;       /* even, 2 .. head_dim; the other elements stay */
  int32_t interleaved;   /* pair i: elements 2i, 2i + 1; 0: i, i + rot_dim / 2 */
  int32_t max_positions; /* positions of the table (16 bytes a pair each) */
  float theta;
  int32_t scaling;            /* Q3H_ROPE_* */
  float factor;               /* all but PLAIN: > 0 */
  int32_t original_positions; /* YARN, BANDS: > 0 */
  float beta_fast, beta_slow; /* YARN: beta_fast > beta_slow > 0 */
  float low_turns, high_turns; /* BANDS: high_turns > low_turns > 0 */
  float magnitude; /* on cosine and sine; 0: 0.1 ln(factor) + 1 for YARN with a
                      factor above 1, else 1 */
} q3h_rope_config;
int q3h_rope_create(q3h_device *dev, const q3h_rope_config *cfg, q3h_rope **out);
/* a table whose pairs turn by positions of several axes (time, height and width of a
   picture's patches), 1 to 4: pair i by that of axis pair_axes[i], pair_axes
   [rot_dim / 2] in host memory. Rows get their positions in q3h_cache_append_at; in
   q3h_cache_append all axes have the row's own. */
int q3h_rope_create_axes(q3h_device *dev, const q3h_rope_config *cfg, int axes,
                         const int32_t *pair_axes, q3h_rope **out);
int q3h_rope_destroy(q3h_rope *r);

/* a K/V cache of several sequences: per sequence keys, then values
   [layers][kv_heads][max_positions][head_dim] in the format (Q3H_KV_*), the
   layout of a context's cache, then for Q3H_KV_Q8 and Q3H_KV_Q4 the scales of the keys and
   of the values [layers][kv_heads][max_positions], then for Q3H_KV_Q4 their steps, four
   bytes each; zeros at first */
typedef struct {
  int32_t sequences, layers, kv_heads, head_dim; /* head_dim 64 or 128 */
  int32_t max_positions, format;
} q3h_cache_config;
int q3h_cache_create(q3h_device *dev, const q3h_cache_config *cfg, q3h_cache **out);
/* a cache whose sequences are made of pages: max_positions of each sequence at most, in
   `pages` pages of page_positions positions (all layers, keys and values) that sequences
   take and may share. Which pages a sequence has is kept on the device; all calls on
   caches take it as any other, a sequence's positions being those that its pages reach
   (none at first), and rows that would go to a page that another sequence holds too
   get NaN queries and are not written. */
#define Q3H_MAX_PAGES (1 << 20)
typedef struct {
  q3h_cache_config cache; /* of all sequences up to 2^24 pages, if all were full */
  int32_t pages;          /* 1 .. Q3H_MAX_PAGES */
  int32_t page_positions; /* 32, 64, 128 or 256 */
} q3h_paged_config;
int q3h_cache_create_paged(q3h_device *dev, const q3h_paged_config *cfg, q3h_cache **out);
int64_t q3h_cache_bytes(const q3h_cache *c);
int q3h_cache_destroy(q3h_cache *c);

/* The drafted rows' keys and values into the cache: k and v [..][kv_heads]
   [head_dim], and with heads > 0 the queries q [..][heads][head_dim] to q_out.
   Queries and keys are RMS-normed over the head (q_norm, k_norm [head_dim],
   nullable: not normed) and turned (rope, nullable: not turned; its
   max_positions not below the cache's), in 64 bits and rounded once to f32;
   then k and v are rounded to the format. q_out may be q itself (the same
   pointer and row distance) and overlap nothing else. A sequence whose rows
   would pass its positions, or of negative length, gets no rows and NaN queries,
   and so does a row on whose path a parent is not below its row. */
typedef struct {
  int32_t layer, sequences, rows, heads;
  const float *q, *k, *v;
  int64_t ldq, ldk, ldv;
  float *q_out;
  int64_t ld_out;
  const float *q_norm, *k_norm;
  float eps;
  const q3h_rope *rope;
  const int32_t *lens, *counts, *parents;
} q3h_append_args;
int q3h_cache_append(q3h_cache *c, const q3h_append_args *a, void *stream);

/* q3h_cache_append with positions [axes of the rope][sequences][rows] (device memory) of
   the rows in place of lens[b] plus depth, which the angles are taken from; the rope is
   needed. A row with a position outside the rope's table gets NaN queries and is not
   written. Where the rows go in the cache stays as it is. */
int q3h_cache_append_at(q3h_cache *c, const q3h_append_args *a, const int32_t *positions,
                        void *stream);

/* positions starts[b] .. + counts[b] - 1 of a layer (starts nullable: 0) as
   the f32 values that the cache holds: k and v (either nullable)
   [sequences][rows][kv_heads][head_dim], contiguous */
int q3h_cache_read(q3h_cache *c, int layer, int sequences, int rows, const int32_t *starts,
                   const int32_t *counts, float *k, float *v, void *stream);

/* out = softmax(scale q . K + mask) V for the drafted rows, whose keys and
   values the cache holds already (q3h_cache_append): q and out
   [..][heads][head_dim], heads a multiple of kv_heads, query head h on kv head
   h / (heads / kv_heads). max_len: no length in lens is above it (the host's
   bound, it sizes the launch; a longer or negative one: NaN rows). scale: 0 for
   1 / sqrt(head_dim). Products and sums keep f32's precision in every format;
   over f16, int8 and 4-bit caches that is relative to the row's largest element (an
   element to which only positions of a weight near 2^-24 add is less exact), and
   an f16 cache's elements below 2^-14 count to 2^-38.
   Infinities and NaN at positions a row does not see do not reach it. workspace:
   q3h_cache_attend_workspace bytes for the same sequences, rows, heads and max_len
   (of the caller, 256-byte aligned, one for each call that may run at once;
   nullable where that is 0). out may be q itself. */
typedef struct {
  int32_t layer, sequences, rows, heads, max_len;
  float scale;
  const float *q;
  int64_t ldq;
  float *out;
  int64_t ld_out;
  const int32_t *lens, *counts, *parents;
  void *workspace;
  int64_t workspace_bytes;
} q3h_attend_args;
/* negative: a Q3H_E* code */
int64_t q3h_cache_attend_workspace(const q3h_cache *c, int sequences, int rows, int heads,
                                   int max_len);
int q3h_cache_attend(q3h_cache *c, const q3h_attend_args *a, void *stream);

/* The drafted rows that are kept, moved to the front: kept [sequences][rows]
   holds kept_counts[b] row numbers, each above the one before (a path from a
   root down); row kept[b][i], at position lens[b] + kept[b][i], goes to
   position lens[b] + i, in every layer. The caller's lengths grow by
   kept_counts. A list that is not of that form leaves its sequence as it is, and so
   does one whose rows would go to a page that another sequence holds too. */
int q3h_cache_keep(q3h_cache *c, int sequences, int rows, const int32_t *lens,
                   const int32_t *kept, const int32_t *kept_counts, void *stream);

/* The pages of a cache of q3h_cache_create_paged, for its first `sequences` sequences. Like
   the operators above these calls only enqueue kernels, on any stream, and can be
   captured (the order in which they run is the caller's to keep, also of two graphs);
   but they change what the cache's other calls read, and share scratch memory
   of the cache: of one cache they run one after another, and not beside a call on
   its rows. Pages are taken from the lowest free one up, for the sequences in their
   order, so that the same calls leave the same tables. What only the device holds and is
   out of range (a negative length, a length beyond a sequence's pages or positions, no
   such source) leaves its sequence as it is.

   reserve: room for rows to come: sequence b gets the pages that positions lens[b] ..
   lens[b] + counts[b] - 1 (counts nullable: rows; taken into [0, rows]) lie in and it
   does not have; lens[b] at most the positions that its pages reach. Pages of that range
   that other sequences hold too are replaced by its own, the positions before lens[b]
   copied; if all that hold such a page write to it in this call, the first of them keeps
   it. ok [sequences] (nullable): 1 where a sequence has all those pages, to itself; 0
   where there were too few (then it, and the ones behind it that want some, get
   none) or its arguments are out of range. */
int q3h_cache_reserve(q3h_cache *c, int sequences, int rows, const int32_t *lens,
                      const int32_t *counts, int32_t *ok, void *stream);
/* fork: sequence b becomes the first lens[b] positions of what sequence sources[b] of the
   cache was before the call (-1: nothing), for all b at once, so that sources may be any
   assignment (beams that are continued, dropped, reordered). Pages are shared, nothing is
   copied; what b held before and no sequence holds any more is free. */
int q3h_cache_fork(q3h_cache *c, int sequences, const int32_t *sources, const int32_t *lens,
                   void *stream);
/* release: sequence b keeps the pages that its first lens[b] positions lie in (0: none) */
int q3h_cache_release(q3h_cache *c, int sequences, const int32_t *lens, void *stream);
/* compact: the pages in use become pages 0 .. *used - 1 (used: device memory, nullable),
   with what they hold: those behind that number go, in their order, to the free ones
   below it, in theirs. */
int q3h_cache_compact(q3h_cache *c, int32_t *used, void *stream);
/* copy: positions 0 .. lens[b] - 1 of every layer of sequence sources[b] of src (-1: none)
   to sequence b of c. Two caches of one device, format, layers, kv heads and head_dim,
   each in pages or not (a sequence moved out and back, a prompt computed elsewhere);
   sequence b has the positions already. Pages of c that other sequences hold too stay as
   they are. */
int q3h_cache_copy(q3h_cache *c, const q3h_cache *src, int sequences, const int32_t *sources,
                   const int32_t *lens, void *stream);
/* the tables as they are, each nullable: table [sequences of the cache]
   [ceil(max_positions / page_positions)] (-1: no page), counts [sequences] of pages that a
   sequence holds, refs [pages] of sequences that hold a page */
int q3h_cache_page_state(const q3h_cache *c, int32_t *table, int32_t *counts, int32_t *refs,
                         void *stream);

/* Scores of rows of logits [rows][vocab] (dtype Q3H_F32 or Q3H_BF16, rows ld
   elements apart, at most 2^20 tokens; fewer than 2^24 rows, of more than 10233
   tokens each 10240 of them count as one), computed in f32 from one read of them:
   with lse = log sum exp of a row,
   - logprobs [rows][tokens_per_row]: logit - lse of the given tokens (tokens
     [rows][tokens_per_row]; a token outside [0, vocab): NaN);
   - entropy [rows] (nullable): lse - sum p logit, logits of -infinity adding
     nothing;
   - top_ids, top_logprobs [rows][top_k] (top_k 0: none; at most Q3H_TOP_MAX and
     vocab): the largest logits from the top, of equal ones the lowest token
     first, NaN last.
   A row with a NaN or +infinity, or of -infinity alone, has NaN scores.
   workspace: q3h_token_logprobs_workspace bytes for the same rows, vocab and
   top_k, as q3h_cache_attend's. */
typedef struct {
  const void *logits;
  int64_t ld;
  int32_t dtype, rows, vocab;
  int32_t tokens_per_row, top_k;
  const int32_t *tokens;
  float *logprobs, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
  void *workspace;
  int64_t workspace_bytes;
} q3h_score_args;
int64_t q3h_token_logprobs_workspace(int rows, int vocab, int top_k);
int q3h_token_logprobs(q3h_device *dev, const q3h_score_args *a, void *stream);

/* The same operators on a context, whose rows go through the stack's layers;
   all pointers are host memory, the calls block as q3h_forward_embeds does. */

/* other rotary positions than the whole head's unscaled halves, for every
   context of a stack with f32 activations: before the first context or frame
   (Q3H_E_STATE); head_dim and max_positions as the stack's. rope_theta of the
   stack's configuration is not used then. Contexts of such a stack, and of one
   with an int8 or 4-bit cache, take the same calls as any other (prompts of
   q3h_frame_start_batch each by itself; not q3h_context_time_attention). */
int q3h_stack_set_rope(q3h_stack *s, const q3h_rope_config *cfg);

/* scores of every row of a forward, as q3h_token_logprobs gives them; entropy
   nullable, tokens and logprobs [rows][tokens_per_row] */
typedef struct {
  int32_t tokens_per_row, top_k;
  const int32_t *tokens;
  float *logprobs, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
} q3h_row_scores;

/* A tree of drafted rows: x [rows][hidden], at most Q3H_TREE_MAX_ROWS, row r
   after row parents[r] (below r; -1: after the context's last position). Every
   row's logits [rows][head rows], normed state [rows][hidden] and scores
   (each nullable; scores need a head). The context's length stays; the rows
   wait behind it for q3h_context_keep, until another call writes to the
   context. f32 activations. rows <= 0 does nothing. */
int q3h_forward_tree(q3h_context *c, const float *x, int rows, const int32_t *parents, int head,
                     const q3h_row_scores *scores, float *logits, float *normed);
/* The rows kept [n] of the last q3h_forward_tree, a path from a root down (each
   row the parent of the next), become the context's next n positions; the
   others are dropped (n 0: all). Q3H_E_STATE when there is no tree. */
int q3h_context_keep(q3h_context *c, const int32_t *kept, int n);
/* q3h_forward_embeds of rows whose every position is scored, the logits (of
   every row, nullable) staying on the device otherwise; normed [rows][hidden]
   nullable. Any stack. As in every forward with a head, the context's buffers hold
   rows x head rows logits (f32) from then on. */
int q3h_forward_score(q3h_context *c, const float *x, int rows, int head,
                      const q3h_row_scores *scores, float *logits, float *normed);

/* ---- helpers ---- */

/* ggml quantize_row_q8_0_ref (InferQuantizeRowQ8_0Ref, lm.pas:265-267) on the
   host: k % 32 == 0, y receives k/32 blocks of 34 bytes */
int q3h_quantize_row_q8_0(const float *x, void *y, int64_t k);

/* no reference counterpart (measurement): the weight products of one
   single-row decode step of stack s - per layer the fused q/k/v, o, gate/up
   and down matrix-vector products, then head `head` (-1: none) - run iters
   times on one stream. mode 0: launched directly, us_per_launch = wall time
   between two hipEvents / launches; mode 1: captured in a hipGraph and
   replayed, same wall-time measure; mode 2: every launch carries its own
   start / end events (hipExtLaunchKernelGGL), us_per_launch = the average
   execution time of the kernels themselves (Q8_0 stacks). launches: products
   per step; bytes: algorithmic bytes per step (weights, norm vectors, input
   and output vectors). The activations are zeros; contexts are untouched. */
int q3h_stack_time_gemv(q3h_stack *s, int head, int iters, int mode, float *us_per_launch,
                        int *launches, int64_t *bytes);

#ifdef __cplusplus
}
#endif
#endif
