/*
 * mrtdf.h - C ABI of the B200 Depthformer decoding engine.
 *
 * This is the drop-in boundary for the per-chunk hot path of the C++ Magenta
 * RealTime reimplementation (rhymeswithlion/magenta-realtime-mlx-cpp). Each
 * entry point names the reference interface it replaces (file:line inside that
 * project). All arguments are plain C types: host pointers unless the name
 * ends in `_dev`, sizes as int, status as int (0 = MRTDF_OK). On failure the
 * thread-local message from mrtdf_last_error() says what went wrong; the
 * reference throws C++ exceptions in the same places.
 *
 * Threading: a handle may be used by one host thread at a time. Different
 * mrtdf_stream handles of one engine may be driven from different threads.
 */
#ifndef MRTDF_H_
#define MRTDF_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes -------------------------------------------------------- */
#define MRTDF_OK 0
#define MRTDF_ERR_INVALID 1 /* bad argument or shape (std::runtime_error in the reference) */
#define MRTDF_ERR_CUDA 2    /* a CUDA runtime call failed */
#define MRTDF_ERR_IO 3      /* file missing or malformed safetensors */
#define MRTDF_ERR_STATE 4   /* call order: e.g. temporal_step before encode */
#define MRTDF_ERR_KEY 5     /* weight key missing (std::out_of_range, weights.cpp:40-41) */
#define MRTDF_ERR_TIMEOUT 6 /* a device-side bounded wait gave up */
#define MRTDF_ERR_RANGE 7   /* index past a maximum (std::out_of_range, model.cpp:216-218) */

#define MRTDF_DTYPE_FP32 0
#define MRTDF_DTYPE_BF16 1

/*
 * Model hyperparameters. Mirrors DepthformerConfig (depthformer/model.h:47-68)
 * plus the vocabulary layout constants of SystemConfig (system.h:51-82) that
 * the decode loop needs, and the compute dtype (parse_dtype, dtype.h:36).
 */
typedef struct mrtdf_config {
  int vocab_size;
  int d_model;
  int d_kv;
  int d_ff;
  int num_heads;
  int num_encoder_layers;
  int num_temporal_layers;
  int num_depth_layers;
  int max_encoder_length;
  int rvq_depth;
  int temporal_num_buckets;
  int temporal_max_distance;
  int depth_num_buckets;
  int depth_max_distance;
  int codebook_size;  /* codec_rvq_codebook_size (system.h:51) */
  int codec_offset;   /* vocab_codec_offset = PAD + MASK (system.h:76) */
  int max_frames;     /* temporal self-KV capacity = chunk_length_frames (system.h:62-64) */
  int dtype;          /* MRTDF_DTYPE_FP32 or MRTDF_DTYPE_BF16 */
} mrtdf_config;

/*
 * Options of one generate_tokens call. Mirrors GenerateOptions
 * (depthformer/decode.h:48-57). The reference seeds MLX's RNG once per chunk
 * (decode.cpp:246-248); this engine draws its uniforms from Philox4x32-10
 * keyed by `seed`, counter = (vocab index / 4, frame * rvq_depth + level), so
 * two runs with the same seed give the same tokens. `use_vocab_masks` = 1
 * applies the per-level codec ranges that System::build_vocab_masks builds
 * (system.cpp:135-157). `uniforms`, when not NULL, replaces the RNG with
 * caller-given draws: num_frames * rvq_depth * vocab_size floats in (0, 1),
 * one row of vocab_size per (frame, level) step.
 */
typedef struct mrtdf_gen_opts {
  int num_frames;
  int rvq_depth;
  float temperature;
  int top_k;
  float guidance_weight;
  int use_vocab_masks;
  uint64_t seed;
  const float* uniforms;
} mrtdf_gen_opts;

typedef struct mrtdf_engine mrtdf_engine;
typedef struct mrtdf_stream mrtdf_stream;

/* Thread-local text of the last error; never NULL. */
const char* mrtdf_last_error(void);

/* Library version string, e.g. "mrtdf 0.1.0 sm_100a". */
const char* mrtdf_version(void);

/*
 * Fill `out` with a named preset: "base" (DepthformerConfig::base(),
 * model.cpp:34-36), "large" (model.cpp:38-48), "hybrid" (d_model 1024, 16x64
 * heads, d_ff 2816, layers 12/20/4, temporal buckets 32/128, vocab 16388) or
 * "tiny" (a small test model). dtype defaults to bf16.
 */
int mrtdf_config_preset(const char* name, mrtdf_config* out);

/*
 * Write a random-init weight bundle with the reference's key names and
 * (out, in) Linear layout (model.cpp:82-109, 173-198; modules.cpp:47-54) as
 * float32 safetensors. Matrices and tables are N(0, stddev) from Philox
 * keyed by `seed`; RMSNorm scales are 1.0 when `norm_ones` != 0, otherwise
 * N(0, stddev) too. The reference has no generator (weights.cpp:29-35 only
 * loads), so this defines one.
 */
int mrtdf_write_random_safetensors(const mrtdf_config* cfg, uint64_t seed, float stddev,
                                   int norm_ones, const char* path);

/* Replaces Depthformer::Depthformer(bundle, config, dtype) (model.h:74-75). */
int mrtdf_create(const mrtdf_config* cfg, int device, mrtdf_engine** out);
int mrtdf_destroy(mrtdf_engine* eng);

/* Load weights from a safetensors bundle: WeightBundle (weights.cpp:29-35)
 * plus load_param's cast to the compute dtype (modules.cpp:47-54). */
int mrtdf_load_safetensors(mrtdf_engine* eng, const char* path);

/* Generate the same weights as mrtdf_write_random_safetensors in memory and
 * upload them, without a file. */
int mrtdf_load_random(mrtdf_engine* eng, uint64_t seed, float stddev, int norm_ones);

/*
 * A decoding stream: `num_sequences` independent sequences, each one CFG pair
 * (2 rows, cond + uncond) when `cfg` != 0, else 1 row. Owns the KV arena
 * (empty_temporal_cache / empty_depth_cache, model.h:103-104; LayerCache,
 * model.h:70): temporal self K/V at max_frames, cross K/V at
 * max_encoder_length, depth self K/V at rvq_depth, all (rows, H, T, d_kv).
 */
int mrtdf_stream_create(mrtdf_engine* eng, int num_sequences, int cfg, mrtdf_stream** out);
int mrtdf_stream_destroy(mrtdf_stream* st);
/* Rows per step of this stream (num_sequences * (cfg ? 2 : 1)). */
int mrtdf_stream_rows(const mrtdf_stream* st);

/*
 * Depthformer::encode (model.h:81, model.cpp:226-241). `ids` is
 * (rows, seq_len) int32. Also projects the cross-attention K/V of every
 * temporal layer (modules.cpp:258-276, 323-333), which the reference does
 * on frame 0 of temporal_step; this resets the temporal cache. `enc_out`,
 * if not NULL, receives (rows, seq_len, d_model) float32.
 */
int mrtdf_encode(mrtdf_stream* st, const int32_t* ids, int seq_len, float* enc_out);

/*
 * Depthformer::temporal_step (model.h:113-117, model.cpp:322-514, eager
 * semantics). `x` is (rows, d_model) float32, rounded to the compute dtype
 * on upload; NULL means token_embedding(PAD=0) as on frame 0
 * (decode.cpp:366-368). Appends to the temporal self-KV at position
 * `frame_idx`, which must equal the number of frames already decoded
 * (frame 0 resets). `out` receives the stack output (rows, d_model) with no
 * final norm.
 */
int mrtdf_temporal_step(mrtdf_stream* st, const float* x, int frame_idx, float* out);

/*
 * Depthformer::depth_step (model.h:121-124, model.cpp:516-659). `x` is
 * (rows, d_model) float32; NULL means the last temporal_step output
 * (decode.cpp:455). depth_idx 0 resets the depth cache (decode.cpp:454).
 * `logits` receives (rows, vocab_size) float32.
 */
int mrtdf_depth_step(mrtdf_stream* st, const float* x, int depth_idx, float* logits);

/* token_embedding()(ids) (model.h:127; modules.cpp:110-112): n rows of d_model. */
int mrtdf_token_embedding(mrtdf_engine* eng, const int32_t* ids, int n, float* out);

/*
 * cfg_combine + apply_vocab_mask + sample_with_temperature
 * (decode.cpp:71-148, 465-474) on the device for one step. `logits` is
 * (cfg ? 2 : 1, vocab_size); `level` selects the vocab mask when
 * opts->use_vocab_masks; `uniforms` (vocab_size floats in (0, 1)) replaces
 * the Philox draws when not NULL, otherwise the draws for (frame, level)
 * of opts->seed are used. MRTDF_ERR_INVALID when no candidate can be drawn
 * (NaN logits, an empty range); `token` is then -1.
 */
int mrtdf_sample(mrtdf_engine* eng, const float* logits, int cfg, int frame, int level,
                 const mrtdf_gen_opts* opts, const float* uniforms, int32_t* token);

/*
 * mrtdf_sample for callers that cannot allocate GPU memory. No counterpart
 * in the reference: it exists for hosts that must not call cudaMalloc /
 * cudaFree on their decode thread - a real-time audio callback, where the
 * implicit device synchronisation and unbounded latency of an allocation
 * would glitch playback, or an embedding application that reserves all GPU
 * memory up front and forbids allocations afterwards.
 *
 * Same semantics and result as mrtdf_sample, but `logits_dev` ((cfg ? 2 : 1)
 * x vocab_size float32), `uniforms_dev` (vocab_size floats, or NULL for the
 * Philox draws of opts->seed) and `token_dev` (one int32) are DEVICE
 * pointers owned by the caller, the work is queued on `stream` (a
 * cudaStream_t, NULL = the legacy default stream) and the call does not
 * wait for it: it queues one kernel launch and nothing else (the seed
 * travels by value). Because the call returns before the draw, a draw that
 * fails (NaN logits, an empty range) is reported in the result: the kernel
 * stores -1 in *token_dev. The sampler's scratch is a fixed 64 KiB device
 * array inside the library, held by every GPU that loads it until the
 * process exits: rows x d_model x dtype bytes must be <= 21,760
 * (MRTDF_ERR_RANGE otherwise); nothing in it needs to start at zero, each
 * call writes what its kernel reads. The first call on a device looks up
 * that array's address; make it before any stream capture. All calls on a
 * device share the scratch, so calls that may overlap on the GPU race;
 * serialise them (one stream). Allocates nothing: no cudaMalloc, cudaFree
 * or allocating library routine.
 */
int mrtdf_sample_noalloc(mrtdf_engine* eng, const float* logits_dev, int cfg, int frame, int level,
                         const mrtdf_gen_opts* opts, const float* uniforms_dev, int32_t* token_dev, void* stream);

/*
 * generate_tokens (decode.h:112-119, decode.cpp:239-573; non-speculative
 * path): encode + num_frames x (temporal_step + rvq_depth x (depth_step +
 * sample)) entirely on the device. `enc_ids` is (rows, seq_len) int32;
 * `out_ids` receives (num_sequences, num_frames, rvq_depth) int32 LLM ids.
 * `seeds` holds one seed per sequence (NULL: opts->seed + sequence index).
 * The whole chunk runs as one CUDA graph, captured on first use.
 */
int mrtdf_generate_tokens(mrtdf_stream* st, const int32_t* enc_ids, int seq_len,
                          const mrtdf_gen_opts* opts, const uint64_t* seeds, int32_t* out_ids);

/* Same with device-resident ids in and out; runs on the stream's CUDA stream
 * and does not synchronize. */
int mrtdf_generate_tokens_dev(mrtdf_stream* st, const int32_t* enc_ids_dev, int seq_len,
                              const mrtdf_gen_opts* opts, const uint64_t* seeds,
                              int32_t* out_ids_dev);

/*
 * Teacher-forced decode: the generate_tokens loop with the sampled token of
 * (frame f, level l) replaced by tokens[f * rvq_depth + l], returning every
 * depth step's logits: (num_frames, rvq_depth, rows, vocab_size) float32.
 * Single-sequence streams only.
 */
int mrtdf_teacher_forced_logits(mrtdf_stream* st, const int32_t* enc_ids, int seq_len,
                                const int32_t* tokens, int num_frames, float* logits);

/* Wait for all work queued on the stream; returns MRTDF_ERR_TIMEOUT if a
 * device-side bounded wait gave up since the last call. */
int mrtdf_stream_sync(mrtdf_stream* st);

/* The stream's cudaStream_t, for callers that order their own work on it. */
void* mrtdf_stream_cuda(mrtdf_stream* st);

/*
 * Failure-detection check (no counterpart in the reference): queue on the
 * stream one CTA that waits on an mbarrier which no thread and no copy ever
 * completes, bounded by `timeout_us` microseconds of the GPU's global timer
 * (1 .. 1,000,000; every production wait uses the same routine with a
 * 0.5 s bound). The wait gives up, sets the timeout bit of the stream's error
 * word and the call returns MRTDF_ERR_TIMEOUT, as every call does after a
 * device-side wait gave up; the error word is cleared and the stream stays
 * usable.
 */
int mrtdf_check_wait_timeout(mrtdf_stream* st, int timeout_us);

/*
 * Measurement hook (no reference counterpart): replay, as one CUDA graph on
 * the stream, only the weight-streaming decode launches of one
 * generate_tokens chunk with options `opts` (same buffers and parameters as
 * the real chunk; encoder and sampler left out) of the stacks in
 * `stack_mask` (bit 0: the temporal layers, bit 1: the depth layers and
 * lm_head), `reps` times between two CUDA events. Returns the milliseconds
 * per replay, the launches per replay and their algorithmic bytes (weights,
 * attention K/V reads, input and output vectors). The stream must have run
 * a chunk or an encode before.
 */
int mrtdf_bench_phases(mrtdf_stream* st, const mrtdf_gen_opts* opts, int stack_mask, int reps, float* ms_per_rep,
                       long long* launches_per_rep, double* bytes_per_rep);

/*
 * Measurement hook (no reference counterpart): read a `bytes` device buffer
 * (rounded down to a multiple of 16 MiB) `reps` times with 16-byte loads
 * spread over every SM, after one untimed pass; a buffer well under the L2
 * size stays L2-resident, so this is the L2 read bandwidth the depth stack
 * can reach. Reports GB/s (bytes read / CUDA-event time).
 */
int mrtdf_bench_l2_read(mrtdf_engine* eng, size_t bytes, int reps, double* gbs);

/*
 * Measurement hook (no counterpart in the reference): the encoder pass
 * (embed + PE, encoder layers, encoder_norm, cross-K/V projection of every
 * temporal layer) for `rows` sequences of `seq_len` uniform-random ids
 * (seed 2), captured as one CUDA graph and replayed `reps` times on a
 * private stream. Reports ms per pass and the pass's algorithmic FLOPs
 * (2 per multiply-add: linears, attention, cross-K/V). Allocates its own
 * workspace (rows x seq_len activations + the cross-K/V cache) for the call.
 */
int mrtdf_bench_encoder(mrtdf_engine* eng, int rows, int seq_len, int reps, float* ms_per_rep,
                        double* flops_per_rep);

/*
 * Measurement hook (no counterpart in the reference): `frames` x rvq_depth
 * sequential depth steps (depth stack + decoder_norm + lm_head level slice
 * + sampler with embedding feedback), each frame starting from an N(0, 1)
 * temporal hidden state (seed 3) instead of a temporal step, captured as one
 * graph and replayed `reps` times on the stream. Reports us per depth step,
 * its algorithmic bytes (GEMV weights, inputs, outputs and the depth K/V
 * reads) and kernel launches per step. Overwrites the stream's depth cache,
 * token and feedback buffers.
 */
int mrtdf_bench_depth(mrtdf_stream* st, const mrtdf_gen_opts* opts, int frames, int reps, float* us_per_step,
                      double* bytes_per_step, long long* launches_per_step);

/*
 * Measurement hook (no counterpart in the reference): kernel nodes of the
 * CUDA graph of the chunk this stream ran last (every one is a kernel of this
 * library), or -1 when that chunk ran as stream launches (MRTDF_GRAPH=0).
 */
long long mrtdf_stream_chunk_kernels(const mrtdf_stream* st);

/* ---- single-layer probes ----------------------------------------------------
 * No counterpart in the reference: each runs ONE step of the production
 * launch sequence (the same kernels, launch shapes and epilogues as a chunk)
 * on caller-given float32 inputs, rounded to the compute dtype on upload, so
 * a CPU restatement can be checked layer by layer on identical inputs. They
 * use and overwrite the stream's activation and cache buffers.
 */

/* EncoderLayer `layer` (modules.cpp:349-358) over x (rows, seq_len,
 * d_model) -> out, same shape. */
int mrtdf_probe_encoder_layer(mrtdf_stream* st, int layer, const float* x, int seq_len, float* out);

/* Overwrite positions [0, len) of one layer's cache with (rows, H, len,
 * d_kv) float32 k / v: kind 0 = temporal self-attention, 1 = depth
 * self-attention, 2 = cross-attention (len = the encoder length the
 * temporal layers then attend over). */
int mrtdf_probe_set_cache(mrtdf_stream* st, int kind, int layer, const float* k, const float* v, int len);

/* DecoderLayer::forward (modules.cpp:384-446) of the temporal (stack 0) or
 * depth (stack 1) stack at cache position `pos`: x (rows, d_model) -> out;
 * the step's k / v are appended to the layer's cache at `pos`. */
int mrtdf_probe_decoder_layer(mrtdf_stream* st, int stack, int layer, int pos, const float* x, float* out);

/* decoder_norm + lm_head (model.cpp:653-658) of x (rows, d_model): the
 * codebook rows of RVQ level `level` (rows x codebook_size logits), or all
 * vocab_size rows when level < 0. */
int mrtdf_probe_lm_head(mrtdf_stream* st, int level, const float* x, float* logits);

/* ---- streaming glue (System, system.cpp) ---------------------------------- */

/*
 * The System::generate_chunk loop (system.cpp:177-333) for `num_chunks`
 * consecutive chunks without returning to the host: per chunk, encoder ids
 * from the context (build_encoder_inputs_host, system.cpp:62-95), the chunk
 * (generate_tokens), tokens -> RVQ codes (llm_to_rvq, rvq.cpp:112-134) and
 * the context roll (system.cpp:320-333), all on the stream.
 * context_dev: (num_sequences, ctx_frames, rvq_depth) int32 RVQ codes,
 * negative = empty, rolled in place; style_dev: (num_sequences,
 * style_depth) int32 LLM ids; rvq_out_dev: (num_chunks, num_sequences,
 * num_frames, rvq_depth) int32 codes. seeds: host (num_chunks *
 * num_sequences) or NULL (opts->seed + chunk, + i << 32 for sequence i).
 * Returns once the work is queued; mrtdf_stream_sync waits and reports
 * device errors (a token outside its level's range: MRTDF_ERR_INVALID).
 */
int mrtdf_generate_stream_dev(mrtdf_stream* st, int32_t* context_dev, int ctx_frames, int enc_depth,
                              const int32_t* style_dev, int style_depth, int num_chunks,
                              const mrtdf_gen_opts* opts, const uint64_t* seeds, int32_t* rvq_out_dev);

/*
 * build_encoder_inputs_host (system.cpp:62-95): context (ctx_frames,
 * rvq_depth) int32 RVQ codes (negative = empty) + style ids ->
 * (2, ctx_frames * enc_depth + style_depth) int32. Row 0 = codec context
 * levels < enc_depth mapped to codec_offset + d * codebook + v (MASK=1 when
 * v < 0) then the style ids; row 1 = same context, style masked.
 */
int mrtdf_build_encoder_inputs(const int32_t* context, int ctx_frames, int rvq_depth,
                               int enc_depth, const int32_t* style, int style_depth,
                               int codebook_size, int codec_offset, int32_t* out);

/* Context roll (system.cpp:320-333): shift left by chunk_frames frames and
 * append new RVQ codes (chunk_frames, rvq_depth). In place. */
int mrtdf_context_roll(int32_t* context, int ctx_frames, int rvq_depth, const int32_t* new_codes,
                       int chunk_frames);

/* llm_to_rvq with safe=true (rvq.cpp:112-134): (n, rvq_depth) LLM ids ->
 * RVQ codes; MRTDF_ERR_INVALID when an id is not in its level's range. */
int mrtdf_llm_to_rvq(const int32_t* llm, int n, int rvq_depth, int codebook_size,
                     int codec_offset, int32_t* out);

/* rvq_to_llm (rvq.cpp:105-110). */
int mrtdf_rvq_to_llm(const int32_t* rvq, int n, int rvq_depth, int codebook_size,
                     int codec_offset, int32_t* out);

/* Paths of the C++ inference bundle under one cache root (InferenceBundlePaths,
 * weights.h:70-78). Each is a NUL-terminated path of at most MRTDF_PATH_MAX - 1 bytes. */
#define MRTDF_PATH_MAX 4096
typedef struct mrtdf_bundle_paths {
  char spectrostream_encoder[MRTDF_PATH_MAX];
  char spectrostream_decoder[MRTDF_PATH_MAX];
  char spectrostream_codebooks[MRTDF_PATH_MAX];
  char musiccoca_encoder[MRTDF_PATH_MAX];
  char musiccoca_codebooks[MRTDF_PATH_MAX];
  char musiccoca_vocab[MRTDF_PATH_MAX];
  char depthformer[MRTDF_PATH_MAX]; /* <root>/depthformer/depthformer_<tag>.safetensors */
} mrtdf_bundle_paths;

/* resolve_inference_bundle (weights.cpp:72-120): the bundle's file paths
 * under `cache_root` for the Depthformer checkpoint `tag` ("base", "large").
 * A root that is not a directory, or any of the seven files missing, is
 * MRTDF_ERR_IO (std::runtime_error in the reference) with the reference's
 * message (the missing files listed one per line). A path longer than
 * MRTDF_PATH_MAX - 1 bytes is MRTDF_ERR_RANGE. No GPU is needed. */
int mrtdf_resolve_inference_bundle(const char* cache_root, const char* tag, mrtdf_bundle_paths* out);

/* ---- operators ---------------------------------------------------------------
 * Operators of speculative and long-running decoding, on device buffers that
 * the caller owns. No counterpart in the reference, whose speculative path
 * (depthformer/decode.cpp:150-237) drafts one chain and re-attends with the
 * single-chain kernels. Each call checks its arguments on the host, queues its
 * kernels on `stream` (a cudaStream_t, NULL = the legacy default stream) of
 * `device` and returns without waiting. A kernel's own waits for its copies and
 * products are bounded (0.5 s); where one runs out the kernel ends all the same
 * and the result rows that it was working on are NaN. It allocates nothing, keeps nothing
 * between calls and may be captured into a CUDA graph; calls on different
 * streams or from different threads may overlap as long as no buffer that one
 * of them writes (workspaces included) is used by another. What a call writes
 * overlaps nothing else that it reads or writes, except where an operator says so
 * (drafted rows are not views of the cache's own rows; buffers of the same address
 * are refused). The caller's
 * current device is as before when a call returns. Nothing on the host sees
 * the values in device memory: what a kernel does with a length, a parent, a
 * path or a position that makes no sense is said with each operator, and none
 * of them makes it read or write outside the buffers.
 *
 * `struct_bytes` is sizeof() of the structure it is in; MRTDF_ERR_INVALID when
 * it is not (a caller compiled against another header).
 */

/* Rows of head_dim contiguous elements of the cache's dtype: row (l, b, h, n)
 * of layer, sequence, head and node starts at ptr + l * stride_l + b * stride_b
 * + h * stride_h + n * stride_n elements. Every row starts on a 16-byte
 * boundary; strides are not negative, and rows that are written do not overlap
 * (a zero stride is refused there; rows that are only read may share memory).
 * (The rows of a fused q|k|v projection are three such views of one buffer.) */
typedef struct mrtdf_rows {
  void* ptr;
  int64_t stride_l, stride_b, stride_h, stride_n;
} mrtdf_rows;

/* A KV cache: row (l, b, h, t) at l * stride_l + b * stride_b + h * stride_h +
 * t * stride_t elements in k and in v, t < capacity; 16-byte boundaries and
 * non-negative strides as above. At most 1024 sequences, layers and kv heads
 * and 2^24 rows (MRTDF_ERR_RANGE). lens[b] rows of sequence b are in use in
 * every layer and head; a sequence whose length is outside [0, capacity] is
 * passed over (each operator says what that means). pos[l][b][h][t], when not
 * NULL, is the position in the text of the token in that row; NULL means row t
 * holds position t. next_pos[b] is the position of the next token (NULL: lens[b]);
 * pos needs it. */
typedef struct mrtdf_cache {
  size_t struct_bytes;
  void* k;
  void* v;
  int64_t stride_l, stride_b, stride_h, stride_t;
  int32_t layers, batch, kv_heads, capacity, head_dim /* 64 or 128 */, dtype /* MRTDF_DTYPE_* */, device;
  const int32_t* lens;     /* (batch) */
  int32_t* pos;            /* (layers, batch, kv_heads, capacity) or NULL */
  const int32_t* next_pos; /* (batch) or NULL */
} mrtdf_cache;

/* The KV cache of a stream as an operator's cache: kind 0 temporal self, 1
 * depth self, 2 cross attention; one layer, or all of them when layer < 0.
 * `len`, if not NULL, receives the rows in use. lens, pos and next_pos of
 * `out` are NULL: the caller adds its own device arrays. The buffers belong to
 * the stream; work on them is ordered with the stream's own by using
 * mrtdf_stream_cuda(st). */
int mrtdf_stream_cache(mrtdf_stream* st, int kind, int layer, mrtdf_cache* out, int* len);

/*
 * Attention of a tree of drafted tokens over a cache. Node i of sequence b
 * hangs below node parents[b][i] < i, or below the last cached token (-1); a
 * node with any other parent, and every node below it, is absent (padding).
 * Query row (h, i) sees the cached rows t < lens[b] and the drafted rows of
 * its ancestors and itself:
 *   x = scale * q . k + rel_bias[h][clamp(next_pos[b] + depth(i) - position(row), 0, rel_len - 1)]
 *   out = sum softmax(x) v,   lse = ln sum exp x
 * where depth(i) counts i's ancestors and a drafted row's position is
 * next_pos[b] + its depth. `heads` query heads share kv_heads in order (head h
 * reads kv head h / (heads / kv_heads)). One node and parents NULL is a plain
 * decode step; parents NULL with more nodes is a chain. 1 <= nodes <= 64,
 * nodes * heads / kv_heads <= 1024. Scores, softmax statistics and sums are
 * float32; bf16 values meet weights of 16 bits (2^-17 relative; the result's own
 * rounding is 2^-9); float32 products use split tf32 operands
 * (2^-23 relative), finite inputs below 2^127 in rows that are seen. The rows of an absent node, and of
 * a sequence that is passed over, are zeros with lse = -inf; so is a row whose
 * every score is -inf. Values in rows that a query row does not see do not
 * reach it, NaN and infinities included. A NaN score makes its row NaN. A NaN or
 * an infinity among the values that a row sees stays in its column, which is then
 * not finite (NaN also for an infinity, if it is a cached one: the weights meet it
 * in parts of either sign). Results are the same from run to run: the same call
 * on the same device repeats bit for bit. How a long cache is cut over the GPU
 * depends on the capacity, the device and the lengths of all sequences, so a
 * sequence's float32 sums, and with them the last bits of out and lse, may
 * differ when its neighbours do.
 */
typedef struct mrtdf_tree_args {
  size_t struct_bytes;
  mrtdf_rows q;     /* (batch, heads, nodes) rows */
  mrtdf_rows k_new; /* (batch, kv_heads, nodes) rows, not in the cache yet */
  mrtdf_rows v_new;
  mrtdf_rows out; /* (batch, heads, nodes) rows */
  float* lse;     /* (batch, heads, nodes) or NULL */
  const int32_t* parents;  /* (batch, nodes) or NULL */
  const float* rel_bias;   /* (heads, rel_len) or NULL */
  void* workspace;         /* mrtdf_tree_attention_workspace bytes, 16-byte aligned; contents do not matter */
  size_t workspace_bytes;
  int32_t heads, nodes, rel_len;
  float scale; /* 1.0 for the T5 attention of this engine */
} mrtdf_tree_args;

/* Workspace of a call with these sizes (0: none). Depends on the sizes and the
 * device only, not on device memory; args' pointers must be set as for the
 * call, workspace aside. */
int mrtdf_tree_attention_workspace(const mrtdf_cache* cache, const mrtdf_tree_args* args, size_t* bytes);
int mrtdf_tree_attention(const mrtdf_cache* cache, const mrtdf_tree_args* args, void* stream);

/* Failure-detection check: the same call, but a wait of its kernels for a copy
 * or a product looks once and gives up instead of after 0.5 s. Rows of out and
 * lse are then NaN as a whole, or right where no wait of theirs ran out. */
int mrtdf_check_tree_attention_wait(const mrtdf_cache* cache, const mrtdf_tree_args* args, void* stream);

/*
 * The attention weight that each cached row collects (what mrtdf_cache_evict
 * ranks rows by). path[b] lists the accepted nodes of sequence b, increasing
 * and ended by the first entry that is not a node above the one before it (or
 * by path_len); nodes that no longer fit into the capacity are left out. With
 * q, k_new and lse of the verification (for every layer of the cache):
 *   mass_out[t] = decay * mass[t] + sum over the query heads of the kv head and
 *                 the path's nodes r of exp(x(r, t) - lse(r))        t < lens[b]
 *   mass_out[lens[b] + j] = the same sum for the path's own row j, over r >= j
 * that is where mrtdf_cache_commit puts the path's rows. Other entries are left
 * as they are; mass_out may be mass. Node r of the path has depth r. A row with
 * lse = -inf adds nothing; a sequence that is passed over is left alone. Sums
 * are float32, one owner and one order each.
 */
typedef struct mrtdf_mass_args {
  size_t struct_bytes;
  mrtdf_rows q;     /* (layers, batch, heads, nodes) rows */
  mrtdf_rows k_new; /* (layers, batch, kv_heads, nodes) rows */
  const float* lse;      /* (layers, batch, heads, nodes) */
  const int32_t* path;   /* (batch, path_len) */
  const float* rel_bias; /* (heads, rel_len) or NULL, shared by the layers */
  const float* mass;     /* (layers, batch, kv_heads, capacity) */
  float* mass_out;
  int32_t heads, nodes, path_len, rel_len;
  float scale, decay;
} mrtdf_mass_args;
int mrtdf_cache_mass(const mrtdf_cache* cache, const mrtdf_mass_args* args, void* stream);

/*
 * Appends the accepted path to the cache of every layer: row lens[b] + j of K
 * and V takes row path[b][j] of k_new and v_new, pos (if any) gets next_pos[b]
 * + j, and lens_out[b] = lens[b] + nodes taken, next_pos_out[b] = next_pos[b] +
 * the same. The path is read as by mrtdf_cache_mass. Rows behind the new length
 * are left as they are. lens_out and next_pos_out are other buffers than lens
 * and next_pos; a sequence that is passed over keeps both.
 */
typedef struct mrtdf_commit_args {
  size_t struct_bytes;
  mrtdf_rows k_new, v_new; /* (layers, batch, kv_heads, nodes) rows */
  const int32_t* path;     /* (batch, path_len) */
  int32_t* lens_out;       /* (batch) */
  int32_t* next_pos_out;   /* (batch) or NULL */
  int32_t nodes, path_len;
} mrtdf_commit_args;
int mrtdf_cache_commit(const mrtdf_cache* cache, const mrtdf_commit_args* args, void* stream);

/*
 * Eviction by collected weight. A sequence with more than `budget` rows keeps,
 * in every layer and kv head by itself, the budget rows that come first by:
 * protected (position >= next_pos[b] - recent, or < sinks), then the larger
 * mass, then the lower row; a mass that is NaN comes last. Rows below the
 * budget that are kept stay where they are; the i-th evicted row below the
 * budget takes K, V, mass and pos of the i-th kept row at or above it, so at
 * most the evicted rows are written (attention goes by pos, not by row order).
 * mass_out and pos_out get the kept rows' entries (and those of sequences
 * within the budget); they may be mass and cache.pos. lens_out[b] = min(lens[b],
 * budget), another buffer than lens; a sequence that is passed over keeps its
 * length and is left alone. Rows and entries at and above the new length are
 * left as they are. recent + sinks <= budget; capacity <= 2^20 rows.
 */
typedef struct mrtdf_evict_args {
  size_t struct_bytes;
  const float* mass; /* (layers, batch, kv_heads, capacity) */
  float* mass_out;
  int32_t* pos_out;  /* (layers, batch, kv_heads, capacity) */
  int32_t* lens_out; /* (batch) */
  int32_t budget, recent, sinks;
} mrtdf_evict_args;
int mrtdf_cache_evict(const mrtdf_cache* cache, const mrtdf_evict_args* args, void* stream);

/*
 * Product with 4-bit weights: out[m][n] = sum_k x[m][k] (scales[n][k / group] *
 * q[n][k] + biases[n][k / group]), q in 0 .. 15. packed[n][j] holds column 2 j
 * in its low half and 2 j + 1 in its high half. x, scales and biases are of
 * `dtype`; out is of out_dtype (float32 for float32 x). The weights are not
 * rounded: sums of x times whole numbers are scaled in float32. x keeps all of a
 * bf16's bits and 22 of a float32's, per group from the largest. 1 <= m <= 64,
 * k <= 2^17 a multiple of the group (32, 64 or 128), n <= 2^24; x's rows and
 * packed on 16-byte boundaries. A row of x with an infinity or a NaN gives
 * results that are not finite, and touches no other row. Finite x gives finite
 * results where the sums of x times the weights, over the columns and over parts
 * of them, fit float32 (scales and biases below 2^100).
 */
typedef struct mrtdf_q4_args {
  size_t struct_bytes;
  const void* x;      /* (m, k), x_stride elements from row to row */
  const void* packed; /* (n, k / 2) bytes */
  const void* scales; /* (n, k / group) */
  const void* biases; /* (n, k / group) */
  void* out;          /* (m, n), out_stride elements from row to row */
  void* workspace;    /* mrtdf_q4_linear_workspace bytes, 16-byte aligned; contents do not matter */
  size_t workspace_bytes;
  int64_t x_stride, out_stride;
  int32_t m, n, k, group, dtype, out_dtype, device;
} mrtdf_q4_args;
/* Workspace of a call with these sizes (x as the product takes it and partial
 * sums, up to 10 MB and some bytes per element of x; 0 where x is small). args' pointers must be set as for the call, workspace
 * aside. */
int mrtdf_q4_linear_workspace(const mrtdf_q4_args* args, size_t* bytes);
int mrtdf_q4_linear(const mrtdf_q4_args* args, void* stream);

/* Failure-detection check: the same call, but a wait of its kernel for a free
 * place to copy to looks once and gives up, where the call streams x. Results
 * are NaN or right, one by one. */
int mrtdf_check_q4_linear_wait(const mrtdf_q4_args* args, void* stream);

/*
 * Weights (n, k) of `dtype` to the form that mrtdf_q4_linear takes: per group
 * of columns bias = min, scale = (max - min) / 15, both rounded to dtype, and
 * q = (w - bias) / scale with those two, rounded to the nearest (ties to even)
 * and clamped to 0 .. 15; a scale of 0 gives q = 0. Weights are finite, max - min too.
 */
typedef struct mrtdf_q4_pack_args {
  size_t struct_bytes;
  const void* w; /* (n, k), w_stride elements from row to row */
  void* packed;
  void* scales;
  void* biases;
  int64_t w_stride;
  int32_t n, k, group, dtype, device;
} mrtdf_q4_pack_args;
int mrtdf_q4_quantize(const mrtdf_q4_pack_args* args, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* MRTDF_H_ */
