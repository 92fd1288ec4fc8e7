/* include/mibc.h — C-ABI of the MI355X-native simplex basecalling engine ("mibc").
 *
 * This is the drop-in boundary: plain C, raw pointers and sizes, no torch types.
 * It replaces what the reference reaches through `extern "C" { #include "koi.h" }` (closed
 * source; call sites only) plus the libtorch ops around it, for the GPU side of
 * basecall::ModelRunnerBase (dorado/basecall/include/basecall/ModelRunnerBase.h:20-38).
 * The host-side C++ mirror of CudaCaller / CudaModelRunner that sits on top of this header is
 * dorado_amd/host/ (HipCaller, HipModelRunner); INTEGRATION.md shows the reference-side binding.
 *
 * Conventions (Koi-like): every entry returns int: 0 = MIBC_OK, >0 = not supported (caller may
 * fall back), <0 = error (text via mibc_last_error).  No exceptions cross this boundary.
 * All device work of one engine is issued on that engine's own HIP stream; entries marked
 * (async) return before the work completes — call mibc_sync().
 */
#ifndef MIBC_H
#define MIBC_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* libmibc.so is built with -fvisibility=hidden: exactly the entry points declared in this header are exported. */
#if defined(__GNUC__) || defined(__clang__)
#define MIBC_API __attribute__((visibility("default")))
#else
#define MIBC_API
#endif

#define MIBC_OK 0
#define MIBC_NOT_SUPPORTED 1
#define MIBC_ERR_ARG (-1)
#define MIBC_ERR_HIP (-2)
#define MIBC_ERR_MEM (-3)

/* Activation ids == dorado/config/include/config/common.h:19 (enum Activation order). */
#define MIBC_ACT_SWISH 0
#define MIBC_ACT_SWISH_CLAMP 1
#define MIBC_ACT_TANH 2

/* The fields of config::BasecallModelConfig the hot path reads
 * (dorado/config/include/config/BasecallModelConfig.h:99-160; ConvParams common.h:41-49). */
typedef struct mibc_model_desc {
    int n_convs;
    int conv_insize[8], conv_size[8], conv_winlen[8], conv_stride[8];
    int conv_act[8];
    int lstm_size, lstm_layers;
    int state_len, outsize;
    int bias;         /* linear1 has a bias (pre-v4 / decomposed head) */
    int clamp;        /* clamp scores to [-5,5] (folded into the decoder's score read, as
                         CUDADecoder does: basecall/model/CRFModel.cpp:107-109) */
    float scale;      /* 5.0 => head applies 5*tanh */
    int out_features; /* >0: two-stage head (linear1 -> linear2); -1: single */
    int num_features;
    /* transformer (sup@v5) fields; tx_d_model <= 0 selects the LSTM-CRF path */
    int tx_d_model, tx_nhead, tx_depth, tx_dim_ff, tx_win_upper, tx_win_lower, tx_max_seq_len;
    float tx_deepnorm_alpha, tx_theta;
    int up_size, up_scale_factor;
    float crf_scale, crf_blank_score;
    int crf_expand_blanks;
    /* 1: the reference's quantised LSTM path (nn/LSTMStack.cpp:127-211, KOI_I8): int8 weights (per-row scales,
     * utils::quantize_tensor) and int8 activations — for EVERY layer when the last convolution's activation is tanh (the
     * v4.3 LSTM-CRF models: nn/ConvStack.cpp:72 hands over CUTLASS_TNC_I8), else layers 2..L with the first layer in f16
     * (:73, LSTMStack.cpp:199-207).  LSTM models with
     * lstm_size 128 / 256 / 384 (any batch) or 512 / 768 / 1024 (batches that are multiples of 256: mibc_batch_granularity()
     * reports 256 then) and >= 2 layers; combinable with variable chunks (mibc_*_var: masked instances of the same kernels —
     * the reference's default GPU mode is both at once, basecall/CudaModelRunner.cpp:21-49).
     * 0: f16 throughout.  Which of the two a model gets by default is the CALLER's rule: the reference-side binding
     * (integration/HipModelRunnerAdapter.h mibc_desc_from_config) and bench.py apply the reference's own
     * (nn/ConvStack.cpp:60-89: int8 for tanh-conv models with 128 < lstm_size <= 1024), both arithmetics have a stated parity
     * contract. */
    int lstm_quant;
} mibc_model_desc;

/* basecall::decode::DecoderOptions (dorado/basecall/include/basecall/DecodedChunk.h:15-23). */
typedef struct mibc_decode_opts {
    int beam_width;    /* 32 */
    float beam_cut;    /* 100.0 */
    float blank_score; /* 2.0 (fixed stay score) */
    float q_shift;     /* config qbias */
    float q_scale;     /* config qscale */
} mibc_decode_opts;

/* Per-stage GPU time of the last mibc_call*/
typedef struct mibc_stage_ms {
    float conv, lstm, head, decode, total;
    float lstm_layer[8]; /* per LSTM layer */
    float h2d, d2h;
} mibc_stage_ms;

typedef struct mibc_engine mibc_engine;

/* ---- devices (replaces torch_utils/cuda_utils.cpp:224-248,364-384 device discovery) ---- */
MIBC_API int mibc_device_count(void);
MIBC_API int mibc_device_memory(int device_id, size_t *free_bytes, size_t *total_bytes); /* cuda_utils.cpp:250-262 */
MIBC_API const char *mibc_last_error(const mibc_engine *e); /* e may be NULL: last global error */
/* Identity of the binary: 16 hex digits of a sha256 over every source file the library was compiled from (tools/build_id.py;
 * "-dbg" appended in libmibc_dbg.so) — what a caller logs next to the model name, the role of the Koi / dorado version strings
 * (dorado/dorado_version.h DORADO_VERSION); the test suite refuses a library whose id is not the tree's. */
MIBC_API const char *mibc_build_id(void);

/* ---- lifetime (replaces CudaCaller ctor: basecall/CudaCaller.cpp:149-200) ----
 * weights: host f32 tensors in module.parameters() order (basecall/crf_utils.cpp:34-88):
 * conv{1..3}.{weight[Cout,Cin,W],bias}, rnn{1..L}.{weight_ih,weight_hh,bias_ih,bias_hh},
 * linear1.weight [,linear1.bias] [,linear2.weight].  Converted to f16 device layouts once. */
MIBC_API int mibc_create(int device_id, const mibc_model_desc *desc, const float *const *weights,
                int n_weights, mibc_engine **out);
MIBC_API void mibc_destroy(mibc_engine *e);

/* ---- memory (replaces CudaCaller memory model :323-369 and WorkingMemory arena) ---- */
MIBC_API int mibc_query_memory(const mibc_engine *e, int T_in, size_t *bytes_per_chunk, size_t *bytes_fixed);
MIBC_API int mibc_reserve(mibc_engine *e, int N_max, int T_in); /* (re)allocates the device workspace */
MIBC_API int mibc_output_steps(const mibc_engine *e, int T_in); /* T = number of output steps */
MIBC_API int mibc_batch_granularity(const mibc_engine *e);      /* N must be a multiple of this */
/* The weight quantisation of the lstm_quant path, host only (no device): utils::quantize_tensor(cat(W_ih, W_hh, 1).half(), 1)
 * (torch_utils/tensor_utils.cpp:293-300 as called by nn/LSTMStack.cpp:160-168), bit for bit — f16 arithmetic included.
 * wih, whh: [4C][C] f32 (module.parameters() layout); q: [4C][2C] int8 (columns < C from W_ih); scale: [4C]. */
MIBC_API int mibc_quantize_lstm_weights(const float *wih, const float *whh, int C, int8_t *q, float *scale);

MIBC_API void *mibc_host_alloc(size_t bytes); /* pinned host memory (CudaCaller.cpp:289-314) */
MIBC_API void mibc_host_free(void *p);
MIBC_API void *mibc_device_alloc(mibc_engine *e, size_t bytes);
MIBC_API void mibc_device_free(mibc_engine *e, void *p);
MIBC_API int mibc_memcpy_h2d(mibc_engine *e, void *dst_dev, const void *src_host, size_t bytes); /* sync */
MIBC_API int mibc_memcpy_d2h(mibc_engine *e, void *dst_host, const void *src_dev, size_t bytes); /* sync */

/* ---- the hot path ----
 * in:     f16 [N, 1, T_in]                (what BasecallerNode hands accept_chunk)
 * scores: f16 [N, T, K], K = 4^(state_len+1)   (CRFModel.cpp:111: NTC f16)
 * out:    int8 [3][N][T] = moves | bases (ASCII, packed at the front, NUL padded) | qstring
 *         (identical to the reference's CUDADecoder buffer: decode/CUDADecoder.cpp:66-71,153-168)
 */
MIBC_API int mibc_forward(mibc_engine *e, const uint16_t *in_dev, int N, int T_in,
                 uint16_t *scores_dev); /* (async) network only; replaces CRFModelImpl::run_koi */
MIBC_API int mibc_decode(mibc_engine *e, const uint16_t *scores_dev, int N, int T,
                const mibc_decode_opts *opts,
                int8_t *out_dev); /* (async) replaces CUDADecoder::beam_search_part_1 */
MIBC_API int mibc_call_device(mibc_engine *e, const uint16_t *in_dev, int N, int T_in,
                     const mibc_decode_opts *opts, int8_t *out_dev); /* (async) forward+decode */
MIBC_API int mibc_call(mibc_engine *e, const uint16_t *in_host, int N, int T_in,
              const mibc_decode_opts *opts,
              int8_t *out_host); /* H2D + forward + decode + D2H, synchronous
                                    (CudaCaller::call_chunks, CudaCaller.cpp:224-271) */
MIBC_API int mibc_sync(mibc_engine *e);
/* Opt-in: run the decoder (backward / forward scans, posteriors, beam search) on its own stream with the scores buffer
 * double-buffered, so that the decoder of one batch (HBM streaming, idle matrix pipes) runs under the network of the next
 * (matrix pipe / L2 bound, 0.7 TB/s of HBM traffic), and — where a batch is decoded in sub-batches — under the head of the next
 * sub-batch.  Results are unchanged.  Costs a second scores buffer; per-stage profiling (mibc_get_stage_ms) is not available
 * while it is on.  Applies to mibc_call_device, mibc_call_device_i16, mibc_call, mibc_call_i16, mibc_call_async (the
 * variable-chunk calls stay serial).  After the asynchronous device calls the output planes are complete once mibc_sync or
 * mibc_memcpy_d2h returns (both join the decoder stream); mibc_query_memory counts the second scores buffer while it is on. */
MIBC_API int mibc_set_decode_overlap(mibc_engine *e, int on);
/* Two-phase form of mibc_call (the overlap CudaCaller gets from its runners' own streams, CudaCaller.cpp:645-719 +
 * decode/CUDADecoder.h:13-15): mibc_call_async enqueues H2D (copy stream) -> network + decode (engine stream) ->
 * D2H (second copy stream) for `slot` (0 or 1) and returns; mibc_call_wait blocks until that slot's output has
 * arrived in out_host.  Two slots in flight: the copies of one batch run beside the kernels of the other.  A slot
 * must be waited for before it is submitted again; in_host / out_host must be pinned (mibc_host_alloc) and stay
 * valid until the wait returns.  shift_scale_host: NULL (in_host holds scaled f16) or float [N][2] (raw int16). */
MIBC_API int mibc_call_async(mibc_engine *e, int slot, const void *in_host, const float *shift_scale_host, int N, int T_in,
                    const mibc_decode_opts *opts, int8_t *out_host);
MIBC_API int mibc_call_wait(mibc_engine *e, int slot);
MIBC_API int mibc_call_poll(mibc_engine *e, int slot); /* 1 = finished (then call mibc_call_wait), 0 = still running */

/* ---- signal scaling in front of the path (the device side of ScalerNode,
 *      dorado/read_pipeline/nodes/ScalerNode.cpp:144-269) ----
 * The reference scales each read on the host (int16 ADC -> f16((x - shift) / scale),
 * torch_utils/tensor_utils.cpp:89-142) before chunking; these entry points take the raw int16 chunk
 * rows instead, with ONE (shift, scale) pair per chunk (its read's), and apply the identical map
 * (f32 subtract, IEEE divide, round-to-nearest-even to f16) inside the first convolution's input read.
 * shift_scale: float [N][2]. */
#define MIBC_SCALE_QUANTILE 0 /* ScalerNode.cpp:42-52 (normalisation), utils::quantile_counting */
#define MIBC_SCALE_MED_MAD 1  /* ScalerNode.cpp:32-40 (med_mad) */
MIBC_API int mibc_forward_i16(mibc_engine *e, const int16_t *in_dev, const float *shift_scale_dev, int N, int T_in,
                     uint16_t *scores_dev);
MIBC_API int mibc_call_device_i16(mibc_engine *e, const int16_t *in_dev, const float *shift_scale_dev, int N, int T_in,
                         const mibc_decode_opts *opts, int8_t *out_dev);
MIBC_API int mibc_call_i16(mibc_engine *e, const int16_t *in_host, const float *shift_scale_host, int N, int T_in,
                  const mibc_decode_opts *opts, int8_t *out_host);
/* Per-read (shift, scale) of the two data-driven strategies.  Reads are concatenated in sig_dev;
 * read r = [offsets_dev[r], offsets_dev[r+1]) (n_reads + 1 offsets).  params4 (quantile only) =
 * {quantile_a, quantile_b, shift_multiplier, scale_multiplier} (config::QuantileScalingParams).
 * raw_dev (optional, [n_reads][2]) receives (q_a, q_b) resp. (median, median |x - median|).
 * Integer work, bit-exact with the reference.  (The PA strategy, ScalerNode.cpp:186-215, is a closed
 * formula of the read's calibration and needs no pass over the samples: host side.) */
MIBC_API int mibc_scaler_stats(mibc_engine *e, const int16_t *sig_dev, const int64_t *offsets_dev, int n_reads,
                      int strategy, const float *params4, float *shift_scale_dev, float *raw_dev);
/* Whole reads: out[i] = f16((float(x[i]) - shift_r) / scale_r); replaces
 * utils::shift_scale_tensor_i16_to_f16_inplace for callers that want the scaled read back
 * (e.g. for the signal trim, torch_utils/trim.cpp). */
MIBC_API int mibc_scale_reads(mibc_engine *e, const int16_t *sig_dev, const int64_t *offsets_dev, int n_reads,
                     const float *shift_scale_dev, uint16_t *out_f16_dev);

/* ---- variable chunk sizes ----
 * The reference's CUDA path packs ragged chunks (utils::generate_variable_chunks, read_pipeline/base/chunk.cpp:
 * 49-107; basecall/CudaModelRunner.cpp:21-49; nn/AuxiliaryData.cpp) so that short reads are not repeat-padded to
 * chunk_size.  Here a batch row [T_in] may hold several chunks: chunk = (row, sample_start, n_samples), both
 * multiples of the model stride, chunks of one row in ascending order and >= 2 output steps (2 * stride samples)
 * apart; samples outside every chunk are ignored.  Every chunk is called exactly as if it stood alone
 * (zero padding at its edges, zero initial LSTM state, its own decode).  Output planes int8 [3][N][T]: chunk c
 * occupies steps [sample_start / stride, (sample_start + n_samples) / stride) of its row in each plane (bases and
 * qstring packed at the front of that interval, NUL padded); everything else is 0.
 * shift_scale: NULL (input rows are scaled f16) or float [N][2] (input rows are raw int16, see above).
 * LSTM models of every supported lstm_size (128 ... 1024; the reference's range: api/runner_creation.cpp:24-44);
 * transformer models return MIBC_NOT_SUPPORTED (the reference's Tx path has no variable chunks either). */
typedef struct mibc_var_chunk {
    int row;
    int sample_start;
    int n_samples;
} mibc_var_chunk;
MIBC_API int mibc_forward_var(mibc_engine *e, const void *in_dev, const float *shift_scale_dev, int N, int T_in,
                     const mibc_var_chunk *chunks_host, int n_chunks, uint16_t *scores_dev);
MIBC_API int mibc_call_device_var(mibc_engine *e, const void *in_dev, const float *shift_scale_dev, int N, int T_in,
                         const mibc_var_chunk *chunks_host, int n_chunks, const mibc_decode_opts *opts,
                         int8_t *out_dev);
MIBC_API int mibc_call_var(mibc_engine *e, const void *in_host, const float *shift_scale_host, int N, int T_in,
                  const mibc_var_chunk *chunks_host, int n_chunks, const mibc_decode_opts *opts, int8_t *out_host);
/* Two-phase form of mibc_call_var on the slots of mibc_call_async (same rules: pinned in_host / out_host, one submission
 * per slot until mibc_call_wait; fixed and variable batches may be mixed across the two slots).  The reference runs its
 * variable-chunk batches on the same stream pipeline as the fixed ones (basecall/CudaModelRunner.cpp:21-49,
 * CudaCaller.cpp:645-719).  chunks_host is consumed before the call returns. */
MIBC_API int mibc_call_var_async(mibc_engine *e, int slot, const void *in_host, const float *shift_scale_host, int N, int T_in,
                        const mibc_var_chunk *chunks_host, int n_chunks, const mibc_decode_opts *opts, int8_t *out_host);

/* ---- POD5 signal decode ----
 * The reference obtains a read's int16 samples from pod5_get_read_complete_signal
 * (dorado/data_loader/DataLoader.cpp:163-170; pod5-file-format 0.3.36, not vendored).  POD5 stores each
 * signal-table row as zstd(svb16(zigzag(delta(int16)))).  The zstd frame is inflated on the host (libzstd);
 * this entry point does the StreamVByte-16 + zig-zag + delta stage for a whole batch of rows on the device,
 * so the samples are born in HBM, next to mibc_scaler_stats / mibc_*_i16.
 * streams_dev: concatenated inflated rows; stream_off_dev / sample_off_dev: n_rows + 1 prefix offsets
 * (bytes / samples); status_dev[r] = 0 ok, 1 = row not consumed exactly (corrupt). */
MIBC_API int mibc_svb16_decode(mibc_engine *e, const uint8_t *streams_dev, const int64_t *stream_off_dev,
                      const int64_t *sample_off_dev, int n_rows, int16_t *out_dev, int *status_dev);

/* ---- operators of transformer layers (no engine, no model) ----
 * The non-GEMM operators of a transformer layer for any width, head size and mask: what the engine's own transformer path has
 * fused for one shape family (nn/TxModules.cpp:184-250 rotary, :279-426 attention, :859-906 layer; nn/RMSNorm.cpp:14-18), as
 * entry points of their own.  All pointers are device pointers of `device`; work is issued on `stream` (a hipStream_t of that
 * device, NULL = its null stream) and the call returns before it completes (async).  No call allocates, copies to the host,
 * synchronises or keeps anything for the next one, so all of them can be captured into a graph; the caller's current device is
 * left as it was.  Refusals are decided from the arguments alone, before anything is launched (text: mibc_last_error(NULL)).
 * Strides count elements; the innermost dimension is contiguous.  A stride may be 0 on inputs (a broadcast dimension), never
 * on outputs.  An output may be x, residual or q where type, shape and strides are the same (in place); an output that shares memory with
 * another operand in any other way is refused. */
#define MIBC_TYPE_F16 0
#define MIBC_TYPE_BF16 1
#define MIBC_TYPE_F32 2
#define MIBC_TYPE_I8 3
#define MIBC_TYPE_E4M3 4 /* OCP e4m3 (no infinity, largest value 448) */

/* h = x + alpha * residual;  y = h / sqrt(mean(h^2) + eps) * weight  over the last dimension, computed in f32 (squares beyond it: y = 0), h
 * not rounded in between.  sum_out (optional) receives h, out receives y, both in `type`; or, out_type I8 / E4M3, out receives
 * round(y / s) (the f32 quotient, then the code, nearest with ties to even), s = max|y| / 127 (I8) or / 448 (E4M3) over the row
 * (group 0) or over each group of 32, 64 or 128 columns, and scale_out [rows][cols / group] receives s.
 * Where max|y| is 0, s = 1; where a value of the group is not finite, s = NaN and the group's codes are 0; codes end at 127 and 448 (a
 * scale of some 2^-149 steps is off by up to a third; below half a step s = 1).  weight: f32 or `type`, NULL = ones; residual NULL = none.
 * 1 <= cols <= 32768. */
typedef struct mibc_rms_norm_args {
    const void *x, *residual, *weight;
    void *sum_out, *out;
    float *scale_out;
    int64_t rows;
    int64_t x_stride, residual_stride, sum_stride, out_stride, scale_stride; /* elements from row to row */
    int32_t cols, type, weight_type, out_type, group;
    float alpha, eps;
    int32_t reserved; /* 0 */
} mibc_rms_norm_args;
MIBC_API int mibc_rms_norm(int device, void *stream, const mibc_rms_norm_args *a);

/* Rotary positions of up to two tensors [batch][tokens][heads][head_dim] (queries and keys) in one launch.  Pair i of the first
 * rot_dim columns of a head at position p turns by p * freqs[i]:  (a, b) -> amplitude * (a cos - b sin, a sin + b cos); pairs
 * are columns (i, i + rot_dim / 2), or (2 i, 2 i + 1) if `interleaved`.  The other columns are copied.  Position of token t of
 * row n: positions[n][t] (contiguous int32 or int64; may be negative, which turns back), or start + t where positions is NULL.
 * freqs: f64 device [rot_dim / 2], radians per position (mibc_rope_frequencies).  Angles are reduced in f64. */
typedef struct mibc_rope_args {
    const void *x[2];  /* x[1] may be NULL */
    void *out[2];
    const void *positions; /* or NULL */
    const double *freqs;
    int64_t start;
    int64_t x_stride[2][3], out_stride[2][3]; /* batch, token, head */
    int64_t batch, tokens;
    int32_t heads[2];
    int32_t head_dim, rot_dim, type, interleaved, positions_64;
    float amplitude;
} mibc_rope_args;
MIBC_API int mibc_rope(int device, void *stream, const mibc_rope_args *a);
#define MIBC_ROPE_PLAIN 0    /* theta^(-2i / rot_dim) */
#define MIBC_ROPE_LINEAR 1   /* ... / factor: positions squeezed into the trained length */
#define MIBC_ROPE_BASE 2     /* theta * factor^(rot_dim / (rot_dim - 2)) as the base: the slowest pair slows by factor, the fastest stays */
#define MIBC_ROPE_BY_PARTS 3 /* pairs with >= turns_high turns over original_length stay, with <= turns_low are / factor, a ramp between */
/* Host only: the frequencies mibc_rope takes, freqs [rot_dim / 2] on the HOST. */
MIBC_API int mibc_rope_frequencies(int scaling, int rot_dim, double theta, double factor, double original_length, double turns_low,
                          double turns_high, double *freqs);

/* out = softmax(scores) v per head, scores = scale * (q . k), then cap * tanh(scores / cap) if softcap > 0, then
 * - slopes[head] * |i - j| if slopes (i, j: positions of query and key), over the keys a query sees.  q, out:
 * [batch][q_tokens][heads][head_dim]; k, v: [batch][k_tokens][kv_heads][head_dim], heads a multiple of kv_heads, query head h
 * reading key head h / (heads / kv_heads).  Row n has len = k_len[n] keys (NULL: k_tokens; clamped to [0, k_tokens]); query t
 * stands at position i = q_start + t (q_start == MIBC_ATTN_END: len - q_tokens + t, the last query on the last key).  It sees
 * key j < len if i - window_back <= j <= i + window_ahead (a negative limit: unlimited; window_ahead = 0: causal) or if
 * j < prefix[n].  doc_offsets [n_docs + 1] (needs batch 1, q_tokens == k_tokens, no k_len, q_start MIBC_ATTN_END; ascending):
 * document d is the tokens [doc_offsets[d], doc_offsets[d + 1]); a token sees its own document only, prefix is then [n_docs] and
 * counts from the document's start, tokens in no document see nothing and are seen by none.  A query that sees nothing, or only
 * scores of -infinity, gives zeros and lse = -infinity.  What a query does not see has no influence on its result, whatever it holds (NaN
 * and infinity included); a NaN or infinity of v that it does see reaches it, however small its weight (as NaN where no key has any).
 * lse (optional) [batch][heads][q_tokens] f32 contiguous: log of the sum of exp(scores).
 * Scores, statistics and sums are f32.  With more than 16 query rows per key head the probabilities are rounded to `type` before their
 * product with v: each is off by at most 2^-8 of itself in bf16, by 2^-11 or 2^-36 of the row's largest in f16; what is summed for the
 * denominator and lse is not rounded.  With at most 16 rows they enter as two such parts (2^-16, 2^-22 or the same 2^-36).  Scores are off
 * by a few 2^-22 of their own size and, for a softcap of up to 64, of the cap's.  softcap / scale may be at most 3e37 and scale / softcap
 * at most 1e38; with slopes, scale and softcap are at least 1e-18, and slopes / scale must stay inside f32.
 * Types F16, BF16; head_dim 32, 64, 96 or 128; token and head strides multiples of 8 elements, pointers aligned to 16 bytes.
 * workspace: mibc_attention_workspace(a) bytes on the device (0, as for any call with fewer than 512 keys: may be NULL), the
 * call's own until it has completed. */
#define MIBC_ATTN_END (-2147483647 - 1)
typedef struct mibc_attention_args {
    const void *q, *k, *v;
    void *out;
    float *lse;
    const int32_t *k_len, *prefix, *doc_offsets;
    const float *slopes;
    void *workspace;
    uint64_t workspace_bytes;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3]; /* batch, token, head */
    int32_t batch, heads, kv_heads, q_tokens, k_tokens, head_dim, n_docs, type;
    int32_t window_back, window_ahead, q_start;
    float scale, softcap;
    int32_t reserved; /* 0 */
} mibc_attention_args;
MIBC_API int mibc_attention(int device, void *stream, const mibc_attention_args *a);
MIBC_API uint64_t mibc_attention_workspace(const mibc_attention_args *a);

/* ---- measurement (replaces CudaCaller.cpp:552-569 timing + gpu_profiling.h ranges) ---- */
MIBC_API int mibc_time_forward(mibc_engine *e, int N, int T_in, float *ms); /* min of 2 runs, like :552-569 */
MIBC_API int mibc_get_stage_ms(mibc_engine *e, mibc_stage_ms *out);         /* hipEvent times, last call */
/* ... of the profiled call BEFORE the last one: blocks only until that earlier call has finished, so a caller that has
 * already enqueued call i can read the stage times of call i - 1 without draining the stream (two event sets alternate) */
MIBC_API int mibc_get_stage_ms_prev(mibc_engine *e, mibc_stage_ms *out);
MIBC_API int mibc_set_profile(mibc_engine *e, int level);                   /* 0 off, 1 per-stage events, 2 + roctx ranges around the
                                                                      stages (utils::ScopedProfileRange,
                                                                      torch_utils/gpu_profiling.h:32-99) for rocprofv3
                                                                      --marker-trace */

/* ---- parity taps (test-only; copy an intermediate of the LAST call to the host) ----
 * tap: 0 conv1 out [N,T_in,16] f16 | 1 conv2 out (padded rows) | 2 conv3 out [T,N,C] f16
 *      3 LSTM stack out [T,N,C] f16 | 4 back-guides [N,T+1,S] f32 (first decode sub-batch)
 *      5 per-block quality prob [N,T] f32 */
MIBC_API int mibc_debug_tap(mibc_engine *e, int tap, void *host_dst, size_t bytes);

#ifdef __cplusplus
}
#endif
#endif /* MIBC_H */
