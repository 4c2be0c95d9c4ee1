/*
 * katago_cuda.h — the C ABI of the katago-rs B200 (sm_100a) neural-net backend.
 *
 * This is the boundary a `cuda` backend of katago-rs binds to. Each entry point replaces one piece of the
 * reference's `NeuralNet` trait (crates/katago-core/src/neuralnet/nninterface.rs:79-214) as implemented by the
 * burn backend (crates/katago-nn-burn/src/backend.rs); the citation is on each declaration. Plain pointers and
 * sizes only; no callbacks; the library never keeps a caller-owned pointer beyond the call.
 *
 * Every function returns an int status (KC_OK = 0). On failure kc_last_error() gives a message for this thread,
 * which the Rust side maps to KataError::StringError (nninterface.rs:202-205).
 *
 * Threading follows the reference: a model and a context may be shared; a handle is used by one thread at a time
 * ("Not thread-safe, each handle should only be used by one thread", nninterface.rs:33-34).
 */
#ifndef KATAGO_CUDA_H
#define KATAGO_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KC_OK 0
#define KC_ERR_INVALID 1    /* bad argument (sizes, null pointers, unsupported option) */
#define KC_ERR_PARSE 2      /* model file could not be parsed */
#define KC_ERR_CUDA 3       /* a CUDA call failed */
#define KC_ERR_TIMEOUT 4    /* kc_wait gave up before the batch finished (the batch is still in flight) */
#define KC_ERR_DEVICE 5     /* a kernel reported a device-side error (a bounded wait expired) */
#define KC_ERR_NO_DEVICE 6  /* no usable sm_100 device */

/* Precision of a context (the reference's useFP16 enabled_t plus an explicit choice, backend.rs:300-340). */
#define KC_PRECISION_F32 0   /* float32 everywhere: the parity tier (SIMT kernels) */
#define KC_PRECISION_F16 1   /* f16 activations and weights, f32 accumulation (tcgen05) */
#define KC_PRECISION_BF16 2  /* bf16 activations and weights, f32 accumulation (tcgen05) */
#define KC_PRECISION_AUTO 3  /* f16 for convolution nets, bf16 for nets with transformer blocks */

typedef struct kc_model kc_model;
typedef struct kc_context kc_context;
typedef struct kc_handle kc_handle;

/* ModelDesc fields the host needs (crates/katago-core/src/neuralnet/desc.rs; the ONNX metadata keys the reference
 * writes in tools/bin2onnx/bin2onnx.py:1566-1614). */
typedef struct kc_desc {
  char name[128];
  int32_t model_version;
  int32_t num_input_channels;
  int32_t num_input_global_channels;
  int32_t num_input_meta_channels;
  int32_t meta_encoder_version;
  int32_t num_policy_channels;
  int32_t num_value_channels;
  int32_t num_score_value_channels;
  int32_t num_ownership_channels;
  int32_t trunk_num_blocks;
  int32_t trunk_num_channels;
  int32_t trunk_norm_kind;
  int32_t has_any_transformer_blocks;
  int32_t has_any_nested_bottleneck_blocks;
  int32_t post_process_from_header;
  int32_t prefer_pass_alive_under_suicide_rules;
  int32_t prefer_exclude_territory_adjacent_to_atari;
  int64_t num_parameters;
  double trunk_spatial_conv_depth;
  /* td_score, score_mean, score_stdev, lead, variance_time, shortterm_value_error, shortterm_score_error,
   * output_scale multipliers (ModelPostProcessParams, bin2onnx.py:843-854) */
  float post_process[8];
} kc_desc;

/* Message of the last failed call on this thread ("" if none). Valid until the next call on this thread. */
const char* kc_last_error(void);

/* Number of CUDA devices the library can run on (sm_100). NeuralNet::printDevices / getNumEffectiveDevices. */
int kc_device_count(int* count);

/* Parse a KataGo model file (.bin, .bin.gz, .txt, .txt.gz) from memory. `file_name` (may be NULL) decides text vs
 * binary floats as the reference does (bin2onnx.py:1074-1082); NULL means: binary if the data holds "@BIN@".
 * A name ending in ".onnx" (or, without a name, data that starts as an ONNX ModelProto) is read as the ONNX export
 * the reference's tools/bin2onnx/bin2onnx.py writes (the files the reference's burn backend is generated from,
 * crates/katago-nn-burn/build.rs:25-30): its layers are rebuilt from the graph and its metadata_props.
 * Replaces NeuralNet::load_model_file (nninterface.rs:137; backend.rs:277-292). No device is touched. */
int kc_model_load(const void* bytes, size_t n, const char* file_name, kc_model** out);

/* NeuralNet::get_model_desc (nninterface.rs:140; backend.rs:295-297). */
int kc_model_desc(const kc_model* model, kc_desc* out);

/* NeuralNet::free of LoadedModel (Drop). Safe on NULL. */
int kc_model_destroy(kc_model* model);

/* NeuralNet::create_compute_context (nninterface.rs:148-162; backend.rs:300-340). `gpu_idxs` lists the devices
 * handles of this context will use (-1 = default device); nn_x_len and nn_y_len must be 19 (the reference's fixed
 * posLen, backend.rs:327-333); `precision` is a KC_PRECISION_* value. */
int kc_context_create(const int* gpu_idxs, int n_gpu_idxs, int nn_x_len, int nn_y_len, int precision,
                      const kc_model* model, kc_context** out);
int kc_context_precision(const kc_context* ctx, int* precision);
int kc_context_destroy(kc_context* ctx);

/* NeuralNet::create_compute_handle (nninterface.rs:166-186; backend.rs:343-389): uploads packed weights to
 * `gpu_idx` (-1 = the context's first device), allocates device activations and pinned host I/O for `max_batch`
 * rows, and prepares the forward pass. `inputs_use_nhwc` must be 0 (NCHW, as the reference). */
int kc_handle_create(kc_context* ctx, int gpu_idx, int max_batch, int inputs_use_nhwc, kc_handle** out);
int kc_handle_destroy(kc_handle* h);

/* Pinned host input buffers of the handle (the reference's BurnInputBuffers, backend.rs:150-212): spatial
 * [max_batch, C, 19, 19] NCHW float32, global [max_batch, G], meta [max_batch, M] (NULL when M = 0). */
int kc_handle_input_ptrs(kc_handle* h, float** spatial, float** global, float** meta);

/* Floats per output row and the offsets of its parts, as the reference's readback concatenates them
 * (backend.rs:584-617): policy [P, 362] (pass last), value [3], score [S_v], ownership [1, 361]. */
int kc_handle_output_layout(const kc_handle* h, int* row_len, int* policy_off, int* value_off, int* score_off,
                            int* ownership_off);

/* Non-blocking: copy rows [0, n) of the pinned inputs to the device, run the forward pass, copy the n output rows
 * into the handle's pinned output buffer, and record completion. The device half of run_network
 * (backend.rs:549-619). */
int kc_enqueue(kc_handle* h, int n);

/* Block until the last enqueue finished, at most `timeout_ms` (negative = no limit). On success `*out_rows` points
 * at n rows of kc_handle_output_layout's row_len floats in pinned memory, valid until the next kc_enqueue. The
 * reference waits on a helper thread (backend.rs:743-753); KC_ERR_TIMEOUT leaves the batch in flight. */
int kc_wait(kc_handle* h, int timeout_ms, const float** out_rows);

/* Bit-packed inputs. Every spatial input feature of the reference (nninputs.rs fill_row_v7 :1336) is 0 or 1, so a
 * row's planes travel as bits: plane c of a row is KC_PACKED_WORDS_PER_PLANE 32-bit words, point p = y * 19 + x at bit
 * p % 32 of word p / 32 (bits past 361 zero); 22 planes are 1,056 bytes instead of 31,768. Each row's symmetry is
 * applied on the device as the planes are read (the inverse of SymmetryHelpers::copy_inputs_with_symmetry,
 * nninputs.rs:872, which the reference runs on the host per row in copy_inputs, backend.rs:497-546). */
#define KC_PACKED_WORDS_PER_PLANE 12

/* NNOutput rows (the reference's copy_outputs, backend.rs:622-731, run on the device): per row KC_FINISHED_ROW_LEN
 * floats: policy [362] (optimism mixed for v12+ nets, symmetry undone, pass last), value [3] (win, loss, noresult),
 * misc [6] (scoreMean, scoreMeanSq, lead, varTimeLeft, shorttermWinlossError, shorttermScoreError, by model version),
 * ownership [361] (symmetry undone). */
#define KC_FINISHED_ROW_LEN 732
#define KC_FINISHED_POLICY 0
#define KC_FINISHED_VALUE 362
#define KC_FINISHED_MISC 365
#define KC_FINISHED_OWNERSHIP 371

/* The handle's pinned staging for kc_enqueue_packed: spatial_bits [max_batch][C][KC_PACKED_WORDS_PER_PLANE],
 * global [max_batch][G], meta [max_batch][M] (NULL when M = 0), symmetry [max_batch] (0..7: bit 0 flipY, bit 1
 * flipX, bit 2 transpose), policy_optimism [max_batch]. The binding of BurnInputBuffers (backend.rs:150-212) for
 * callers that write packed rows. */
int kc_handle_packed_input_ptrs(kc_handle* h, uint32_t** spatial_bits, float** global, float** meta,
                                int32_t** symmetry, float** policy_optimism);

/* kc_enqueue for the packed staging: one host-to-device copy of rows [0, n), the forward pass with each row's
 * symmetry applied on the device, and the readback. finish = 0 reads back the raw output rows (as kc_enqueue);
 * finish = 1 runs the reference's copy_outputs on the device and reads back NNOutput rows of KC_FINISHED_ROW_LEN
 * floats. kc_wait returns the rows of whichever the last enqueue read back. */
int kc_enqueue_packed(kc_handle* h, int n, int finish);

/* Pack one row's float planes [n_planes][361] into [n_planes][KC_PACKED_WORDS_PER_PLANE] words; KC_ERR_INVALID when a
 * value is neither 0 nor 1. */
int kc_pack_spatial(const float* planes, int n_planes, uint32_t* bits);

/* The point mappings of the device-side symmetry, for tests of the host logic (no device is used): reverse = 0:
 * table[y * 19 + x] = the input point the network sees at (y, x); reverse = 1: table[p] = the point an output p is
 * moved to. Equal to kc_copy_with_symmetry's moves (nninputs.rs:756-831). */
int kc_symmetry_table(int symmetry, int reverse, int* table);

/* Same as kc_enqueue but the inputs and outputs are device pointers (no host copies): spatial [n,C,19,19],
 * global [n,G], meta [n,M] (may be NULL when M = 0), out [n,row_len] float32. For callers that keep their
 * batches on the GPU. */
int kc_enqueue_device(kc_handle* h, int n, const float* d_spatial, const float* d_global, const float* d_meta,
                      float* d_out);

/* The CUDA stream (cudaStream_t) the handle's work runs on, for callers that order their own work or timing
 * events against it. */
int kc_handle_stream(kc_handle* h, void** stream);

/* Synchronise the handle's stream (bounded like kc_wait). */
int kc_synchronize(kc_handle* h, int timeout_ms);

/* The whole reference get_output for one batch (backend.rs:410-731): per row, copy the inputs into the handle's
 * staging buffers with `symmetry[i]` (SymmetryHelpers::copy_inputs_with_symmetry, nninputs.rs:872), run the net,
 * then for each row mix the optimistic policy with `policy_optimism[i]` (v12+ nets), undo the symmetry on policy
 * and ownership, and write the NNOutput fields. Rows travel bit-packed with the symmetry applied on the device when
 * every spatial value is 0 or 1 (always, for the reference's inputs), else as floats with the symmetry applied on
 * the host; the output handling runs on the device (kc_enqueue_packed with finish = 1). Row inputs: `spatial_rows[i]` [C*19*19] NCHW,
 * `global_rows[i]` [G], `meta_rows[i]` [M] (NULL when M = 0). Outputs per row i:
 *   policy_out + i*362 (362 floats, pass last), value_out + i*3 (win, loss, noresult),
 *   misc_out + i*6 (scoreMean, scoreMeanSq, lead, varTimeLeft, shorttermWinlossError, shorttermScoreError,
 *   filled per model version as backend.rs:690-729), ownership_out + i*361 (may be NULL: no ownership map). */
int kc_get_output(kc_handle* h, int n, const float* const* spatial_rows, const float* const* global_rows,
                  const float* const* meta_rows, const int* symmetry, const float* policy_optimism, int timeout_ms,
                  float* policy_out, float* value_out, float* misc_out, float* ownership_out);

/* Per-kernel-class device time of the forward passes since profiling was switched on, in ms: with profiling on,
 * each kernel launch of the forward is bracketed by CUDA events on the handle's stream (recorded inside the CUDA
 * graph when graphs are used), and kc_handle_profile waits for the last pass and accumulates its launches.
 * class: 0 conv3x3 GEMM, 1 conv1x1/linear GEMM, 2 stem GEMM, 3 attention, 4 other kernels. */
int kc_handle_set_profiling(kc_handle* h, int on);
int kc_handle_profile(kc_handle* h, double* ms_by_class, int64_t* launches_by_class, int n_classes);
/* Kernel launches per forward pass of n positions (1 <= n <= the handle's max_batch; some boundaries of a net take
 * one fused kernel or two kernels depending on n), and algorithmic FLOPs per row. */
int kc_handle_launch_count(kc_handle* h, int n, int* launches);
int kc_model_flops(const kc_model* model, double* flops_per_row, double* conv3x3_flops_per_row);

/* KataGo's masked global pooling followed by the gpool-to-bias matmul, on device tensors in the reference layout:
 * x [n][c][19*19] float32 (already masked), mask [n][19*19] (input channel 0), w [3c][oc], out [n][oc]:
 *   out[b] = [mean, mean * (sqrt(area) - 14) / 10, max over on-board points] x w
 * (tools/bin2onnx/bin2onnx.py gpool :1222-1230 and the matmul after it, :1255 / :1501). Enqueued on `stream`
 * (a cudaStream_t, NULL = legacy default stream); the pooled [n][3c] scratch is taken from the stream-ordered
 * allocator (cudaMallocAsync) and released after use. 3c <= 12288. */
int kc_gpool_fc(const float* d_x, const float* d_mask, int n, int c, const float* d_w, int oc, float* d_out,
                void* stream);

/* kc_gpool_fc for callers that cannot allocate GPU memory — for instance a host that reserves the device memory up
 * front for its own pools and forbids later allocations, or a latency-critical thread that cannot afford
 * cudaMalloc's device-wide synchronisation. This entry point has no counterpart in the reference; it allocates
 * nothing (no cudaMalloc, cudaFree or allocating library call). Its pooled [n][3c] scratch is one fixed array of
 * KC_GPOOL_NOALLOC_MAX_FLOATS floats (1 MiB) in device memory, present on every GPU that loads this library until
 * the process exits; larger n * 3c is rejected with KC_ERR_INVALID. The first call on a device looks up that
 * array's device address (once per device, with that device current), so make the first call on each device
 * before any stream capture. With CUDA's lazy module loading (the default) the array is only placed in device
 * memory when that first call loads this part of the library on the device: make the first call before reserving
 * the device's memory for other pools (or load modules eagerly, CUDA_MODULE_LOADING=EAGER). All calls share the one array and it keeps the last call's contents (every entry a
 * call reads is written by that call first): calls whose work overlaps on the GPU (different streams, or
 * different host threads on one device) race on it and must be ordered by the caller. Inputs, outputs and
 * stream are as for kc_gpool_fc. */
#define KC_GPOOL_NOALLOC_MAX_FLOATS 262144
int kc_gpool_fc_noalloc(const float* d_x, const float* d_mask, int n, int c, const float* d_w, int oc, float* d_out,
                        void* stream);

/* ---------------------------------------------------------------------------------------------------------------
 * Standalone operators on board tokens: rows of consecutive channels, one row per point (channels last), in
 * float32, f16 or bf16 (KC_PRECISION_F32 / F16 / BF16), with 32-bit statistics and sums. They have no counterpart in
 * the reference's graph; the neighbours there are its merged batch norm with activation and mask
 * (tools/bin2onnx/bin2onnx.py bn_act_mask, trunk_tip_rmsnorm :1440-1463) and its 2D rotary positions (:449-484,
 * :1388-1396), whose table layouts and activations they keep.
 *
 * All pointers are device pointers of one device, aligned to their element (speed wants 16 bytes, and strides that
 * are multiples of 16 bytes). Work is enqueued on `stream` (a cudaStream_t of that device, NULL = its legacy default
 * stream) without a host wait or an allocation, so that calls can be captured into a CUDA graph; the device need not
 * be current. Strides are in elements and not negative; rows of an output must not share memory. An output may be
 * the input of its own shape (same pointer and strides: in place); any other overlap of an output is refused.
 * `d_workspace` (16-byte aligned, contents not kept) must not be used by two calls that can overlap on the GPU, nor
 * be freed before a graph that captured it. Calls on different streams are otherwise independent. Results do not
 * depend on timing: the same call gives the same bits. Rows that do not lie on 16 bytes may be read in the aligned
 * 16-byte pieces that hold them; what else such a piece holds has no effect, and is not written.
 * --------------------------------------------------------------------------------------------------------------- */
#define KC_ACT_IDENTITY 0
#define KC_ACT_RELU 1
#define KC_ACT_MISH 2
#define KC_ACT_SILU 3

/* Group norm of n boards of `points` rows of `channels`, in `groups` groups of channels / groups neighbours. */
typedef struct kc_group_norm_desc {
  int32_t dtype; /* KC_PRECISION_* of x, y, dy and dx */
  int32_t act;   /* KC_ACT_* */
  int32_t n, points, channels, groups; /* n and points 0 .. 2^30, channels 1 .. 2^30, n * channels at most 2^46; where
                                          a group or a board is too large for a cluster of 16 blocks, n * groups
                                          below 2^31 */
  float eps;     /* >= 0 */
  int32_t reserved; /* 0 */
  int64_t x_board_stride, x_row_stride; /* x and dx */
  int64_t y_board_stride, y_row_stride; /* y and dy */
  int64_t mask_board_stride;
} kc_group_norm_desc;

/* Bytes of workspace a call needs (0: d_workspace may be NULL). backward: 0 kc_group_norm_act, 1 its backward. A
 * descriptor whose sizes or strides the calls refuse is refused here too. */
int kc_group_norm_act_workspace(const kc_group_norm_desc* desc, int backward, size_t* bytes);

/* y = act((x - mean) * rstd * weight[c] + bias[c]) at the points whose mask is not 0, 0 at the others, where mean and
 * rstd = 1 / sqrt(variance + eps) are those of the point's board and channel group over the points that are on
 * (whatever x holds at the others, NaN and infinities too, has no effect). Squares are summed in float32: where a
 * group's sum of squared distances from one of its values passes 3.4e38 (distances of 2.8e17 in 361 points x 12
 * channels) its y and rstd are NaN. d_mask: [n][points] float32 rows at mask_board_stride, NULL = every point;
 * d_weight, d_bias: [channels] float32, NULL = 1 and 0. d_stats (NULL = not wanted): [n][groups][2] float32 mean and
 * rstd, both 0 for a board without points. */
int kc_group_norm_act(const kc_group_norm_desc* desc, const void* d_x, const float* d_mask, const float* d_weight,
                      const float* d_bias, void* d_y, float* d_stats, void* d_workspace, size_t workspace_bytes,
                      void* stream);

/* The gradients by x, weight and bias, given dy and the forward pass's x and d_stats: dx (0 at points that are off),
 * d_dweight and d_dbias [channels] float32 (sums over all boards, overwritten; each may be NULL). relu has slope 0
 * at 0. */
int kc_group_norm_act_backward(const kc_group_norm_desc* desc, const void* d_x, const float* d_mask,
                               const float* d_weight, const float* d_bias, const float* d_stats, const void* d_dy,
                               void* d_dx, float* d_dweight, float* d_dbias, void* d_workspace,
                               size_t workspace_bytes, void* stream);

/* Rotary positions with several axes, on Q and K heads. Pair j of a head, j < rotary_dim / 2, is turned by
 * angle[t][table][j] = sum over axes a of pos[t][a] * freqs[table][j][a]; head dimensions from rotary_dim on pass
 * unchanged. The frequencies are the reference's learned table layout (bin2onnx.py :1388-1396: [kv_heads][pairs][2]
 * with the axes x, y); kc_rope_axes_freqs makes fixed ones. */
#define KC_ROPE_HALVES 0 /* pair j = dimensions j and j + rotary_dim / 2 */
#define KC_ROPE_PAIRS 1  /* pair j = dimensions 2 j and 2 j + 1 */
#define KC_ROPE_MAX_AXES 4
typedef struct kc_rope_desc {
  int32_t dtype;   /* KC_PRECISION_* of q, k and their outputs and gradients */
  int32_t layout;  /* KC_ROPE_* */
  int32_t axes;    /* 1 .. KC_ROPE_MAX_AXES */
  int32_t q_heads, k_heads; /* 1 .. 4096, 0 .. 4096; k_heads 0: no k (all k pointers and strides are
                               ignored) */
  int32_t head_dim, rotary_dim; /* rotary_dim even, 2 .. head_dim; head_dim <= 1024 */
  int32_t tables;  /* 1, or a divisor of q_heads and k_heads: head h of H uses table h / (H / tables) */
  int64_t tokens;  /* 0 .. 2^46 */
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
  int64_t q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride;
} kc_rope_desc;

/* The frequencies of fixed rotary positions, into the host array freqs [rotary_dim / 2][axes]: axis a turns
 * sections[a] pairs (the sections add up to rotary_dim / 2; axis 0 has the first ones), pair i of its section by
 * theta^(-i / sections[a]) per step. No device is used. */
int kc_rope_axes_freqs(int axes, const int32_t* sections, double theta, int rotary_dim, float* freqs);

/* Turns q and k: q_out[t][h] = R(angle) q[t][h]. d_pos: [tokens][axes] int32 (any sign), d_freqs:
 * [tables][rotary_dim / 2][axes] float32. Angles are held in 64 bits: positions keep their full resolution. */
int kc_rope_axes(const kc_rope_desc* desc, const void* d_q, const void* d_k, const int32_t* d_pos,
                 const float* d_freqs, void* d_q_out, void* d_k_out, void* stream);

/* The gradients by q and k (turned back by the same angles), and by the frequencies when d_dfreqs is not NULL:
 * d_dq_out, d_dk_out are the gradients of kc_rope_axes' outputs (at q_out's and k_out's strides), d_q and d_k its
 * inputs (only read for d_dfreqs, may be NULL otherwise), d_dq and d_dk the results (at q's and k's strides; in place
 * of d_dq_out / d_dk_out where those strides are the same), d_dfreqs [tables][rotary_dim / 2][axes] float32
 * (overwritten). The workspace is for d_dfreqs only. */
int kc_rope_axes_backward_workspace(const kc_rope_desc* desc, size_t* bytes);
int kc_rope_axes_backward(const kc_rope_desc* desc, const void* d_dq_out, const void* d_dk_out, const void* d_q,
                          const void* d_k, const int32_t* d_pos, const float* d_freqs, void* d_dq, void* d_dk,
                          float* d_dfreqs, void* d_workspace, size_t workspace_bytes, void* stream);

/* Norm of each token's row: n boards of `points` rows of `channels`. The transformer blocks of the nets use the RMS form
 * (bin2onnx.py transformer_rmsnorm :1330-1340), which the engine has inside its forward pass. */
#define KC_NORM_LAYER 0 /* mean and variance of the row */
#define KC_NORM_RMS 1   /* root of the mean square, no mean */
typedef struct kc_layer_norm_desc {
  int32_t dtype; /* KC_PRECISION_* of x, y, dy and dx */
  int32_t kind;  /* KC_NORM_* */
  int32_t n, points, channels; /* n and points 0 .. 2^30 (n * points at most 2^46), channels 1 .. 2^30 */
  float eps;     /* >= 0; with 0 a row of equal values, to float32's rounding (RMS: of zeros), has NaN in y and rstd */
  int64_t x_board_stride, x_row_stride; /* x and dx */
  int64_t y_board_stride, y_row_stride; /* y and dy */
  int64_t mask_board_stride;
} kc_layer_norm_desc;

/* y = (x - mean) * rstd * weight[c] + bias[c] at the tokens whose mask is not 0, 0 at the others (whatever x holds there
 * has no effect), with the mean (0 for RMS) and rstd = 1 / sqrt(mean square distance from it + eps) of the token's row.
 * Squares are summed in float32: a row whose sum passes 3.4e38 has NaN in y and rstd. d_mask: [n][points] float32 rows
 * at mask_board_stride, NULL = every token; d_weight, d_bias: [channels] float32, NULL = 1 and 0. d_stats (NULL = not
 * wanted): [n][points][2] float32 mean and rstd, both 0 where the token is off. */
int kc_layer_norm(const kc_layer_norm_desc* desc, const void* d_x, const float* d_mask, const float* d_weight,
                  const float* d_bias, void* d_y, float* d_stats, void* stream);

/* The gradients by x, weight and bias, given dy and the forward pass's x and d_stats: dx (0 at tokens that are off; in
 * place of x, or of dy where the strides are the same), d_dweight and d_dbias [channels] float32 (sums over all tokens,
 * added in float32, overwritten; each may be NULL). (x - mean) * rstd is taken from the saved float32 mean: it is off
 * by up to |mean| * rstd * 2^-24, the same in a whole row. The workspace is for d_dweight and d_dbias only. */
int kc_layer_norm_backward_workspace(const kc_layer_norm_desc* desc, size_t* bytes);
int kc_layer_norm_backward(const kc_layer_norm_desc* desc, const void* d_x, const float* d_mask, const float* d_weight,
                           const float* d_stats, const void* d_dy, void* d_dx, float* d_dweight, float* d_dbias,
                           void* d_workspace, size_t workspace_bytes, void* stream);

/* Learned rows looked up by token: y[t] = x[t] + scale * table[id[t]]. Points, moves or states of a token, the learned
 * counterpart of rotary positions. */
typedef struct kc_embed_desc {
  int32_t dtype;      /* KC_PRECISION_* of table, x, y and dy */
  int32_t channels;   /* 1 .. 2^20 */
  int64_t tokens;     /* 0 .. 2^30 */
  int64_t table_rows; /* 1 .. 2^30 */
  float scale;        /* finite */
  int32_t reserved;   /* 0 */
  int64_t table_stride, x_stride, y_stride; /* elements from one row to the next; y_stride is dy's too */
} kc_embed_desc;

/* d_ids: [tokens] int32. An id outside 0 .. table_rows - 1 (padding) adds nothing: y[t] = x[t]. d_x NULL = 0; y may be
 * x (same pointer and stride). The gradient by x is dy itself. */
int kc_embed_rows(const kc_embed_desc* desc, const int32_t* d_ids, const void* d_table, const void* d_x, void* d_y,
                  void* stream);

/* The table's gradient, d_dtable [table_rows][channels] float32 (overwritten): scale times the sum of dy over the tokens
 * that have the row's id, added in float32, in the tokens' order within pieces of a fixed length; 0 for a row that none
 * has. table_stride and x_stride are ignored. */
int kc_embed_rows_backward_workspace(const kc_embed_desc* desc, size_t* bytes);
int kc_embed_rows_backward(const kc_embed_desc* desc, const int32_t* d_ids, const void* d_dy, float* d_dtable,
                           void* d_workspace, size_t workspace_bytes, void* stream);

/* Distillation: the loss of a student's logits (policy rows of 362 moves, or any classes) against a teacher's top
 * logits. With q = softmax(logits / T) and p[j] = exp(top_logits[j] / T - L) over the row's entries j,
 *   loss = T^2 * sum over j of p[j] * (log p[j] - log q[id[j]]),
 * L = the entries' own log sum of exp(top_logits / T) (p adds up to 1), or d_teacher_log_sum[row], the teacher's over
 * all its classes (p adds up to what the entries hold of it; the rest of the teacher's distribution is left out).
 * Exponentials and their sums are float32, off by up to 2^-16 of themselves (rows of up to 131,072 classes; 2^-18 up to
 * 2,048): the loss is off by up to that times T^2 * sum of p, the gradient by up to that times dloss * T * (q + p). The
 * loss of a student near its teacher does not grow with T, hence the limit of T. */
typedef struct kc_distill_desc {
  int32_t dtype;     /* KC_PRECISION_* of logits and dlogits */
  int32_t classes;   /* 1 .. 2^30 */
  int64_t rows;      /* 0 .. 2^30 */
  int32_t top;       /* 1 .. 1024 entries of a row */
  float temperature; /* T, 2^-20 .. 32 */
  int64_t logits_stride, dlogits_stride; /* elements from one row to the next */
  int64_t top_stride;                    /* of d_ids and of d_top_logits */
} kc_distill_desc;

/* d_ids: [rows][top] int32, d_top_logits: [rows][top] float32. An entry whose id is outside 0 .. classes - 1 or whose
 * logit is -inf is absent; entries of one class add up. A row without entries has loss 0 and gradient 0, whatever its
 * logits hold. Logits of -inf (illegal moves) have probability 0: an entry there makes the loss infinite, unless its p
 * is below about 1e-300, which counts as 0. NaN among a row's logits, +inf, or nothing but -inf make its loss NaN, and
 * so does NaN or +inf as an entry's logit, with all of the row's gradient. d_loss: [rows] float32. d_stats (NULL = not
 * wanted): [rows][2] float32, the row's largest logit and the sum of exp((logit - largest) / T), both 0 without
 * entries. */
int kc_distill_top(const kc_distill_desc* desc, const void* d_logits, const int32_t* d_ids, const float* d_top_logits,
                   const float* d_teacher_log_sum, float* d_loss, float* d_stats, void* stream);

/* The gradient by the logits, dlogits[i] = dloss * T * (q[i] * sum of p - sum of p[j] at id[j] = i), given the forward
 * pass's inputs and d_stats. d_dloss: [rows] float32, NULL = 1. dlogits may be the logits (same pointer and stride). */
int kc_distill_top_backward(const kc_distill_desc* desc, const void* d_logits, const int32_t* d_ids,
                            const float* d_top_logits, const float* d_teacher_log_sum, const float* d_stats,
                            const float* d_dloss, void* d_dlogits, void* stream);

/* Failure-detection self-test. Every spin-wait in this library's kernels is bounded: when a wait runs out, the
 * kernel records an error code in the handle's device error word, releases what it holds and returns, and the next
 * kc_wait / kc_synchronize reports KC_ERR_DEVICE (the handle stays usable). This enqueues on the handle's stream
 * one kernel that makes the same bounded wait on a barrier nothing completes, with a limit of `limit_us`
 * microseconds (1 .. 2,000,000) instead of the forward pass's 2 s, so that a caller can check the whole error path
 * without a fault. No counterpart in the reference, whose kernels have no bounded waits. */
int kc_selftest_device_timeout(kc_handle* h, int limit_us);

/* Host-side symmetry helpers of the reference (nninputs.rs:756-879), exported for tests of the host logic.
 * NCHW copy of one row with `c_size` channels; `reverse` = copyOutputsWithSymmetry semantics. */
int kc_copy_with_symmetry(const float* src, float* dst, int n_size, int h_size, int w_size, int c_size,
                          int symmetry, int reverse);

#ifdef __cplusplus
}
#endif

#endif /* KATAGO_CUDA_H */
