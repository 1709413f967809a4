/*
 * ctmr_b200 — C ABI of the B200 (sm_100a) convolution stack that replaces the
 * reference's native path in mlx-generate-ctmr (v0.7.0):
 *   implicit-GEMM Conv3d (3x3x3 pad 1 / 1x1x1, stride 1 / 2, nearest-2x and
 *   trilinear-2x inputs) with the group-norm affine, SiLU, 2x average pool and
 *   a two-tensor channel concat fused into its input preparation, and the bias
 *   (per channel or per batch item) and residual add fused into its epilogue,
 *   plus the GroupNorm statistics that feed it.
 *
 * Conventions
 *   - Activations are channels-last (NDHWC): voxel rows of `channels` values,
 *     `cstride` elements apart (a view into a wider row is allowed). The
 *     reference's Python surface is NCDHW; torch's channels_last_3d storage of
 *     an NCDHW tensor is exactly this layout.
 *   - Weights use the Torch layout (O, C, k, k, k), fp32, and are packed once
 *     with ctmr_pack_weight.
 *   - Every call is asynchronous on `stream` (a cudaStream_t, NULL = legacy
 *     default stream) and returns a status code; nothing throws across the ABI.
 *   - No call allocates device memory: the caller passes workspace buffers
 *     whose sizes the *_workspace_size functions return.
 *   - All device-side waits are bounded; a kernel that gives up sets a bit in
 *     the library's device error word (ctmr_get_device_error) instead of hanging.
 */
#ifndef CTMR_B200_H
#define CTMR_B200_H

#include <stddef.h>

#if defined(__GNUC__)
#define CTMR_API __attribute__((visibility("default")))
#else
#define CTMR_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. CTMR_ERR_INVALID corresponds to the reference's ValueError
 * for shape/dtype mismatches (`_nax_conv.py:523-526, 537-541, 559-560`). */
enum {
  CTMR_OK = 0,
  CTMR_ERR_INVALID = 1,
  CTMR_ERR_UNSUPPORTED = 2,
  CTMR_ERR_WORKSPACE = 3,
  CTMR_ERR_CUDA = 4
};

enum {
  CTMR_DTYPE_F32 = 0,
  CTMR_DTYPE_BF16 = 1,
  CTMR_DTYPE_F16 = 2,    /* ctmr_transform outputs only */
  /* Conv input `x` only: one int16 label id per voxel (cstride elements apart), read as 8
   * channels, channel k = bit k of the id (0.0 or 1.0): the ControlNet condition of
   * `condition.binarize_labels_ncdhw` (`condition.py:20-43`) formed in the operand pass.
   * channels must be 8; no x2, resampling or in-call GroupNorm. */
  CTMR_DTYPE_LABEL8 = 3
};

/* CTMR_PRECISION_FP32: fp32 operands carried as fp16 hi/lo pairs, three
 *   tensor-core products per step, fp32 accumulation (~2^-22 relative product
 *   error; needs |value| < 65504), the reference's "exact" mode
 *   (`_nax_conv.py:27-35`).
 * CTMR_PRECISION_BF16: bf16 operands, fp32 accumulation.
 * CTMR_PRECISION_FP16: fp16 operands (needs |value| < 65504), fp32 accumulation;
 *   the same tensor-core rate as bf16 with 3 more mantissa bits.
 * CTMR_PRECISION_TF32: operands rounded to TF32 (fp32 range, 10 mantissa bits,
 *   stored as fp32), fp32 accumulation, at half the 16-bit tensor-core rate: the
 *   TF32-input mode beside the reference's exact mode. */
enum { CTMR_PRECISION_FP32 = 0, CTMR_PRECISION_BF16 = 1, CTMR_PRECISION_FP16 = 2, CTMR_PRECISION_TF32 = 3 };

/* An NDHWC activation view. data == NULL means "absent". */
typedef struct ctmr_tensor {
  const void* data;
  int dtype;            /* CTMR_DTYPE_* */
  int channels;
  long long cstride;    /* elements between consecutive voxel rows, >= channels */
} ctmr_tensor;

/* One convolution: y = conv(prepare(x ++ x2)) + bias (+ residual).
 * Replaces `nax_conv3d(x, packed, bias, *, affine, silu, stride, upsample,
 * trilinear, residual, mx)` (`_nax_conv.py:475-487`) together with the 1x1x1
 * route of `fast_fp32.pointwise_conv_ncdhw` (`fast_fp32.py:121-130`) and the
 * pooled conv1 of `fast_fp32.residual_block_ncdhw` (`fast_fp32.py:250-265`). */
typedef struct ctmr_conv3d_desc {
  int batch, depth, height, width; /* grid of x (and x2) */
  ctmr_tensor x;
  ctmr_tensor x2;                  /* optional second input, concatenated after x's channels */
  int out_channels;
  int kernel_size;                 /* 3 (padding 1) or 1 */
  int stride;                      /* 1, or 2 with kernel_size 3 */
  int upsample;                    /* convolve the nearest-2x upsampling of x (weights packed with upsample=1) */
  int trilinear;                   /* convolve the half-pixel trilinear-2x upsampling of x */
  int avgpool;                     /* convolve the 2x2x2 mean of silu?(affine?(x)) */
  int precision;                   /* CTMR_PRECISION_* */
  const void* weight;              /* ctmr_pack_weight output (bf16 / fp16, or the fp16 hi plane) */
  const void* weight_lo;           /* fp16 lo plane for CTMR_PRECISION_FP32 */
  const float* affine;             /* (batch, C, 2) (scale, offset) pairs, or NULL */
  int silu;                        /* apply SiLU after the affine */
  const float* bias;               /* (out_channels) or (batch, out_channels), or NULL */
  int bias_per_batch;
  ctmr_tensor residual;            /* optional, on the output grid (half grid if residual_upsampled) */
  int residual_upsampled;          /* residual is nearest-2x upsampled on the fly */
  void* y;                         /* NDHWC output on the output grid */
  int y_dtype;
  long long y_cstride;
  int y_coffset;                   /* first channel written in each output row */
  /* Optional GroupNorm statistics of the output, for ctmr_group_norm_affine_from_stats:
   * float[batch][stats_slots][out_channels][3] moments (count, mean, M2) per
   * (batch item, slot, channel). stats_slots must be ctmr_conv3d_stats_slots(desc)
   * (> 0). Null: none. */
  float* stats;
  int stats_slots;
  /* Optional GroupNorm of the input computed inside the call (instead of passing
   * `affine`): gamma/beta per input channel (NULL: 1/0), gn_groups > 0 groups over
   * x ++ x2, gn_eps. The statistics are those of ctmr_group_norm_affine, reduced by
   * the call before its operand pass (with CTMR_GN_FUSED=1 in the environment, small
   * tensors use one kernel that reduces them and writes the operand). `affine` must
   * be NULL. */
  const float* gn_gamma;
  const float* gn_beta;
  int gn_groups;
  float gn_eps;
  /* Elements between consecutive batch items' rows of a per-batch bias (0: out_channels,
   * i.e. a dense (batch, out_channels) array; otherwise >= out_channels, e.g. a column
   * slice of a wider (batch, N) table). */
  long long bias_row_stride;
} ctmr_conv3d_desc;

/* Packed-weight element count per plane for a Torch (O, C, k, k, k) weight:
 * taps x round16(O) x round16(C), taps = k^3, or 64 with upsample.
 * Replaces the shapes of `pack_weight` / `pack_upsample_weight` (`_nax_conv.py:391-445`). */
CTMR_API size_t ctmr_packed_weight_elems(int out_channels, int in_channels, int kernel_size, int upsample);

/* Bytes of one packed-weight plane in `precision`: 2 x ctmr_packed_weight_elems in the 16-bit
 * and split modes; for CTMR_PRECISION_TF32, taps x round16(O) x round8(C) fp32 values. The
 * size counterpart of `pack_weight` (`_nax_conv.py:391-404`) per precision; 0 when invalid. */
CTMR_API size_t ctmr_packed_weight_bytes(int out_channels, int in_channels, int kernel_size, int upsample,
                                         int precision);

/* Pack an fp32 Torch-layout weight (device pointer). bf16 for CTMR_PRECISION_BF16,
 * fp16 for CTMR_PRECISION_FP16, TF32-rounded fp32 for CTMR_PRECISION_TF32 (packed_lo
 * unused), fp16 hi/lo planes for CTMR_PRECISION_FP32.
 * Replaces `pack_weight` (`_nax_conv.py:391-404`) and, with upsample = 1,
 * `pack_upsample_weight` (`_nax_conv.py:407-445`). */
CTMR_API int ctmr_pack_weight(const float* weight, int out_channels, int in_channels, int kernel_size, int upsample,
                     int precision, void* packed, void* packed_lo, void* stream);

/* ctmr_pack_weight for a weight stored channels-last, (O, k, k, k, C) (device pointer): the
 * layout of released safetensors checkpoints, which the reference transposes to Torch
 * layout on load (`weights.py:152-156`, LAYOUT_CONV3D_W); packed here without that copy.
 * Same packed result, bit for bit. */
CTMR_API int ctmr_pack_weight_channels_last(const float* weight, int out_channels, int in_channels,
                     int kernel_size, int upsample, int precision, void* packed, void* packed_lo,
                     void* stream);

/* Multi-head self-attention with head size 32, out = softmax(Q K^T * scale) V per head, on
 * the tensor cores in one flash-attention pass. `qkv` is the fused projection (batch, tokens,
 * 3 * heads * 32) of 16-bit values (dtype CTMR_DTYPE_BF16, or CTMR_DTYPE_F16 for fp16),
 * contiguous, head h at columns h*32 (q), C + h*32 (k), 2C + h*32 (v); `out` is
 * (batch, tokens, heads * 32) of the same type. tokens must be a multiple of 128.
 * Replaces `_flash_attention.flash_attention` (`_flash_attention.py:320-360`) as called by
 * `fast_fp32.self_attention_tokens` (`fast_fp32.py:352-396`). */
CTMR_API int ctmr_attention_d32(const void* qkv, int dtype, int batch, int tokens, int heads, float scale, void* out,
                       void* stream);

/* Workspace bytes ctmr_conv3d needs for this descriptor (the prepared operand). */
CTMR_API size_t ctmr_conv3d_workspace_size(const ctmr_conv3d_desc* desc);

/* Replaces `nax_conv3d` (`_nax_conv.py:475-684`): operand preparation (when
 * needed) followed by the implicit-GEMM kernel. */
CTMR_API int ctmr_conv3d(const ctmr_conv3d_desc* desc, void* workspace, size_t workspace_bytes, void* stream);

/* The two launches of ctmr_conv3d separately, as the reference's pack and
 * GEMM kernels are (`_nax_conv.py:583-646`): stages = CTMR_CONV_PREPARE,
 * CTMR_CONV_GEMM or both. The GEMM stage reads the operand a previous
 * PREPARE stage left in the same workspace. */
enum { CTMR_CONV_PREPARE = 1, CTMR_CONV_GEMM = 2 };
CTMR_API int ctmr_conv3d_stages(const ctmr_conv3d_desc* desc, void* workspace, size_t workspace_bytes, int stages,
                                void* stream);

/* The convolution of ctmr_conv3d for callers that cannot allocate device
 * memory. (No counterpart in the reference: its MLX runtime allocates every
 * buffer itself.) Plugins living inside another framework's memory pool and
 * real-time or safety-constrained callers whose allocations are all made up
 * front cannot call cudaMalloc for the workspace ctmr_conv3d needs; this
 * variant takes that scratch from one static device
 * array of CTMR_CONV3D_NOALLOC_SCRATCH_BYTES that every GPU loading the
 * library holds until exit, and allocates nothing.
 *   - Inputs and outputs are passed exactly as for ctmr_conv3d.
 *   - Convolutions whose prepared operand (ctmr_conv3d_workspace_size) exceeds
 *     the scratch are rejected with CTMR_ERR_WORKSPACE, nothing launched.
 *   - The first call on a device looks up the array's address on that device
 *     (cudaGetSymbolAddress); make it before any stream capture.
 *   - All calls share the array and it keeps the last call's contents; nothing
 *     in it needs to start at zero. Calls whose kernels overlap on the GPU
 *     (unordered streams) race on it and must not be issued. */
#define CTMR_CONV3D_NOALLOC_SCRATCH_BYTES (32u << 20)
CTMR_API int ctmr_conv3d_noalloc(const ctmr_conv3d_desc* desc, void* stream);

/* Workspace bytes for ctmr_group_norm_affine. */
CTMR_API size_t ctmr_group_norm_workspace_size(int batch, long long voxels, int groups);

/* GroupNorm statistics of (x ++ x2) over each (batch item, group) ->
 * affine[b][c] = (gamma[c] * rstd, beta[c] - mean * gamma[c] * rstd), fp32.
 * Replaces `medmlx_core.group_norm.group_norm_affine` (called at `fast_fp32.py:183-189`;
 * layout (B*C*2) consumed at `_nax_conv.py:174-176`). gamma/beta may be NULL (1/0). */
CTMR_API int ctmr_group_norm_affine(ctmr_tensor x, ctmr_tensor x2, int batch, long long voxels, const float* gamma,
                           const float* beta, int groups, float eps, float* affine, void* workspace,
                           size_t workspace_bytes, void* stream);

/* The GroupNorm statistics of ctmr_group_norm_affine stopped before the affine: the merged
 * (count, mean, M2) of each (batch item, group) of (x ++ x2), float moments[batch][groups][3].
 * Same workspace as ctmr_group_norm_affine. For a tensor split across devices (depth shards
 * of one volume, each holding `voxels` of it): each part computes its moments, the parts
 * exchange them, and ctmr_group_norm_affine_from_moments forms the affine of the whole
 * tensor. The reference normalises whole tensors only (`fast_fp32.py:183-189`); this is the
 * same statistic, split at the boundary between the two kernels of its computation. */
CTMR_API int ctmr_group_norm_moments(ctmr_tensor x, ctmr_tensor x2, int batch, long long voxels, int groups,
                                     float* moments, void* workspace, size_t workspace_bytes, void* stream);

/* The affine of group_norm_affine (`fast_fp32.py:183-189`) from the moments of `parts` parts
 * of one tensor, float moments[parts][batch][groups][3] (1 <= parts <= 64), merged in part
 * order in double precision, so every caller holding the same moments gets the same affine. */
CTMR_API int ctmr_group_norm_affine_from_moments(const float* moments, int parts, int batch, int channels,
                                                 const float* gamma, const float* beta, int groups, float eps,
                                                 float* affine, void* stream);

/* Kernel launches one ctmr_conv3d call with this descriptor issues (instrumentation;
 * no reference counterpart), or 0 for an invalid descriptor. */
CTMR_API int ctmr_conv3d_launch_count(const ctmr_conv3d_desc* desc);

/* Kernel launches one ctmr_group_norm_affine call over `voxels` voxels per batch item and
 * `channels` channels in `groups` groups issues for dense, 16-byte aligned fp32 sources: 1 for
 * small groups (one block per group and batch item computes the affine directly), 2 otherwise
 * (partials, then the merge); 0 for invalid extents. Instrumentation; no reference counterpart. */
CTMR_API int ctmr_group_norm_launch_count(long long voxels, int channels, int groups);

/* Statistics slots a convolution writes when desc->stats is set, or 0 when this
 * convolution does not produce them. The kh-concatenated persistent kernel (16-bit
 * operands, stride-1 3x3x3, 64 padded output channels) writes four per SM, one per
 * epilogue lane quarter of each CTA; the atom-shifted persistent kernel (at least 128
 * output channels, batch x out_channels <= 512) one per SM; other routes none. Has no
 * reference counterpart: the reference recomputes the statistics from the tensor. */
CTMR_API int ctmr_conv3d_stats_slots(const ctmr_conv3d_desc* desc);

/* The affine of ctmr_group_norm_affine from convolution output statistics instead
 * of a pass over the tensor: stats_a (channels_a) ++ stats_b (channels_b, may be
 * NULL with channels_b 0) in the ctmr_conv3d_desc.stats layout, each with `slots`
 * slots. Same result definition as `group_norm_affine` (`fast_fp32.py:183-189`);
 * the moments are merged in double precision in a fixed order. */
CTMR_API int ctmr_group_norm_affine_from_stats(const float* stats_a, int channels_a, const float* stats_b,
                                               int channels_b, int slots, int batch, const float* gamma,
                                               const float* beta, int groups, float eps, float* affine,
                                               void* stream);

enum { CTMR_TRANSFORM_COPY = 0, CTMR_TRANSFORM_TRILINEAR = 1, CTMR_TRANSFORM_AVGPOOL = 2 };

/* y = mode(silu?(affine?(x ++ x2))) materialised as fp32 or bf16 NDHWC, channels
 * past the input zero-filled up to y_channels. Replaces the materialising ops of
 * the operator surface: `fast_fp32.group_norm_ncdhw` (`fast_fp32.py:102-118`),
 * `silu`, `avg_pool3d_ncdhw` and `upsample_trilinear_ncdhw` (`source_vae.py:95-111`). */
typedef struct ctmr_transform_desc {
  int batch, depth, height, width; /* grid of x */
  ctmr_tensor x;
  ctmr_tensor x2;
  int mode;                        /* CTMR_TRANSFORM_* */
  const float* affine;
  int silu;
  void* y;
  int y_dtype;
  int y_channels;
  long long y_cstride;
} ctmr_transform_desc;

CTMR_API int ctmr_transform(const ctmr_transform_desc* desc, void* stream);

/* (B, C, S) <-> (B, S, C) layout change (NCDHW <-> NDHWC), fp32/bf16 in and out. */
CTMR_API int ctmr_ncdhw_to_ndhwc(const void* x, int x_dtype, void* y, int y_dtype, int batch, int channels,
                        long long voxels, void* stream);
CTMR_API int ctmr_ndhwc_to_ncdhw(const void* x, int x_dtype, void* y, int y_dtype, int batch, int channels,
                        long long voxels, void* stream);

/* Sliding-window blend (`decode.py:115-184`): acc += pred * w, wsum += w over one
 * window at (z0, y0, x0) of the output grid, w = max(gz[z/scale] gy[y/scale] gx[x/scale], floor). */
CTMR_API int ctmr_window_accumulate(ctmr_tensor pred, int batch, int wd, int wh, int ww, int z0, int y0, int x0,
                           int od, int oh, int ow, const float* gz, const float* gy, const float* gx, int scale,
                           float floor_value, float* acc, float* wsum, void* stream);

/* out (NCDHW, B x C x cd x ch x cw) = acc / wsum over the crop at (cz0, cy0, cx0). */
CTMR_API int ctmr_window_finalize(const float* acc, const float* wsum, float* out, int batch, int channels, int od, int oh,
                         int ow, int cz0, int cy0, int cx0, int cd, int ch, int cw, void* stream);

/* Guided Euler step of the rectified-flow sampler (`image.py:163-175`, `rflow.py:101-121`):
 * v = vel[n:] + guidance * (vel[:n] - vel[n:]) when guided, else vel[:n]; out = z + v * dt.
 * When dt_device is not NULL the step reads dt from that device scalar instead
 * (so one captured CUDA graph serves every step). out may alias z. */
CTMR_API int ctmr_rflow_step(const float* z, const float* vel, long long n, float guidance, int guided, float dt,
                             const float* dt_device, float* out, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Packed tokens: several requests (volumes of different extents) in one call. `offsets` are int32
 * values in device memory, documents + 1 of them, not falling: document d holds the rows
 * [offsets[d], offsets[d + 1]) of the packed tensor. The host never reads them; the kernels clamp
 * them into the tensor, and what a clamp changed sets bit 5 of the device error word
 * (ctmr_get_device_error). The reference runs one request at a time and has no counterpart. */

/* Rotary positions along several axes. A head's first 2 * (section[0] + .. + section[axes - 1])
 * channels are rotated in pairs, (2c, 2c + 1) when interleaved, (c, c + pairs) otherwise, the rest
 * copied. Pair c of axis a: angle = positions[token][a] * inv_freq[c] (the product and its reduction
 * to a turn in 64 bits), (u, v) -> (u cos - v sin, v cos + u sin); inverse: the opposite angle (the
 * transpose, which carries gradients back). Any strides; y may be x. */
#define CTMR_MAX_ROTARY_AXES 8
typedef struct ctmr_rotary_desc {
  const void* x;                   /* (tokens, heads, head_dim), channels contiguous */
  void* y;
  int dtype;                       /* CTMR_DTYPE_F32, _BF16 or _F16 */
  long long tokens;
  int heads, head_dim;
  long long x_token_stride, x_head_stride, y_token_stride, y_head_stride; /* elements */
  const void* positions;           /* (tokens, axes), rows positions_stride elements apart */
  int positions_f32;               /* fp32 positions; int32 otherwise */
  long long positions_stride;
  const float* inv_freq;           /* one per pair */
  int axes;                        /* 1 .. CTMR_MAX_ROTARY_AXES */
  int section[CTMR_MAX_ROTARY_AXES]; /* pairs of each axis */
  int interleaved;
  int inverse;
} ctmr_rotary_desc;
CTMR_API int ctmr_rotary_axes(const ctmr_rotary_desc* desc, void* stream);

/* A projection shared by all rows and a low-rank adapter for each segment of rows:
 *   y_i = weight x_i + bias + scale[a] * up[a] (down[a] x_i),  a = index[segment of row i],
 * without the adapter's term where a is negative or no segment holds the row. 16-bit operands,
 * fp32 sums; the adapter's inner product (scaled) is rounded once to the operands' type, whose range it must
 * not leave (fp16: 65,504). Infinities and NaN stay in the rows and outputs that the formula gives them to:
 * an adapter that holds some does not touch the rows of other segments. */
typedef struct ctmr_adapter_linear_desc {
  const void* x;                   /* (rows, in_features), rows x_stride elements apart */
  long long x_stride;              /* a multiple of 8 */
  int dtype;                       /* CTMR_DTYPE_BF16 or _F16: x, weight, down, up and y */
  int rows, in_features, out_features; /* in_features a multiple of 8 */
  const void* weight;              /* (out_features, in_features), rows weight_stride elements apart */
  long long weight_stride;
  const void* bias;                /* (out_features) or NULL */
  int bias_dtype;                  /* CTMR_DTYPE_F32 or dtype */
  const void* down;                /* (adapters, rank, in_features), dense */
  const void* up;                  /* (adapters, out_features, rank), dense */
  const float* scale;              /* (adapters) */
  int adapters, rank;              /* rank: a multiple of 8 up to 128 */
  const int* offsets;              /* (segments + 1) */
  const int* index;                /* (segments): the segment's adapter; negative: none */
  int segments;                    /* 0: no adapters (the fields above are not read) */
  void* y;                         /* (rows, out_features), rows y_stride elements apart; not x */
  long long y_stride;
} ctmr_adapter_linear_desc;
CTMR_API size_t ctmr_adapter_linear_workspace_size(const ctmr_adapter_linear_desc* desc);
CTMR_API int ctmr_adapter_linear(const ctmr_adapter_linear_desc* desc, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* out_i = sum_j softmax_j(s_ij) v_j over the keys j that query i sees, in its own document:
 *   s_ij = cap(scale q_i . k_j) - slopes[head] * |p_i - j|,  p_i = i + Lk - Lq,
 * i and j counted inside the document of Lq queries and Lk keys, cap(x) = cap * tanh(x / cap) (x when
 * cap is 0). Not causal: every key of the document is seen. Causal: j <= p_i, or j < prefix[document].
 * A query that sees nothing gets zeros (and lse -infinity). Query head h reads key head
 * h / (heads / kv_heads). Sums and softmax statistics are fp32; the softmax weights are rounded to
 * the operands' type for their product with v.
 *
 * Two forms. Packed: q_offsets and k_offsets given, q_tokens and k_tokens the packed totals, document
 * strides unused; rows of q before the first document or past the last give zeros (and lse -infinity).
 * Batched: both NULL, each document has q_tokens queries and k_tokens key rows, of
 * which the first k_lengths[document] are used (all when NULL). Values of keys outside the used ones
 * are never part of a result, whatever they are; values of used keys must be finite. */
typedef struct ctmr_attention_desc {
  const void *q, *k, *v;           /* [document][token][head][head_dim], channels contiguous */
  void* out;
  float* lse;                      /* ([document][token][heads]) natural log of the softmax sum, or NULL */
  int dtype;                       /* CTMR_DTYPE_BF16 or _F16 */
  int documents, q_tokens, k_tokens;
  int heads, kv_heads, head_dim;   /* head_dim: a multiple of 8 up to 128 */
  /* Element strides, multiples of 8; addresses 16-byte aligned. */
  long long q_doc_stride, q_token_stride, q_head_stride;
  long long k_doc_stride, k_token_stride, k_head_stride;
  long long v_doc_stride, v_token_stride, v_head_stride;
  long long out_doc_stride, out_token_stride, out_head_stride;
  const int *q_offsets, *k_offsets; /* (documents + 1) each, or both NULL */
  const int* k_lengths;            /* (documents), batched form only, or NULL */
  const int* prefix;               /* (documents), causal only, or NULL */
  const float* slopes;             /* (heads), or NULL */
  float scale;                     /* positive */
  float cap;                       /* 0: none */
  int causal;
  int max_q;                       /* packed form: no document has more queries (0: not known) */
} ctmr_attention_desc;
CTMR_API int ctmr_attention(const ctmr_attention_desc* desc, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Rows in 8 bits: e4m3 values with a scale for every 128 channels, the last group maybe shorter. The
 * scale of a group is the least power of two 2^k, k >= -100, with which its largest magnitude is at most
 * 448, and value = e4m3(v / scale) to nearest, ties to even: the bytes of v's formula in 64 bits. A group that
 * holds an infinity, a NaN or a value past 448 * 2^127 (no scale of fp32 reaches further) becomes NaN as a whole.
 * Strides in elements (bytes for 8-bit values); rows of inputs may overlap one another, rows of outputs not. */

/* Root-mean-square norm of rows: h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, and h itself,
 * rounded to x's type, in `sum`. A row is (token, head): heads is 1 for (tokens, channels). y is of x's
 * type, or in 8 bits where scale is not NULL (heads must then be 1). The norm is taken of h before it is
 * rounded to x's type; squares are added in 64 bits. Of 16-bit x, h is the sum in fp32, exact unless one term is
 * 2^13 times the other; past fp32's range it is an infinity. The bytes are exact for rows of a root mean square
 * up to 2^126 and weights up to 2^15; beyond, values within 2^-20 of a tie may fall to either side, and what
 * h / sqrt(...) has below 2^-126 is lost. sum may be x or residual, and y of x's type may be x or residual
 * (not sum); other overlaps are not allowed. */
typedef struct ctmr_rms_norm_desc {
  const void* x;                   /* [token][head][channels], channels contiguous */
  const void* residual;            /* like x, or NULL */
  const void* weight;              /* (channels), dense, or NULL */
  int dtype;                       /* CTMR_DTYPE_F32, _BF16 or _F16: x, residual, sum, and y without scale */
  int weight_dtype;                /* CTMR_DTYPE_F32 or dtype */
  int tokens, heads, channels;     /* channels: up to 32768 */
  long long x_token_stride, x_head_stride, residual_token_stride, residual_head_stride;
  float eps;                       /* positive */
  void* y;
  long long y_token_stride, y_head_stride;
  void* sum;                       /* or NULL */
  long long sum_token_stride, sum_head_stride;
  float* scale;                    /* (tokens, groups), or NULL */
  long long scale_token_stride, scale_group_stride;
} ctmr_rms_norm_desc;
CTMR_API int ctmr_rms_norm(const ctmr_rms_norm_desc* desc, void* stream);

/* Rows to 8 bits: v = x, or with gate v = silu(a) * b, a the first `channels` of a row and b the next. */
typedef struct ctmr_quantize_rows_desc {
  const void* x;                   /* (rows, channels), (rows, 2 * channels) with gate */
  int dtype;                       /* CTMR_DTYPE_F32, _BF16 or _F16 */
  int rows, channels;
  int gate;
  long long x_stride;
  void* values;                    /* (rows, channels) e4m3; not x */
  long long values_stride;
  float* scale;                    /* (rows, groups) */
  long long scale_row_stride, scale_group_stride;
} ctmr_quantize_rows_desc;
CTMR_API int ctmr_quantize_rows(const ctmr_quantize_rows_desc* desc, void* stream);

/* The product of 8-bit rows with an 8-bit weight, fp32 sums:
 *   y_mn = sum_b x_scale[m][b] weight_scale[n / 128][b] (sum of x_mk weight_nk over block b of 128 inputs) + bias_n,
 * scales of any value; the product of a row's and a weight's scale must be in fp32's normal range. What is NaN or
 * not finite in a row, or in an output's weights, stays in that row, or output. Values and weights are e4m3,
 * 16-byte aligned, rows a multiple of 16 bytes apart; inputs, outputs and rows of any number. */
typedef struct ctmr_scaled_linear_desc {
  const void* x;                   /* (rows, in_features) e4m3 */
  long long x_stride;
  const float* x_scale;            /* (rows, in blocks), strides in elements */
  long long x_scale_row_stride, x_scale_block_stride;
  int rows, in_features, out_features;
  const void* weight;              /* (out_features, in_features) e4m3 */
  long long weight_stride;
  const float* weight_scale;       /* (out blocks, in blocks) */
  long long weight_scale_row_stride, weight_scale_block_stride;
  const void* bias;                /* (out_features) or NULL */
  int bias_dtype;                  /* CTMR_DTYPE_F32 or y_dtype */
  void* y;                         /* (rows, out_features), rows y_stride elements apart */
  int y_dtype;                     /* CTMR_DTYPE_F32, _BF16 or _F16 */
  long long y_stride;
} ctmr_scaled_linear_desc;
CTMR_API int ctmr_scaled_linear(const ctmr_scaled_linear_desc* desc, void* stream);

/* Device error word (bits 0-4 set when a bounded wait gave up or a launch was inconsistent, bit 5 when
 * offsets, lengths or adapter numbers in device memory were out of range); optionally cleared.
 * Synchronises the current device. */
CTMR_API int ctmr_get_device_error(unsigned* bits, int clear);

CTMR_API const char* ctmr_status_string(int status);

/* Human-readable reason of the last failed call on this thread. */
CTMR_API const char* ctmr_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* CTMR_B200_H */
