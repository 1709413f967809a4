// The extern "C" entry points of the 8-bit row operators: argument checks and dispatch.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"

namespace {

using ctmr::api_fail;

bool float_type(int dtype) { return dtype == CTMR_DTYPE_F32 || dtype == CTMR_DTYPE_BF16 || dtype == CTMR_DTYPE_F16; }

bool aligned_to(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == CTMR_DTYPE_F32 ? 4 : 2) == 0;
}

long long scale_groups(int channels) { return (channels + ctmr::kScaleGroup - 1LL) / ctmr::kScaleGroup; }

bool stride_ok(long long s) { return s >= 0 && s < (1LL << 38); }

// Whether rows of `width` elements at i a + j b, i < na and j < nb, lie apart from one another.
bool rows_apart(long long na, long long a, long long nb, long long b, long long width) {
  if (na > 1 && nb > 1 && a > b) return rows_apart(nb, b, na, a, width);
  if (na > 1 && a < width) return false;
  if (nb > 1 && b < width) return false;
  if (na <= 1 || nb <= 1) return true;
  const __int128 end = static_cast<__int128>(a) * (na - 1) + width;  // of j = 0
  // Where rows of different j lie between one another, each j's start against its neighbours of j = 0.
  __int128 at = b;
  for (long long j = 1; j < nb && at < end; ++j, at += b) {
    const __int128 i = at / a, after = (i + 1) * a - at;
    if (i < na && at - i * a < width) return false;
    if (i + 1 < na && after < width) return false;
  }
  return true;
}

int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? CTMR_OK : api_fail(CTMR_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int ctmr_rms_norm(const ctmr_rms_norm_desc* d, void* stream) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (!float_type(d->dtype)) return api_fail(CTMR_ERR_INVALID, "rms_norm dtype");
  if (d->weight != nullptr && d->weight_dtype != CTMR_DTYPE_F32 && d->weight_dtype != d->dtype)
    return api_fail(CTMR_ERR_INVALID, "weight must be fp32 or of x's type");
  if (d->tokens < 0 || d->heads <= 0 || d->channels <= 0) return api_fail(CTMR_ERR_INVALID, "rms_norm extents");
  if (d->channels > ctmr::kMaxNormChannels)
    return api_fail(CTMR_ERR_UNSUPPORTED, "more than %d channels", ctmr::kMaxNormChannels);
  if (static_cast<long long>(d->tokens) * d->heads > 0x7fffffffLL)
    return api_fail(CTMR_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if (!(d->eps > 0.f) || !std::isfinite(d->eps)) return api_fail(CTMR_ERR_INVALID, "eps must be positive");
  if (d->scale != nullptr && d->heads != 1) return api_fail(CTMR_ERR_UNSUPPORTED, "8-bit rows have no heads");
  const long long strides[10] = {d->x_token_stride, d->x_head_stride, d->residual_token_stride, d->residual_head_stride,
                                 d->y_token_stride, d->y_head_stride, d->sum_token_stride, d->sum_head_stride,
                                 d->scale_token_stride, d->scale_group_stride};
  for (const long long s : strides)
    if (!stride_ok(s)) return api_fail(CTMR_ERR_INVALID, "strides must not be negative");
  if (d->tokens == 0) return CTMR_OK;
  if (d->x == nullptr || d->y == nullptr) return api_fail(CTMR_ERR_INVALID, "null x or y");
  if (!aligned_to(d->x, d->dtype) || !aligned_to(d->residual, d->dtype) || !aligned_to(d->sum, d->dtype) ||
      !aligned_to(d->weight, d->weight_dtype) || (d->scale == nullptr && !aligned_to(d->y, d->dtype)) ||
      !aligned_to(d->scale, CTMR_DTYPE_F32))
    return api_fail(CTMR_ERR_INVALID, "tensors must be aligned to their elements");
  if (!rows_apart(d->tokens, d->y_token_stride, d->heads, d->y_head_stride, d->channels) ||
      (d->sum != nullptr && !rows_apart(d->tokens, d->sum_token_stride, d->heads, d->sum_head_stride, d->channels)) ||
      (d->scale != nullptr &&
       !rows_apart(d->tokens, d->scale_token_stride, scale_groups(d->channels), d->scale_group_stride, 1)))
    return api_fail(CTMR_ERR_INVALID, "rows of y, of sum or of scale overlap one another");
  if (d->sum == d->y) return api_fail(CTMR_ERR_INVALID, "y and sum must be two tensors");
  ctmr::RowNormParams p{};
  p.x = d->x, p.residual = d->residual, p.weight = d->weight, p.y = d->y, p.sum = d->sum, p.scale = d->scale;
  p.x_token = strides[0], p.x_head = strides[1], p.r_token = strides[2], p.r_head = strides[3];
  p.y_token = strides[4], p.y_head = strides[5], p.s_token = strides[6], p.s_head = strides[7];
  p.scale_token = strides[8], p.scale_group = strides[9];
  p.tokens = d->tokens, p.heads = d->heads, p.channels = d->channels;
  p.weight_f32 = d->weight_dtype == CTMR_DTYPE_F32, p.eps = d->eps;
  return finish(ctmr::launch_row_norm(p, d->dtype, static_cast<cudaStream_t>(stream)), "rms_norm launch");
}

int ctmr_quantize_rows(const ctmr_quantize_rows_desc* d, void* stream) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (!float_type(d->dtype)) return api_fail(CTMR_ERR_INVALID, "quantize_rows dtype");
  if (d->rows < 0 || d->channels <= 0) return api_fail(CTMR_ERR_INVALID, "quantize_rows extents");
  if (d->channels > 0x3fffffff) return api_fail(CTMR_ERR_UNSUPPORTED, "more than 2^30 - 1 channels");
  if (!stride_ok(d->x_stride) || !stride_ok(d->values_stride) || !stride_ok(d->scale_row_stride) ||
      !stride_ok(d->scale_group_stride))
    return api_fail(CTMR_ERR_INVALID, "strides must not be negative");
  if (d->rows == 0) return CTMR_OK;
  if (d->x == nullptr || d->values == nullptr || d->scale == nullptr)
    return api_fail(CTMR_ERR_INVALID, "null x, values or scale");
  if (!aligned_to(d->x, d->dtype) || !aligned_to(d->scale, CTMR_DTYPE_F32))
    return api_fail(CTMR_ERR_INVALID, "tensors must be aligned to their elements");
  if (!rows_apart(d->rows, d->values_stride, 1, 0, d->channels) ||
      !rows_apart(d->rows, d->scale_row_stride, scale_groups(d->channels), d->scale_group_stride, 1))
    return api_fail(CTMR_ERR_INVALID, "rows of values or of scale overlap one another");
  ctmr::QuantizeParams p{};
  p.x = d->x, p.values = d->values, p.scale = d->scale;
  p.x_stride = d->x_stride, p.values_stride = d->values_stride;
  p.scale_row = d->scale_row_stride, p.scale_group = d->scale_group_stride;
  p.rows = d->rows, p.channels = d->channels, p.gate = d->gate != 0;
  return finish(ctmr::launch_quantize(p, d->dtype, static_cast<cudaStream_t>(stream)), "quantize_rows launch");
}

int ctmr_scaled_linear(const ctmr_scaled_linear_desc* d, void* stream) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (!float_type(d->y_dtype)) return api_fail(CTMR_ERR_INVALID, "scaled_linear output type");
  if (d->bias != nullptr && d->bias_dtype != CTMR_DTYPE_F32 && d->bias_dtype != d->y_dtype)
    return api_fail(CTMR_ERR_INVALID, "bias must be fp32 or of the output's type");
  if (d->rows < 0 || d->in_features <= 0 || d->out_features <= 0)
    return api_fail(CTMR_ERR_INVALID, "scaled_linear extents");
  if (d->rows > 0x3fffffff || d->in_features > 0x3fffffff || d->out_features > 0x3fffffff)
    return api_fail(CTMR_ERR_UNSUPPORTED, "scaled_linear extents above 2^30 - 1");
  if (d->x_stride < d->in_features || d->weight_stride < d->in_features || d->x_stride % 16 != 0 ||
      d->weight_stride % 16 != 0 || d->x_stride >= (1LL << 38) || d->weight_stride >= (1LL << 38))
    return api_fail(CTMR_ERR_INVALID, "rows of x and weight cover a row and lie a multiple of 16 bytes apart");
  if (d->y_stride < d->out_features || !stride_ok(d->y_stride) || !stride_ok(d->x_scale_row_stride) ||
      !stride_ok(d->x_scale_block_stride) || !stride_ok(d->weight_scale_row_stride) ||
      !stride_ok(d->weight_scale_block_stride))
    return api_fail(CTMR_ERR_INVALID, "strides must not be negative, and rows of y must cover a row");
  if (d->rows == 0) return CTMR_OK;
  if (d->x == nullptr || d->weight == nullptr || d->x_scale == nullptr || d->weight_scale == nullptr || d->y == nullptr)
    return api_fail(CTMR_ERR_INVALID, "null x, weight, scale or y");
  if (reinterpret_cast<uintptr_t>(d->x) % 16 != 0 || reinterpret_cast<uintptr_t>(d->weight) % 16 != 0)
    return api_fail(CTMR_ERR_INVALID, "x and weight must be 16-byte aligned");
  if (!aligned_to(d->x_scale, CTMR_DTYPE_F32) || !aligned_to(d->weight_scale, CTMR_DTYPE_F32) ||
      !aligned_to(d->y, d->y_dtype) || !aligned_to(d->bias, d->bias_dtype))
    return api_fail(CTMR_ERR_INVALID, "tensors must be aligned to their elements");
  ctmr::ScaledLinearParams p{};
  p.x = d->x, p.weight = d->weight, p.bias = d->bias, p.x_scale = d->x_scale, p.w_scale = d->weight_scale, p.y = d->y;
  p.x_stride = d->x_stride, p.weight_stride = d->weight_stride, p.y_stride = d->y_stride;
  p.xs_row = d->x_scale_row_stride, p.xs_block = d->x_scale_block_stride;
  p.ws_row = d->weight_scale_row_stride, p.ws_block = d->weight_scale_block_stride;
  p.rows = d->rows, p.in = d->in_features, p.out = d->out_features;
  p.bias_f32 = d->bias_dtype == CTMR_DTYPE_F32;
  return ctmr::launch_scaled_linear(p, d->y_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
