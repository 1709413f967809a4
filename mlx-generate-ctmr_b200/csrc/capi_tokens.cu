// The extern "C" entry points of the packed-token operators: argument checks and dispatch.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "tokens.cuh"

namespace {

using ctmr::api_fail;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? CTMR_OK : api_fail(CTMR_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (need == 0) return CTMR_OK;
  if (workspace == nullptr || bytes < need)
    return api_fail(CTMR_ERR_WORKSPACE, "workspace holds %zu bytes, needs %zu", workspace ? bytes : size_t(0), need);
  return aligned16(workspace) ? CTMR_OK : api_fail(CTMR_ERR_INVALID, "workspace must be 16-byte aligned");
}

int linear_params(const ctmr_adapter_linear_desc* d, ctmr::LinearParams& p) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (d->dtype != CTMR_DTYPE_BF16 && d->dtype != CTMR_DTYPE_F16)
    return api_fail(CTMR_ERR_INVALID, "adapter_linear takes bf16 or fp16");
  if (d->rows < 0 || d->in_features <= 0 || d->out_features <= 0)
    return api_fail(CTMR_ERR_INVALID, "adapter_linear extents");
  if (d->rows > 0x3fffffff || d->in_features > 0x3fffffff || d->out_features > 0x3fffffff)
    return api_fail(CTMR_ERR_UNSUPPORTED, "adapter_linear extents above 2^30 - 1");
  if (d->in_features % 8 != 0) return api_fail(CTMR_ERR_UNSUPPORTED, "in_features must be a multiple of 8");
  if (d->weight == nullptr || (d->rows > 0 && (d->x == nullptr || d->y == nullptr)))
    return api_fail(CTMR_ERR_INVALID, "null x, weight or y");
  if (!aligned16(d->x) || !aligned16(d->weight))
    return api_fail(CTMR_ERR_INVALID, "x and weight must be 16-byte aligned");
  if (d->x_stride < d->in_features || d->weight_stride < d->in_features || d->x_stride % 8 != 0 ||
      d->weight_stride % 8 != 0 || d->y_stride < d->out_features || d->x_stride >= (1LL << 38) ||
      d->weight_stride >= (1LL << 38))
    return api_fail(CTMR_ERR_INVALID, "row strides cover a row; those of x and weight are multiples of 8");
  if (d->bias != nullptr && d->bias_dtype != CTMR_DTYPE_F32 && d->bias_dtype != d->dtype)
    return api_fail(CTMR_ERR_INVALID, "bias must be fp32 or of the operands' type");
  if (d->segments < 0 || d->segments > 0x3fffffff) return api_fail(CTMR_ERR_INVALID, "segment count");
  if (d->segments > 0) {
    if (d->down == nullptr || d->up == nullptr || d->scale == nullptr || d->offsets == nullptr || d->index == nullptr)
      return api_fail(CTMR_ERR_INVALID, "null adapter pointer");
    if (d->adapters <= 0) return api_fail(CTMR_ERR_INVALID, "no adapters");
    if (d->rank <= 0 || d->rank % 8 != 0 || d->rank > 128)
      return api_fail(CTMR_ERR_UNSUPPORTED, "rank must be a multiple of 8 up to 128, got %d", d->rank);
    if (!aligned16(d->down) || !aligned16(d->up))
      return api_fail(CTMR_ERR_INVALID, "down and up must be 16-byte aligned");
  }
  p = ctmr::LinearParams{};
  p.x = d->x, p.weight = d->weight, p.bias = d->bias, p.y = d->y;
  p.bias_f32 = d->bias_dtype == CTMR_DTYPE_F32;
  p.x_stride = d->x_stride, p.weight_stride = d->weight_stride, p.y_stride = d->y_stride;
  p.rows = d->rows, p.in = d->in_features, p.out = d->out_features;
  if (d->segments > 0) {
    p.down = d->down, p.up = d->up, p.scale = d->scale, p.offsets = d->offsets, p.index = d->index;
    p.adapters = d->adapters, p.rank = d->rank, p.segments = d->segments;
  }
  return CTMR_OK;
}

int attention_params(const ctmr_attention_desc* d, ctmr::AttentionParams& p) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (d->dtype != CTMR_DTYPE_BF16 && d->dtype != CTMR_DTYPE_F16)
    return api_fail(CTMR_ERR_INVALID, "attention takes bf16 or fp16");
  if (d->documents <= 0 || d->q_tokens < 0 || d->k_tokens < 0 || d->heads <= 0 || d->kv_heads <= 0)
    return api_fail(CTMR_ERR_INVALID, "attention extents");
  if (d->heads % d->kv_heads != 0) return api_fail(CTMR_ERR_INVALID, "heads must be a multiple of kv_heads");
  if (d->heads > 65535 || d->documents > 0x3fffffff)
    return api_fail(CTMR_ERR_UNSUPPORTED, "more than 65535 heads or 2^30 - 1 documents");
  if (d->head_dim <= 0 || d->head_dim % 8 != 0 || d->head_dim > 128)
    return api_fail(CTMR_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, got %d", d->head_dim);
  const bool packed = d->q_offsets != nullptr;
  if (packed != (d->k_offsets != nullptr))
    return api_fail(CTMR_ERR_INVALID, "q_offsets and k_offsets come together");
  if (packed && d->k_lengths != nullptr) return api_fail(CTMR_ERR_INVALID, "k_lengths belong to the batched form");
  if (d->prefix != nullptr && !d->causal) return api_fail(CTMR_ERR_INVALID, "a prefix needs a causal mask");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return api_fail(CTMR_ERR_INVALID, "scale must be positive");
  if (!(d->cap >= 0.f) || !std::isfinite(d->cap)) return api_fail(CTMR_ERR_INVALID, "cap must not be negative");
  if (d->max_q < 0) return api_fail(CTMR_ERR_INVALID, "negative max_q");
  if (d->q_tokens > 0x3fffffff || d->k_tokens > 0x3fffffff ||
      (!packed && static_cast<long long>(d->documents) * d->q_tokens > 0x3fffffffLL))
    return api_fail(CTMR_ERR_UNSUPPORTED, "more than 2^30 - 1 rows");
  if (d->q_tokens > 0 && (d->q == nullptr || d->out == nullptr)) return api_fail(CTMR_ERR_INVALID, "null q or out");
  if (d->q_tokens > 0 && d->k_tokens > 0 && (d->k == nullptr || d->v == nullptr))
    return api_fail(CTMR_ERR_INVALID, "null k or v");
  if (!aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out))
    return api_fail(CTMR_ERR_INVALID, "q, k, v and out must be 16-byte aligned");
  const long long strides[12] = {d->q_doc_stride, d->q_token_stride, d->q_head_stride, d->k_doc_stride,
                                 d->k_token_stride, d->k_head_stride, d->v_doc_stride, d->v_token_stride,
                                 d->v_head_stride, d->out_doc_stride, d->out_token_stride, d->out_head_stride};
  for (const long long s : strides)
    if (s < 0 || s % 8 != 0 || s >= (1LL << 38))
      return api_fail(CTMR_ERR_INVALID, "strides must be multiples of 8 and not negative");
  p = ctmr::AttentionParams{};
  p.q = d->q, p.k = d->k, p.v = d->v, p.out = d->out, p.lse = d->lse;
  p.q_offsets = d->q_offsets, p.k_offsets = d->k_offsets, p.k_lengths = d->k_lengths, p.prefix = d->prefix;
  p.slopes = d->slopes;
  p.q_doc = strides[0], p.q_token = strides[1], p.q_head = strides[2];
  p.k_doc = strides[3], p.k_token = strides[4], p.k_head = strides[5];
  p.v_doc = strides[6], p.v_token = strides[7], p.v_head = strides[8];
  p.o_doc = strides[9], p.o_token = strides[10], p.o_head = strides[11];
  p.documents = d->documents, p.q_tokens = d->q_tokens, p.k_tokens = d->k_tokens;
  p.heads = d->heads, p.kv_heads = d->kv_heads, p.dim = d->head_dim;
  p.causal = d->causal != 0, p.scale = d->scale, p.cap = d->cap;
  // The largest query count that any document can have.
  p.max_q = packed && d->max_q > 0 && d->max_q < d->q_tokens ? d->max_q : d->q_tokens;
  return CTMR_OK;
}

}  // namespace

extern "C" {

int ctmr_rotary_axes(const ctmr_rotary_desc* d, void* stream) {
  if (d == nullptr) return api_fail(CTMR_ERR_INVALID, "null descriptor");
  if (d->dtype != CTMR_DTYPE_F32 && d->dtype != CTMR_DTYPE_BF16 && d->dtype != CTMR_DTYPE_F16)
    return api_fail(CTMR_ERR_INVALID, "rotary dtype");
  if (d->tokens < 0 || d->heads <= 0 || d->head_dim <= 0) return api_fail(CTMR_ERR_INVALID, "rotary extents");
  if (d->tokens > 0x7fffffffLL || d->head_dim > 4096 || d->heads > 8192)
    return api_fail(CTMR_ERR_UNSUPPORTED, "rotary extents too large");
  if (d->axes < 1 || d->axes > CTMR_MAX_ROTARY_AXES)
    return api_fail(CTMR_ERR_INVALID, "between 1 and %d rotary axes", CTMR_MAX_ROTARY_AXES);
  ctmr::RotaryParams p{};
  for (int a = 0; a < d->axes; ++a) {
    if (d->section[a] < 0 || d->section[a] > d->head_dim) return api_fail(CTMR_ERR_INVALID, "rotary section %d", a);
    p.pairs += d->section[a];
    p.section_end[a] = p.pairs;
  }
  if (p.pairs < 1 || 2 * p.pairs > d->head_dim)
    return api_fail(CTMR_ERR_INVALID, "the sections hold %d pairs, a head of %d at least 1 and at most %d", p.pairs,
                    d->head_dim, d->head_dim / 2);
  if (d->x_token_stride < 0 || d->x_head_stride < 0 || d->y_token_stride < 0 || d->y_head_stride < 0 ||
      d->positions_stride < 0)
    return api_fail(CTMR_ERR_INVALID, "negative stride");
  if (d->tokens == 0) return CTMR_OK;
  if (d->x == nullptr || d->y == nullptr || d->positions == nullptr || d->inv_freq == nullptr)
    return api_fail(CTMR_ERR_INVALID, "null rotary pointer");
  const uintptr_t size = d->dtype == CTMR_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d->x) % size != 0 || reinterpret_cast<uintptr_t>(d->y) % size != 0)
    return api_fail(CTMR_ERR_INVALID, "x and y must be aligned to their elements");
  p.x = d->x, p.y = d->y, p.tokens = d->tokens, p.heads = d->heads, p.dim = d->head_dim;
  p.x_token = d->x_token_stride, p.x_head = d->x_head_stride;
  p.y_token = d->y_token_stride, p.y_head = d->y_head_stride;
  p.positions = d->positions, p.positions_f32 = d->positions_f32, p.pos_stride = d->positions_stride;
  p.inv_freq = d->inv_freq, p.axes = d->axes, p.interleaved = d->interleaved, p.inverse = d->inverse;
  return finish(ctmr::launch_rotary(p, d->dtype, static_cast<cudaStream_t>(stream)), "rotary launch");
}

size_t ctmr_adapter_linear_workspace_size(const ctmr_adapter_linear_desc* d) {
  ctmr::LinearParams p;
  return linear_params(d, p) == CTMR_OK && p.rows > 0 ? ctmr::adapter_linear_workspace(p) : 0;
}

int ctmr_adapter_linear(const ctmr_adapter_linear_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  ctmr::LinearParams p;
  int st = linear_params(d, p);
  if (st != CTMR_OK || p.rows == 0) return st;
  st = check_workspace(ctmr::adapter_linear_workspace(p), workspace, workspace_bytes);
  if (st != CTMR_OK) return st;
  p.inner = workspace;
  return ctmr::launch_adapter_linear(p, d->dtype == CTMR_DTYPE_BF16, static_cast<cudaStream_t>(stream));
}

int ctmr_attention(const ctmr_attention_desc* d, void* stream) {
  ctmr::AttentionParams p;
  const int st = attention_params(d, p);
  if (st != CTMR_OK || p.q_tokens == 0) return st;
  return ctmr::launch_attention_packed(p, d->dtype == CTMR_DTYPE_BF16, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
