// Attention over packed documents: softmax over the keys of a query's own document, with causal and
// prefix masks, capped scores and a bias that falls with distance, grouped heads.
//   s_ij = cap(scale q_i . k_j) - slope_h |p_i - j|,  p_i = i + Lk - Lq,  cap(x) = c tanh(x / c)
// First form: one warp per query and head, the online softmax over its keys one by one.
#include "launch.cuh"
#include "tokens.cuh"

namespace ctmr {
namespace {

template <typename T>
__global__ void attention_warp_kernel(const AttentionParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, h = blockIdx.y, hk = h / (p.heads / p.kv_heads);
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
  int doc, i, q_len, k_len;
  long long qo, ko, vo, oo, at;
  if (p.q_offsets != nullptr) {
    if (row >= p.q_tokens) return;
    doc = segment_of_row(p.q_offsets, p.documents, row);
    if (doc < 0) {
      flag_error(kErrBadOffsets);
      return;
    }
    int qb, qe, kb, ke;
    segment_range(p.q_offsets, doc, p.q_tokens, qb, qe);
    segment_range(p.k_offsets, doc, p.k_tokens, kb, ke);
    i = row - qb, q_len = qe - qb, k_len = ke - kb;
    qo = row * p.q_token, oo = row * p.o_token, ko = kb * p.k_token, vo = kb * p.v_token, at = row;
  } else {
    if (row >= p.q_tokens * p.documents) return;
    doc = row / p.q_tokens, i = row - doc * p.q_tokens, q_len = p.q_tokens, k_len = p.k_tokens;
    if (p.k_lengths != nullptr) {
      const int n = p.k_lengths[doc];
      if (n < 0 || n > k_len) flag_error(kErrBadOffsets);
      k_len = min(max(n, 0), k_len);
    }
    qo = doc * p.q_doc + i * p.q_token, oo = doc * p.o_doc + i * p.o_token;
    ko = doc * p.k_doc, vo = doc * p.v_doc, at = row;
  }
  if (q_len > p.max_q) flag_error(kErrBadOffsets);
  const int place = i + k_len - q_len;
  const int prefix = p.prefix != nullptr ? p.prefix[doc] : 0;
  const int seen = p.causal ? min(k_len, max(place + 1, prefix)) : k_len;
  const float slope = p.slopes != nullptr ? p.slopes[h] : 0.f;
  const T* q = static_cast<const T*>(p.q) + qo + h * p.q_head;
  const T* k = static_cast<const T*>(p.k) + ko + hk * p.k_head;
  const T* v = static_cast<const T*>(p.v) + vo + hk * p.v_head;
  float qv[4], acc[4] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) qv[c] = lane + 32 * c < p.dim ? to_float(q[lane + 32 * c]) : 0.f;
  for (int j = 0; j < seen; ++j) {
    float s = 0.f, vv[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool in = lane + 32 * c < p.dim;
      s = fmaf(qv[c], in ? to_float(k[j * p.k_token + lane + 32 * c]) : 0.f, s);
      vv[c] = in ? to_float(v[j * p.v_token + lane + 32 * c]) : 0.f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.scale;
    if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
    s -= slope * fabsf(static_cast<float>(place - j));
    const float m_new = fmaxf(m, s), f = __expf(m - m_new), e = __expf(s - m_new);
    l = l * f + e;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = acc[c] * f + e * vv[c];
    m = m_new;
  }
  T* out = static_cast<T*>(p.out) + oo + h * p.o_head;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < p.dim) out[lane + 32 * c] = from_float<T>(l > 0.f ? acc[c] / l : 0.f);
  if (p.lse != nullptr && lane == 0) p.lse[at * p.heads + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

size_t attention_packed_workspace(const AttentionParams&) { return 0; }

cudaError_t launch_attention_packed(const AttentionParams& p, bool bf16, cudaStream_t stream) {
  const int rows = p.q_offsets != nullptr ? p.q_tokens : p.q_tokens * p.documents;
  auto kern = bf16 ? attention_warp_kernel<__nv_bfloat16> : attention_warp_kernel<__half>;
  return launch_kernel(kern, dim3((rows + 3) / 4, p.heads), dim3(128), 0, stream, p);
}

}  // namespace ctmr
