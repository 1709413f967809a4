// Operators on packed tokens (several requests in one call): rotary positions (rotary.cu), a shared
// projection with per-request low-rank adapters (adapter_linear.cu) and masked attention
// (attention_packed.cu). Their parameters, launchers, and what they share on the device.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"

namespace ctmr {

constexpr int kMaxRotaryAxes = 8;

struct RotaryParams {
  const void* x;
  void* y;                              // may be x
  long long tokens;
  int heads, dim, pairs;                // pairs: rotated (first, second) pairs per head
  long long x_token, x_head, y_token, y_head;  // element strides
  const void* positions;                // (tokens, axes) int32 or fp32, rows pos_stride elements apart
  int positions_f32;
  long long pos_stride;
  const float* inv_freq;                // (pairs)
  int axes, section_end[kMaxRotaryAxes];  // running sums of the pairs per axis
  int interleaved, inverse;
};

struct LinearParams {
  const void *x, *weight, *bias, *down, *up;
  const float* scale;
  const int *offsets, *index;
  void* y;
  void* inner;                          // workspace: the adapters' inner products, 16-bit
  long long x_stride, weight_stride, y_stride;
  int rows, in, out, rank, adapters, segments;
  int bias_f32;
};

struct AttentionParams {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int *q_offsets, *k_offsets, *k_lengths, *prefix;
  const float* slopes;
  long long q_doc, q_token, q_head, k_doc, k_token, k_head, v_doc, v_token, v_head, o_doc, o_token, o_head;
  int documents, q_tokens, k_tokens;    // tokens of the packed rows, or of each batch item without offsets
  int heads, kv_heads, dim;
  int causal, max_q;                    // max_q: no document has more queries
  float scale, cap;
};

cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream);
size_t adapter_linear_workspace(const LinearParams& p);
int launch_adapter_linear(const LinearParams& p, bool bf16, cudaStream_t stream);  // a CTMR_ status
int launch_attention_packed(const AttentionParams& p, bool bf16, cudaStream_t stream);  // a CTMR_ status

// The form for few query rows per key head, and whether it takes the call.
bool attention_few_takes(const AttentionParams& p);
cudaError_t launch_attention_few(const CUtensorMap& k, const CUtensorMap& v, const AttentionParams& p, bool bf16,
                                 cudaStream_t stream);
// A (channel, head, token, document) view of an attention operand in boxes of 64 channels x box_tokens
// tokens, 128-byte swizzled; a CTMR_ status.
int encode_tokens_map(CUtensorMap* map, const void* base, bool bf16, int dim, int heads, long long tokens,
                      long long docs, long long s_head, long long s_token, long long s_doc, int box_tokens,
                      const char* what);

// ---------------------------------------------------------------- ragged rows
// offsets[s] clamped into [0, total] (a negative or excessive offset never indexes memory) and, with
// it, the end of segment s clamped into [start, total]. A clamp that changed anything sets
// kErrBadOffsets: the call's answer is then not what the caller meant.
__device__ __forceinline__ void segment_range(const int* offsets, int s, int total, int& begin, int& end) {
  const int a = offsets[s], b = offsets[s + 1];
  begin = min(max(a, 0), total);
  end = min(max(b, begin), total);
  if (begin != a || end != b) flag_error(kErrBadOffsets);
}

// Reports every offset that segment_range would clamp, whether or not a block of the kernel comes to read it (a
// segment whose offsets make it empty may own no block). By one block.
__device__ __forceinline__ void report_offsets(const int* offsets, int segments, int total) {
  for (int s = threadIdx.x; s < segments; s += blockDim.x) {
    int begin, end;
    segment_range(offsets, s, total, begin, end);
  }
}

// The last s in [0, n) that `holds` for, by a whole warp: it holds up to some s and not after (it is not asked for 0,
// which is the answer where it holds for none). Log32(n) loads.
template <typename Holds>
__device__ __forceinline__ int last_segment(int n, int lane, Holds holds) {
  int lo = 0;  // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const bool ok = lane == 0 || (lane * step < n && holds(lo + lane * step));
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, ok));
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

// Tiles of `tile` rows that start afresh in each segment, without a table of them: segment s owns the
// numbers [f(s), f(s + 1)), f(s) = offsets[s] / tile + s, which are at least as many as its tiles
// (floor(b / t) - floor(a / t) + 1 >= ceil((b - a) / t)), so a grid of total / tile + segments + 1
// blocks covers every segment and few blocks find nothing to do. Block `id` belongs to the last s with
// f(s) <= id; f grows strictly, so a 32-way search by a warp finds it in log32(segments) loads.
// Returns the segment, all lanes of the warp together.
__device__ __forceinline__ int segment_of_tile(const int* offsets, int segments, int tile, int id, int lane) {
  return last_segment(segments, lane, [&](int s) { return max(offsets[s], 0) / tile + s <= id; });
}

// d += a b, 16 x 8 x 16, 16-bit operands, fp32 sums.
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- 16-bit values
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

}  // namespace ctmr
