// Root-mean-square norm of rows, with the residual's addition before it and an output in 8 bits where wanted:
//   h = x + r,  s = h / sqrt(mean(h^2) + eps) * w,
// h rounded to x's type beside it, where it is kept (the residual stream of a block).
//
// One pass over memory: a row's values stay in registers between the sum and the scaling, 8 channels (16 bytes of a
// 16-bit row) to an access. A warp takes a row of up to 1,024 channels, a block one of more. What bounds it is
// memory: 7 bytes a channel for 16-bit rows with a residual and an 8-bit output. The squares are added in 64
// bits: at the rate that memory allows, 3 channels a clock and SM, the conversions take a fifth of their unit's time,
// and the 8-bit rounding gets a mean that its 64-bit recomputation can rely on. The norm is taken of the
// unrounded sum h, so that it does not see the stream's rounding.
#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"
#include "launch.cuh"

namespace ctmr {
namespace {

// BLOCK: a block to a row; otherwise a warp. V: eights of channels to a thread.
template <typename T, int V, bool BLOCK, bool EIGHT, bool WIDE>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) row_norm_kernel(const __grid_constant__ RowNormParams p) {
  __shared__ double part[BLOCK ? 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int span = BLOCK ? blockDim.x : 32, mine = BLOCK ? threadIdx.x : lane;
  const long long row = BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (!BLOCK && row >= static_cast<long long>(p.tokens) * p.heads) return;  // whole warps
  const int token = p.heads == 1 ? static_cast<int>(row) : static_cast<int>(row / p.heads);
  const int head = p.heads == 1 ? 0 : static_cast<int>(row - static_cast<long long>(token) * p.heads);
  const T* x = static_cast<const T*>(p.x) + token * p.x_token + head * p.x_head;
  const T* r = static_cast<const T*>(p.residual) + (p.residual ? token * p.r_token + head * p.r_head : 0);

  float h[V][8];
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (mine + i * span) * 8;
    load8<T, WIDE>(x + c, p.channels - c, h[i]);
  }
  if (p.residual != nullptr) {
    float add[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (mine + i * span) * 8;
      load8<T, WIDE>(r + c, p.channels - c, add[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] += add[i][e];
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) total = fma(static_cast<double>(h[i][e]), static_cast<double>(h[i][e]), total);
#pragma unroll
  for (int i = 16; i > 0; i /= 2) total += __shfl_xor_sync(0xffffffffu, total, i);
  if constexpr (BLOCK) {
    if (lane == 0) part[warp] = total;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    total = lane < warps ? part[lane] : 0.0;
#pragma unroll
    for (int i = 16; i > 0; i /= 2) total += __shfl_xor_sync(0xffffffffu, total, i);
  }
  const double by64 = 1.0 / sqrt(total / p.channels + static_cast<double>(p.eps));
  const float by = static_cast<float>(by64);

#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (mine + i * span) * 8, left = p.channels - c;
    float w[8], s[8];
    if (p.weight == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
    } else if (p.weight_f32) {
      load8<float, WIDE>(static_cast<const float*>(p.weight) + c, left, w);
    } else {
      load8<T, WIDE>(static_cast<const T*>(p.weight) + c, left, w);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = left > 0 ? h[i][e] * by * w[e] : 0.f;
    if constexpr (EIGHT) {
      if (!WIDE)  // what lies past the row's end in a half-filled eight
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = e < left ? s[e] : 0.f;
      float scale;
      // Read again: the sum in 32 bits may have been rounded.
      auto exact = [&](int e) {
        if (e >= left) return 0.0;
        double v = static_cast<double>(to_float(x[c + e]));
        if (p.residual != nullptr) v += static_cast<double>(to_float(r[c + e]));
        if (p.weight != nullptr)
          v *= static_cast<double>(p.weight_f32 ? static_cast<const float*>(p.weight)[c + e]
                                                : to_float(static_cast<const T*>(p.weight)[c + e]));
        return v * by64;
      };
      const uint2 q = quantize_group<true>(s, exact, scale);
      store_bytes<WIDE>(static_cast<uint8_t*>(p.y) + token * p.y_token + c, left, q);
      if ((lane & 15) == 0 && left > 0) p.scale[token * p.scale_token + (c / kScaleGroup) * p.scale_group] = scale;
    } else {
      store8<T, WIDE>(static_cast<T*>(p.y) + token * p.y_token + head * p.y_head + c, left, s);
    }
    // Last, as it may lie where x or r did.
    if (p.sum != nullptr) store8<T, WIDE>(static_cast<T*>(p.sum) + token * p.s_token + head * p.s_head + c, left, h[i]);
  }
}

template <typename T, int V, bool BLOCK, bool EIGHT>
cudaError_t launch(const RowNormParams& p, bool wide, unsigned grid, int threads, cudaStream_t stream) {
  return wide ? launch_kernel(row_norm_kernel<T, V, BLOCK, EIGHT, true>, dim3(grid), dim3(threads), 0, stream, p)
              : launch_kernel(row_norm_kernel<T, V, BLOCK, EIGHT, false>, dim3(grid), dim3(threads), 0, stream, p);
}

template <typename T, bool EIGHT>
cudaError_t launch_rows(const RowNormParams& p, cudaStream_t stream) {
  // 16-byte accesses where every row allows them.
  constexpr int kEach = 16 / sizeof(T);
  auto row_ok = [](const void* at, long long token, long long head, int each) {
    return at == nullptr || (reinterpret_cast<uintptr_t>(at) % 16 == 0 && token % each == 0 && head % each == 0);
  };
  const bool wide = p.channels % 8 == 0 && row_ok(p.x, p.x_token, p.x_head, kEach) &&
                    row_ok(p.residual, p.r_token, p.r_head, kEach) && row_ok(p.sum, p.s_token, p.s_head, kEach) &&
                    (EIGHT ? reinterpret_cast<uintptr_t>(p.y) % 8 == 0 && p.y_token % 8 == 0
                           : row_ok(p.y, p.y_token, p.y_head, kEach)) &&
                    (p.weight == nullptr || reinterpret_cast<uintptr_t>(p.weight) % 16 == 0);
  const long long rows = static_cast<long long>(p.tokens) * p.heads;
  const int eights = (p.channels + 7) / 8;
  if (eights <= 128) {
    const int warps = 8;
    const unsigned grid = static_cast<unsigned>((rows + warps - 1) / warps);
    if (eights <= 32) return launch<T, 1, false, EIGHT>(p, wide, grid, warps * 32, stream);
    if (eights <= 64) return launch<T, 2, false, EIGHT>(p, wide, grid, warps * 32, stream);
    return launch<T, 4, false, EIGHT>(p, wide, grid, warps * 32, stream);
  }
  auto threads = [&](int v) { return ((eights + v - 1) / v + 31) / 32 * 32; };
  const unsigned grid = static_cast<unsigned>(rows);
  if (threads(1) <= 512) return launch<T, 1, true, EIGHT>(p, wide, grid, threads(1), stream);
  if (threads(2) <= 1024) return launch<T, 2, true, EIGHT>(p, wide, grid, threads(2), stream);
  return launch<T, 4, true, EIGHT>(p, wide, grid, threads(4), stream);
}

}  // namespace

cudaError_t launch_row_norm(const RowNormParams& p, int dtype, cudaStream_t stream) {
  const bool eight = p.scale != nullptr;
  switch (dtype) {
    case CTMR_DTYPE_F32: return eight ? launch_rows<float, true>(p, stream) : launch_rows<float, false>(p, stream);
    case CTMR_DTYPE_BF16:
      return eight ? launch_rows<__nv_bfloat16, true>(p, stream) : launch_rows<__nv_bfloat16, false>(p, stream);
    default: return eight ? launch_rows<__half, true>(p, stream) : launch_rows<__half, false>(p, stream);
  }
}

}  // namespace ctmr
