// A projection shared by all rows, beside it a low-rank adapter for each segment of rows:
//   y_i = W x_i + b + scale_a up_a (down_a x_i),  a = index[segment of i], no adapter where a < 0.
// First form: a plain tiled product on the FMA pipe; the adapters' inner products are computed by a
// kernel before it.
#include "launch.cuh"
#include "tokens.cuh"

namespace ctmr {
namespace {

constexpr int kTile = 64, kStep = 16;

__device__ __forceinline__ int adapter_of_row(const LinearParams& p, int row) {
  const int s = p.segments > 0 ? segment_of_row(p.offsets, p.segments, row) : -1;
  if (s < 0) return -1;
  int begin, end;
  segment_range(p.offsets, s, p.rows, begin, end);
  const int a = p.index[s];
  if (a >= p.adapters) flag_error(kErrBadOffsets);
  return a >= p.adapters ? -1 : a;
}

// inner[i][r] = scale_a * sum_c down_a[r][c] x[i][c]: one warp per row.
template <typename T>
__global__ void adapter_inner_kernel(const LinearParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= p.rows) return;
  const int a = adapter_of_row(p, row);
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  for (int r = 0; r < p.rank && a >= 0; ++r) {
    const T* d = static_cast<const T*>(p.down) + (static_cast<long long>(a) * p.rank + r) * p.in;
    float sum = 0.f;
    for (int c = lane; c < p.in; c += 32) sum = fmaf(to_float(d[c]), to_float(x[c]), sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) static_cast<float*>(p.inner)[static_cast<long long>(row) * p.rank + r] = sum * p.scale[a];
  }
}

template <typename T>
__global__ void __launch_bounds__(256) linear_kernel(const LinearParams p) {
  __shared__ float xs[kStep][kTile + 1], ws[kStep][kTile + 1];
  griddep_wait();
  griddep_launch_dependents();
  const int r0 = blockIdx.y * kTile, o0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int c0 = 0; c0 < p.in; c0 += kStep) {
    for (int i = threadIdx.x; i < kStep * kTile; i += 256) {
      const int c = i & 15, j = i >> 4;
      const bool in = c0 + c < p.in;
      xs[c][j] = in && r0 + j < p.rows
                     ? to_float(static_cast<const T*>(p.x)[(r0 + j) * p.x_stride + c0 + c]) : 0.f;
      ws[c][j] = in && o0 + j < p.out
                     ? to_float(static_cast<const T*>(p.weight)[(o0 + j) * p.weight_stride + c0 + c]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kStep; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[c][ty + 16 * i], ws[c][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + ty + 16 * i;
    if (row >= p.rows) continue;
    const int a = adapter_of_row(p, row);
    for (int j = 0; j < 4; ++j) {
      const int o = o0 + tx + 16 * j;
      if (o >= p.out) continue;
      float v = acc[i][j];
      if (p.bias != nullptr)
        v += p.bias_f32 ? static_cast<const float*>(p.bias)[o] : to_float(static_cast<const T*>(p.bias)[o]);
      if (a >= 0) {
        const T* u = static_cast<const T*>(p.up) + (static_cast<long long>(a) * p.out + o) * p.rank;
        const float* t = static_cast<const float*>(p.inner) + static_cast<long long>(row) * p.rank;
        for (int r = 0; r < p.rank; ++r) v = fmaf(t[r], to_float(u[r]), v);
      }
      static_cast<T*>(p.y)[row * p.y_stride + o] = from_float<T>(v);
    }
  }
}

template <typename T>
cudaError_t launch(const LinearParams& p, cudaStream_t stream) {
  if (p.segments > 0) {
    const cudaError_t e =
        launch_kernel(adapter_inner_kernel<T>, dim3((p.rows + 3) / 4), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(linear_kernel<T>, dim3((p.out + kTile - 1) / kTile, (p.rows + kTile - 1) / kTile), dim3(256), 0,
                       stream, p);
}

}  // namespace

size_t adapter_linear_workspace(const LinearParams& p) {
  return p.segments > 0 ? static_cast<size_t>(p.rows) * p.rank * sizeof(float) : 0;
}

cudaError_t launch_adapter_linear(const LinearParams& p, bool bf16, cudaStream_t stream) {
  return bf16 ? launch<__nv_bfloat16>(p, stream) : launch<__half>(p, stream);
}

}  // namespace ctmr
