// Rows to 8 bits, as they are or as a gated pair: v = x, or v = silu(a) b for the halves a and b of a row;
// then e4m3 values with a scale for every 128 channels.
//
// Bound by memory (5 bytes a channel of a gated 16-bit row, 3 of a plain one) as long as the arithmetic stays below
// some 25 instructions a channel: silu is one exponential and one reciprocal, with the exponent's product taken
// in two parts so that the error stays near 2^-22 for any size of a. Groups of 128 channels, 16 threads each, follow one
// another over the rows without regard to where a row ends, so that no size leaves threads idle.
#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"
#include "launch.cuh"

namespace ctmr {
namespace {

constexpr int kThreads = 256;

// silu(a) b. e^-a is infinite below -88, and the product then zero: below what any scale keeps.
__device__ __forceinline__ float gated(float a, float b) {
  constexpr float kLog2E = 1.44269504f, kRest = 1.92596299e-8f;
  const float n = fminf(fmaxf(-a, -128.f), 128.f);  // further out nothing changes, but the product would overflow
  const float t = n * kLog2E, rest = fmaf(n, kRest, fmaf(n, kLog2E, -t));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, rest * 0.693147181f, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return a * r * b;
}

__device__ __noinline__ double gated64(double a, double b) { return a / (1.0 + exp(-a)) * b; }

// U eights of channels to a thread.
template <typename T, int U, bool GATE, bool WIDE>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const __grid_constant__ QuantizeParams p) {
  const uint32_t per_row = (p.channels + kScaleGroup - 1) / kScaleGroup * (kScaleGroup / 8);
  // The block's first eight; 32-bit arithmetic from there on.
  const unsigned long long first = static_cast<unsigned long long>(blockIdx.x) * (kThreads * U);
  const unsigned long long row0 = first / per_row;
  const uint32_t col0 = static_cast<uint32_t>(first - row0 * per_row);
  griddep_wait();
  griddep_launch_dependents();
  float v[U][8], b[U][8];
  int row[U], c[U], left[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t at = col0 + i * kThreads + threadIdx.x, down = at / per_row;
    const unsigned long long r = row0 + down;
    const bool in = r < static_cast<unsigned long long>(p.rows);
    row[i] = in ? static_cast<int>(r) : 0;
    c[i] = static_cast<int>(at - down * per_row) * 8;
    left[i] = in ? p.channels - c[i] : 0;
    const T* x = static_cast<const T*>(p.x) + row[i] * p.x_stride + c[i];
    load8<T, WIDE>(x, left[i], v[i]);
    if constexpr (GATE) load8<T, WIDE>(x + p.channels, left[i], b[i]);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if constexpr (GATE)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = gated(v[i][e], b[i][e]);
    float scale;
    const T* x = static_cast<const T*>(p.x) + row[i] * p.x_stride + c[i];
    auto exact = [&](int e) { return e < left[i] ? gated64(to_float(x[e]), to_float(x[p.channels + e])) : 0.0; };
    const uint2 q = quantize_group<GATE>(v[i], exact, scale);
    store_bytes<WIDE>(static_cast<uint8_t*>(p.values) + row[i] * p.values_stride + c[i], left[i], q);
    if ((threadIdx.x & 15) == 0 && left[i] > 0)
      p.scale[row[i] * p.scale_row + (c[i] / kScaleGroup) * p.scale_group] = scale;
  }
}

template <typename T, bool GATE>
cudaError_t launch(const QuantizeParams& p, cudaStream_t stream) {
  const bool wide = p.channels % 8 == 0 && p.x_stride % (16 / static_cast<int>(sizeof(T))) == 0 &&
                    reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.values_stride % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(p.values) % 8 == 0;
  const unsigned long long per_row = (p.channels + kScaleGroup - 1) / kScaleGroup * (kScaleGroup / 8);
  const unsigned long long eights = per_row * p.rows;
  const bool small = eights <= 4ull * kThreads * device_sm_count();  // fewer than four blocks an SM: no second eight
  const int each = kThreads * (small ? 1 : 2);
  const unsigned long long grid = (eights + each - 1) / each;
  if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  auto go = [&](auto kern) { return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, p); };
  if (small) return wide ? go(quantize_kernel<T, 1, GATE, true>) : go(quantize_kernel<T, 1, GATE, false>);
  return wide ? go(quantize_kernel<T, 2, GATE, true>) : go(quantize_kernel<T, 2, GATE, false>);
}

template <typename T>
cudaError_t launch_any(const QuantizeParams& p, cudaStream_t stream) {
  return p.gate ? launch<T, true>(p, stream) : launch<T, false>(p, stream);
}

}  // namespace

cudaError_t launch_quantize(const QuantizeParams& p, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case CTMR_DTYPE_F32: return launch_any<float>(p, stream);
    case CTMR_DTYPE_BF16: return launch_any<__nv_bfloat16>(p, stream);
    default: return launch_any<__half>(p, stream);
  }
}

}  // namespace ctmr
