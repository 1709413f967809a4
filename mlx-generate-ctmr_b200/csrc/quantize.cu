// Rows to 8 bits, as they are or as a gated pair: v = x, or v = silu(a) b for the halves a and b of a row;
// then e4m3 values with a scale for every 128 channels.
//
// Bound by memory (5 bytes a channel of a gated 16-bit row, 3 of a plain one) as long as the arithmetic stays below
// some 25 instructions a channel: silu is one exponential and one reciprocal, with the exponent's product taken
// in two parts so that the error stays near 2^-22 for any size of a. Groups of 128 channels, eight lanes each, follow one
// another over the rows without regard to where a row ends, so that no size leaves threads idle. 8,192 gated rows of
// 11,264: 88 us, 5.3 TB/s, where one output is written over and over (part of its 92 MB then stays in L2), 94 to 96 with
// outputs of their own; what is left are instructions, 24 a channel.
#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"
#include "launch.cuh"

namespace ctmr {
namespace {

constexpr int kThreads = 256, kBlocks = 3, kGroups = kThreads / kGroupLanes;

// Below this silu(a) nears the end of 32 bits' normal numbers, from where a large b can bring it back: groups that hold
// both at once are computed in 64 bits. (Up to 128, b leaves less than 2^-110, half the least step of the least scale.)
constexpr float kFarGate = -86.f, kFarOther = 128.f;

// silu(a) b, two at a time, for a from kFarGate on. The reciprocal meets b first: a may be subnormal, and then b large.
__device__ __forceinline__ float2 gated2(float2 a, float2 b) {
  constexpr float kLog2E = 1.44269504f, kRest = 1.92596299e-8f;
  // Further out nothing changes, but the product would overflow.
  const float2 n = make_float2(fmaxf(-a.x, -128.f), fmaxf(-a.y, -128.f));
  const float2 log2e = make_float2(kLog2E, kLog2E), minus = make_float2(-kLog2E, -kLog2E);
  const float2 t = mul2(n, log2e);
  // What t's rounding cut off, with the other sign, times ln 2: e^n = 2^t (1 - rest).
  const float2 rest = mul2(fma2(n, make_float2(-kRest, -kRest), fma2(n, minus, t)), make_float2(0.693147181f, 0.693147181f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  // 1 + e (1 - rest)
  const float2 one = make_float2(1.f, 1.f), less = fma2(rest, make_float2(-1.f, -1.f), one);
  const float2 d = fma2(e, less, one);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  return mul2(mul2(b, r), a);
}

// In units of 2^-24: the exponential's approximation 4 and its correction 1, the sum 1, the reciprocal 2, the three
// products 3.
constexpr int kGatedUnits = 12;

__device__ __forceinline__ double gated64(double a, double b) { return a / (1.0 + exp(-a)) * b; }

// What 64 bits decide, by single lanes: calls, so that the kernel's registers are not laid out for it.
template <typename T, bool WIDE>
__device__ __noinline__ double gated_top(const T* x, int channels, int group, int lane8) {
  double most = 0.0;
  for (int i = 0; i < kEach; ++i) {
    const int c = channel_of<WIDE>(group, lane8, i);
    if (c < channels) most = max_nan(most, fabs(gated64(to_float(x[c]), to_float(x[channels + c]))));
  }
  return most;
}

template <typename T, bool WIDE>
__device__ __noinline__ void gated_patch(const T* x, uint8_t* values, int channels, int group, int lane8, uint32_t differ,
                                         float by) {
  for (; differ != 0; differ &= differ - 1) {
    const int c = channel_of<WIDE>(group, lane8, __ffs(differ) - 1);
    if (c < channels) values[c] = static_cast<uint8_t>(e4m3_exact(gated64(to_float(x[c]), to_float(x[channels + c])) * by));
  }
}

// A block takes 32 groups of channels at a time, eight lanes each, then those p.skip_rows rows and p.skip_groups
// groups further: no division but the first.
template <typename T, bool GATE, bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocks) quantize_kernel(const __grid_constant__ QuantizeParams p) {
  const int lane8 = threadIdx.x % kGroupLanes;
  const uint32_t start = blockIdx.x * kGroups + threadIdx.x / kGroupLanes, rows = static_cast<uint32_t>(p.rows);
  uint32_t row = start / p.per_row, group = start - row * p.per_row;
  griddep_wait();
  griddep_launch_dependents();
  Loaded<T, WIDE> a, b;
  auto load = [&]() {
    const bool in = row < rows;
    const T* x = static_cast<const T*>(p.x) + (in ? row * p.x_stride : 0);
    a.load(x, in ? p.channels : 0, group, lane8);
    if constexpr (GATE) b.load(x + p.channels, in ? p.channels : 0, group, lane8);
  };
  load();
  while (__any_sync(0xffffffffu, row < rows)) {  // whole warps, for the shuffles
    const bool in = row < rows;
    const uint32_t row_now = in ? row : 0, group_now = group;
    const int channels = in ? p.channels : 0;
    const T* x = static_cast<const T*>(p.x) + row_now * p.x_stride;
    float v[kEach];
    bool far = false;
    a.values(v, channels, group, lane8);
    if constexpr (GATE) {
      float other[kEach], least = 0.f;
      b.values(other, channels, group, lane8);
#pragma unroll
      for (int e = 0; e < kEach; e += 2) least = min3(least, v[e], v[e + 1]);
      if (__any_sync(0xffffffffu, least < kFarGate)) {  // (ahead of the products, after which b would have to be kept)
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < kEach; e += 2) most = max_nan(most, other[e], other[e + 1]);
        far = least < kFarGate && !(most <= kFarOther);
      }
#pragma unroll
      for (int e = 0; e < kEach; e += 2) {
        const float2 g = gated2(make_float2(v[e], v[e + 1]), make_float2(other[e], other[e + 1]));
        v[e] = g.x, v[e + 1] = g.y;
      }
    }
    if (in) {  // (a row past the end stays where it is)
      row += p.skip_rows, group += p.skip_groups;
      if (group >= p.per_row) group -= p.per_row, ++row;
    }
    load();  // the next group, on its way while this one is rounded
    uint32_t q[4];
    float scale, by;
    uint8_t* values = static_cast<uint8_t*>(p.values) + row_now * p.values_stride;
    const uint32_t differ = quantize_group<GATE ? kGatedUnits : 0, GATE>(
        v, far, [&]() { return gated_top<T, WIDE>(x, channels, group_now, lane8); }, q, scale, by);
    store_bytes<WIDE>(values, channels, group_now, lane8, q);
    if (differ != 0) gated_patch<T, WIDE>(x, values, channels, group_now, lane8, differ, by);
    if (lane8 == 0 && in) p.scale[row_now * p.scale_row + group_now * p.scale_group] = scale;
  }
}

template <typename T, bool GATE>
cudaError_t launch(QuantizeParams p, cudaStream_t stream) {
  const bool wide = p.channels % 8 == 0 && p.x_stride % (16 / static_cast<int>(sizeof(T))) == 0 &&
                    reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.values_stride % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(p.values) % 8 == 0;
  p.per_row = (static_cast<uint32_t>(p.channels) + kScaleGroup - 1) / kScaleGroup;
  const unsigned long long groups = static_cast<unsigned long long>(p.per_row) * p.rows;
  const unsigned long long blocks = (groups + kGroups - 1) / kGroups;
  const uint32_t resident = kBlocks * device_sm_count();
  const uint32_t grid = blocks < resident ? static_cast<uint32_t>(blocks) : resident;
  p.skip_rows = grid * kGroups / p.per_row, p.skip_groups = grid * kGroups % p.per_row;
  auto go = [&](auto kern) { return launch_kernel(kern, dim3(grid), dim3(kThreads), 0, stream, p); };
  return wide ? go(quantize_kernel<T, GATE, true>) : go(quantize_kernel<T, GATE, false>);
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
