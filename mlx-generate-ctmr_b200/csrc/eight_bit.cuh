// Rows in 8 bits: e4m3 values with a scale for every 128 channels, the parameters of the operators that make and
// take them, and how a group of channels is rounded.
//
// The scale of a group is a power of two, the least 2^k (k >= -100) with which its largest magnitude is at most 448:
// dividing by it is exact, so the rounding to e4m3 is the only one, and e4m3's relative step does not depend on
// the scale's mantissa. A group that holds an infinity or a NaN becomes NaN as a whole, scale and values.
//
// The bytes are those that the formula in 64 bits rounds to. Values are computed in 32 bits with an error below
// kNear of themselves; where both ends of that interval round to the same byte, so does everything between. Where
// they do not (one value in some 2^16), that value is computed again in 64 bits. The scale likewise, where the
// largest magnitude is as near to 448 times a power of two.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "tokens.cuh"

namespace ctmr {

constexpr int kScaleGroup = 128;  // channels to a scale
constexpr int kMaxNormChannels = 32768;

struct RowNormParams {
  const void *x, *residual, *weight;  // residual, weight: may be null
  void *y, *sum;                      // sum: may be null, x or residual
  float* scale;                       // null: y is of x's type
  // A row is (token, head); element strides, x's type except y's where y is in 8 bits (bytes).
  long long x_token, x_head, r_token, r_head, y_token, y_head, s_token, s_head, scale_token, scale_group;
  int tokens, heads, channels, weight_f32;
  float eps;
};

struct QuantizeParams {
  const void* x;  // (rows, channels), or (rows, 2 channels) where gated
  void* values;
  float* scale;
  long long x_stride, values_stride, scale_row, scale_group;
  int rows, channels, gate;
};

struct ScaledLinearParams {
  const void *x, *weight, *bias;       // e4m3 rows; bias: fp32 or y's type, or null
  const float *x_scale, *w_scale;      // (rows, blocks of 128 inputs), (blocks of 128 outputs, blocks of 128 inputs)
  void* y;
  long long x_stride, weight_stride, y_stride, xs_row, xs_block, ws_row, ws_block;
  int rows, in, out, bias_f32;
};

cudaError_t launch_row_norm(const RowNormParams& p, int dtype, cudaStream_t stream);
cudaError_t launch_quantize(const QuantizeParams& p, int dtype, cudaStream_t stream);
int launch_scaled_linear(const ScaledLinearParams& p, int y_dtype, cudaStream_t stream);  // a CTMR_ status

// ---------------------------------------------------------------- eight values of a row
// 8 consecutive elements of a row from memory, zeros past `left` of them. WIDE: the row's address, stride and
// length allow 16-byte accesses.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* at, int left, float (&v)[8]) {
  if constexpr (WIDE) {
    uint4 raw[sizeof(T) == 4 ? 2 : 1];
    const bool in = left > 0;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(raw) / 16; ++i)
      raw[i] = in ? reinterpret_cast<const uint4*>(at)[i] : make_uint4(0, 0, 0, 0);
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_float(at[i]) : 0.f;
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store8(T* at, int left, const float (&v)[8]) {
  if constexpr (WIDE) {
    if (left <= 0) return;
    uint4 raw[sizeof(T) == 4 ? 2 : 1];
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
#pragma unroll
    for (uint32_t i = 0; i < sizeof(raw) / 16; ++i) reinterpret_cast<uint4*>(at)[i] = raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) at[i] = from_float<T>(v[i]);
  }
}

// ---------------------------------------------------------------- rounding to e4m3
constexpr float kNear = 0x1p-20f;  // what the 32-bit formulas stay within, several times over

// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two values as e4m3 bytes, to nearest, ties to even, at most 448; the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float by) {
  return make_uint2(e4m3x2(v[0] * by, v[1] * by) | e4m3x2(v[2] * by, v[3] * by) << 16,
                    e4m3x2(v[4] * by, v[5] * by) | e4m3x2(v[6] * by, v[7] * by) << 16);
}

// The byte of a 64-bit value, rounded once: to 32 bits first, with the last bit set where that cut something off, so
// that no tie of the second rounding is one that the first has made.
__device__ __forceinline__ uint32_t e4m3_exact(double v) {
  float f = __double2float_rz(v);
  if (static_cast<double>(f) != v) f = __uint_as_float(__float_as_uint(f) | 1u);
  return e4m3x2(f, 0.f) & 0xffu;
}

// k of the scale 2^k for a finite largest magnitude: 448 is 1.75 * 2^8, so a mantissa above 1.75 carries.
__device__ __forceinline__ int scale_power(float top) {
  return max(static_cast<int>((__float_as_uint(top) + 0x1fffffu) >> 23) - 135, -100);
}

__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

// Rounds a group of 128 channels, 8 to each of the 16 lanes of half a warp, all of which call this. `exact(i)` gives
// value i in 64 bits; without EXACT the values are as they are meant. Returns the 8 bytes, and the scale.
template <bool EXACT, typename Exact>
__device__ __forceinline__ uint2 quantize_group(const float (&v)[8], Exact exact, float& scale) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
#pragma unroll
  for (int i = 8; i > 0; i /= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, i));
  const bool finite = top <= 3.402823466e38f;
  int k = finite ? scale_power(top) : 0;
  if constexpr (EXACT) {
    const int low = finite ? scale_power(top * (1.f - kNear)) : 0;
    if (finite && scale_power(fminf(top * (1.f + kNear), 3.402823466e38f)) != low) {
      double most = 0.0;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) most = fmax(most, fabs(exact(i)));
#pragma unroll
      for (int i = 8; i > 0; i /= 2) most = fmax(most, __shfl_xor_sync(0xffffu << (threadIdx.x & 16), most, i));
      k = most <= ldexp(448.0, low) ? low : low + 1;
    }
  }
  scale = finite ? power_of_two(k) : __int_as_float(0x7fc00000);
  const float by = finite ? power_of_two(-k) : scale;
  if constexpr (EXACT) {
    uint2 q = e4m3x8(v, by * (1.f - kNear));
    const uint2 other = e4m3x8(v, by * (1.f + kNear));
    if (q.x != other.x || q.y != other.y) {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const uint32_t at = (i & 3) * 8, diff = i < 4 ? q.x ^ other.x : q.y ^ other.y;
        if (!(diff >> at & 0xffu)) continue;
        const uint32_t byte = e4m3_exact(ldexp(exact(i), -k)) << at, keep = ~(0xffu << at);
        if (i < 4) q.x = (q.x & keep) | byte;
        else q.y = (q.y & keep) | byte;
      }
    }
    return q;
  } else {
    return e4m3x8(v, by);
  }
}

// Stores 8 bytes, `left` of which are the row's.
template <bool WIDE>
__device__ __forceinline__ void store_bytes(uint8_t* at, int left, uint2 q) {
  if constexpr (WIDE) {
    if (left > 0) *reinterpret_cast<uint2*>(at) = q;
  } else if (left >= 8 && (reinterpret_cast<uintptr_t>(at) & 7) == 0) {
    *reinterpret_cast<uint2*>(at) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) at[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> ((i & 3) * 8));
  }
}

}  // namespace ctmr
