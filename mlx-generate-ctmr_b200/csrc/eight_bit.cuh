// Rows in 8 bits: e4m3 values with a scale for every 128 channels, the parameters of the operators that make and
// take them, and how a group of channels is rounded.
//
// The scale of a group is a power of two, the least 2^k (k >= -100) with which its largest magnitude is at most 448:
// dividing by it is exact, so the rounding to e4m3 is the only one, and e4m3's relative step does not depend on
// the scale's mantissa. A group that holds an infinity or a NaN becomes NaN as a whole, scale and values.
//
// The bytes are those that the formula in 64 bits rounds to. Values are computed in 32 bits and stay within a few
// units of 2^-24 of themselves; where both ends of that interval round to the same byte, so does everything between.
// Where they do not (one value in some 2^17), that value is computed again in 64 bits. The scale likewise, where the
// largest magnitude is as near to 448 times a power of two.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

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
  double per_channel;  // 1 / channels, set by the launcher
};

struct QuantizeParams {  // the last three: set by the launcher
  const void* x;  // (rows, channels), or (rows, 2 channels) where gated
  void* values;
  float* scale;
  long long x_stride, values_stride, scale_row, scale_group;
  int rows, channels, gate;
  uint32_t per_row, skip_rows, skip_groups;
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

// ---------------------------------------------------------------- a group of a row
// Eight lanes hold a group of 128 channels, 16 each: eight consecutive ones of either half where the row's address, stride
// and length allow 16-byte accesses (WIDE), every eighth one otherwise: the eight lanes' accesses lie side by side then, but
// are 8 elements, half a sector of 16-bit ones, and a warp's four groups lie apart (rows of 4,097 take two to three times
// those of 4,096).
constexpr int kEach = 16, kGroupLanes = kScaleGroup / kEach;

template <bool WIDE>
__device__ __forceinline__ int channel_of(int group, int lane8, int e) {
  return group * kScaleGroup + (WIDE ? e / 8 * 64 + lane8 * 8 + e % 8 : lane8 + kGroupLanes * e);
}

// 16 bytes, kept in order with the stores over the same row.
__device__ __forceinline__ uint4 load_bytes16(const void* at) {
  uint4 r;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(at) : "memory");
  return r;
}

// v[at] of registers.
__device__ __forceinline__ float pick(const float (&v)[kEach], int at) {
  float r = v[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) r = at == i ? v[i] : r;
  return r;
}

// A lane's 16 channels of a row as they lie in memory. Past the row's end `values`, by whole warps, gives zeros.
template <typename T, bool WIDE>
struct Loaded {
  static constexpr uint32_t kWords = kEach * sizeof(T) / 4;
  uint32_t raw[WIDE ? kWords : 1];
  T each[WIDE ? 1 : kEach];

  __device__ __forceinline__ void load(const T* row, int channels, int group, int lane8) {
    if constexpr (WIDE) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = channel_of<true>(group, lane8, 8 * half);
        if (c < channels) {
#pragma unroll
          for (uint32_t i = 0; i < kWords / 8; ++i) {
            const uint4 r = load_bytes16(row + c + 4 * i);
            const uint32_t to = half * (kWords / 2) + 4 * i;
            raw[to] = r.x, raw[to + 1] = r.y, raw[to + 2] = r.z, raw[to + 3] = r.w;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int c = channel_of<false>(group, lane8, i);
        each[i] = c < channels ? row[c] : from_float<T>(0.f);
      }
    }
  }

  __device__ __forceinline__ void values(float (&v)[kEach], int channels, int group, int lane8) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if constexpr (!WIDE) {
        v[i] = to_float(each[i]);
      } else if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(raw[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw[i / 2]));
        v[i] = i % 2 ? f.y : f.x;
      } else {
        v[i] = __uint_as_float(i % 2 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
      }
    }
    // (A branch: selects, or zeros ahead of the load, would cost every warp.)
    if (WIDE && __any_sync(0xffffffffu, channel_of<WIDE>(group, lane8, kEach - 1) >= channels))
#pragma unroll
      for (int i = 0; i < kEach; ++i) v[i] = channel_of<WIDE>(group, lane8, i / 8 * 8) < channels ? v[i] : 0.f;
  }
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load16(const T* row, int channels, int group, int lane8, float (&v)[kEach]) {
  Loaded<T, WIDE> in;
  in.load(row, channels, group, lane8);
  in.values(v, channels, group, lane8);
}

// Two values to the 16-bit type, the first in the low half.
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store16(T* row, int channels, int group, int lane8, const float (&v)[kEach]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = channel_of<true>(group, lane8, 8 * half);
      const float* w = v + 8 * half;
      if (c >= channels) continue;
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(row + c)[0] = make_float4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<float4*>(row + c)[1] = make_float4(w[4], w[5], w[6], w[7]);
      } else {
        *reinterpret_cast<uint4*>(row + c) =
            make_uint4(pack2(w[0], w[1], T()), pack2(w[2], w[3], T()), pack2(w[4], w[5], T()), pack2(w[6], w[7], T()));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = channel_of<false>(group, lane8, i);
      if (c < channels) row[c] = from_float<T>(v[i]);
    }
  }
}

template <bool WIDE>
__device__ __forceinline__ void store_bytes(uint8_t* row, int channels, int group, int lane8, const uint32_t (&q)[4]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = channel_of<true>(group, lane8, 8 * half);
      if (c < channels) *reinterpret_cast<uint2*>(row + c) = make_uint2(q[2 * half], q[2 * half + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = channel_of<false>(group, lane8, i);
      if (c < channels) row[c] = static_cast<uint8_t>(q[i / 4] >> (i % 4 * 8));
    }
  }
}

// Products and sums at two to an instruction.
__device__ __forceinline__ void mul16(float (&v)[kEach], const float (&a)[kEach], const float (&b)[kEach]) {
#pragma unroll
  for (int i = 0; i < kEach; i += 2)
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "=f"(v[i]), "=f"(v[i + 1])
        : "f"(a[i]), "f"(a[i + 1]), "f"(b[i]), "f"(b[i + 1]));
}

__device__ __forceinline__ void mul16(float (&v)[kEach], const float (&a)[kEach], float b) {
#pragma unroll
  for (int i = 0; i < kEach; i += 2)
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmul.rn.f32x2 z, x, y;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "=f"(v[i]), "=f"(v[i + 1])
        : "f"(a[i]), "f"(a[i + 1]), "f"(b));
}

// a b + c.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ void add16(float (&v)[kEach], const float (&a)[kEach]) {
#pragma unroll
  for (int i = 0; i < kEach; i += 2)
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 z, x, y;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "+f"(v[i]), "+f"(v[i + 1])
        : "f"(a[i]), "f"(a[i + 1]));
}

// ---------------------------------------------------------------- rounding to e4m3
constexpr float kUnit = 0x1p-24f;  // one rounding of a 32-bit value

__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// The largest of three magnitudes, or of two numbers; NaN if any is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a >= b || a != a ? a : b; }

// The least of three numbers; NaN is none.
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two values as e4m3 bytes, to nearest, ties to even, at most 448; the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

__device__ __forceinline__ void e4m3x16(uint32_t (&q)[4], const float (&v)[kEach], float by) {
  float u[kEach];
  mul16(u, v, by);
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = e4m3x2(u[4 * i], u[4 * i + 1]) | e4m3x2(u[4 * i + 2], u[4 * i + 3]) << 16;
}

// The byte of a 64-bit value, rounded once: to 32 bits first, with the last bit set where that cut something off, so
// that no tie of the second rounding is one that the first has made.
__device__ __forceinline__ uint32_t e4m3_exact(double v) {
  float f = __double2float_rz(v);
  if (static_cast<double>(f) != v) f = __uint_as_float(__float_as_uint(f) | 1u);
  return e4m3x2(f, 0.f) & 0xffu;
}

// k of the scale 2^k for a largest magnitude (any k if it is not finite): 448 is 1.75 * 2^8, so a mantissa above 1.75
// carries.
__device__ __forceinline__ int scale_power(float top) {
  return max(static_cast<int>((__float_as_uint(top) + 0x1fffffu) >> 23) - 135, -100);
}

__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

// Rounds a group of channels, held by eight lanes of a warp all of whose lanes call this. UNITS: how many roundings
// the values are off by at most, the one of scaling them here included; 0: they are as they are meant. `top64()` gives
// the largest magnitude of the lane's values in 64 bits. Gives the 16 bytes, the scale and its inverse, and returns (bit
// i: value i) which values 64 bits have to decide. FAR: a lane that is `far` does not have its values; 64 bits decide its
// whole group, and one whose values left 32 bits' range.
template <int UNITS, bool FAR, typename Top>
__device__ __forceinline__ uint32_t quantize_group(const float (&v)[kEach], bool far, Top top64, uint32_t (&q)[4], float& scale,
                                                   float& by) {
  constexpr float kLow = 1.f - UNITS * kUnit, kHigh = 1.f + 2 * ((UNITS + 1) / 2) * kUnit;
  const float nan = __int_as_float(0x7fc00000);
  float top = max_nan(v[0], v[1], v[2]);
#pragma unroll
  for (int i = 3; i + 1 < kEach; i += 2) top = max_nan(top, v[i], v[i + 1]);
  top = max_nan(top, v[kEach - 1], 0.f);
  if (FAR && far) top = nan;
#pragma unroll
  for (int i = kGroupLanes / 2; i > 0; i /= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, i));
  int k = scale_power(top);
  if constexpr (UNITS > 0) {
    const int low = scale_power(top * kLow);
    k = scale_power(top * kHigh);
    if (FAR ? k != low || !is_finite(top) : k != low && is_finite(top)) {
      double most = top64();
#pragma unroll
      for (int i = kGroupLanes / 2; i > 0; i /= 2)
        most = max_nan(most, __shfl_xor_sync(0xffu << (threadIdx.x & 24), most, i));
      if (!FAR || is_finite(top)) {
        if (most <= ldexp(448.0, low)) k = low;
      } else if (most <= 448.0 * 0x1p127) {  // (an infinity's or a NaN's group stays as it is)
        int exponent;
        const double fraction = frexp(most, &exponent);  // 448 is 0.875 * 2^9
        k = max(most == 0.0 ? -100 : exponent - 9 + (fraction > 0.875), -100);
        scale = power_of_two(k), by = ldexpf(1.f, -k);
        e4m3x16(q, v, 0.f);
        return 0xffffu;
      }
    }
  }
  scale = is_finite(top) ? power_of_two(k) : nan;
  by = is_finite(top) ? power_of_two(-k) : nan;
  uint32_t differ = 0;
  if constexpr (UNITS > 0) {
    uint32_t other[4];
    e4m3x16(q, v, by * kLow);
    e4m3x16(other, v, by * kHigh);
    if ((q[0] ^ other[0]) | (q[1] ^ other[1]) | (q[2] ^ other[2]) | (q[3] ^ other[3]))
#pragma unroll
      for (int i = 0; i < kEach; ++i) differ |= ((q[i / 4] ^ other[i / 4]) >> (i % 4 * 8) & 0xffu) != 0 ? 1u << i : 0u;
  } else {
    e4m3x16(q, v, by);
  }
  return differ;
}

}  // namespace ctmr
