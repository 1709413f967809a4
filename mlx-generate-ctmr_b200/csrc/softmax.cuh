// What the two attention kernels share: base-2 exponentials and reciprocals of the special-function unit, paired fp32
// operations, capped scores, 16-bit pairs.
#pragma once

#include <cmath>

#include "tokens.cuh"

namespace ctmr {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_unit(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_unit(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// How scores (products of q and k, before their scale) become capped base-2 scores.
struct ScoreCap {
  float in;    // scale / cap, at most 1e38 so that a zero score stays zero
  float unit;  // scale * log2(e)
  float out;   // cap * log2(e)
};

__device__ __forceinline__ ScoreCap score_cap(float scale, float cap) {
  return {fminf(scale / cap, 1e38f), scale * kLog2e, cap * kLog2e};
}

// c tanh(x / c) of N scores, by how near the largest of any lane comes to the cap:
//   below 0.3 of it  an odd polynomial (x / c times a cubic in its square, maximum relative error 1e-8), with
//                    the powers of the scale in its coefficients: five operations to a pair of scores;
//   below 0.6        x / c times a quartic, 1e-7 (2e-7 with fp32's roundings): eight to a pair;
//   else             that for the scores below 0.6 and c - 2 c / (e^(2 x / c) + 1) for the others: two operations
//                    of the exponential unit to a score. Its absolute error is 2e-7 c, which a small score under a
//                    large cap would feel (a score of 1 under a cap of 1e6 by 0.1).
// So a lane's scores may be capped by one polynomial or the other, 1e-7 apart, as its neighbours' are large or not.
// (Four sequences of 1 to 2,300 tokens, 16 heads of 128, cap 30: 75 us; without the cubic 81, with the last form alone
// 103. 8 heads of 8,192 tokens: 350 to 370 us, 370 to 395 and 515, 545 under a cap of 3; 246 uncapped.)
template <int N>
__device__ __forceinline__ void cap_scores(float (&s)[N], const ScoreCap& cap) {
  float big = 0.f;
#pragma unroll
  for (int c = 0; c < N; ++c) big = fmaxf(big, fabsf(s[c]));
  const float2 zero = make_float2(0.f, 0.f);
  const float in = cap.in, unit = cap.unit;
  auto quartic = [&](float2 v, float2 x) {
    const float2 u = fma2(x, x, zero);
    float2 q = fma2(make_float2(0.015414500613641403f, 0.015414500613641403f), u,
                    make_float2(-0.052054543053197115f, -0.052054543053197115f));
    q = fma2(q, u, make_float2(0.13309036526297813f, 0.13309036526297813f));
    q = fma2(q, u, make_float2(-0.3333222964170574f, -0.3333222964170574f));
    q = fma2(q, u, make_float2(0.9999999342091528f, 0.9999999342091528f));
    return fma2(q, fma2(v, make_float2(unit, unit), zero), zero);
  };
  // (in^6 stays a normal number, and no coefficient grows past the scale itself)
  if (__all_sync(0xffffffffu, big * in <= 0.3f && in >= 1e-4f && in <= 1.f)) {
    const float in2 = in * in, c0 = 0.9999999896019268f * unit, c1 = -0.3333296267971552f * in2 * unit;
    const float c2 = 0.1331259723418185f * in2 * in2 * unit;
    const float c3 = -0.050222438703983206f * in2 * in2 * in2 * unit;
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 v = make_float2(s[c], s[c + 1]), u = fma2(v, v, zero);
      float2 q = fma2(make_float2(c3, c3), u, make_float2(c2, c2));
      q = fma2(q, u, make_float2(c1, c1));
      q = fma2(q, u, make_float2(c0, c0));
      q = fma2(q, v, zero);
      s[c] = q.x, s[c + 1] = q.y;
    }
  } else if (__all_sync(0xffffffffu, big * in <= 0.6f)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 v = make_float2(s[c], s[c + 1]), q = quartic(v, fma2(v, make_float2(in, in), zero));
      s[c] = q.x, s[c + 1] = q.y;
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 v = make_float2(s[c], s[c + 1]), x = fma2(v, make_float2(in, in), zero), q = quartic(v, x);
      auto far = [&](float x) {
        return fmaf(-2.f * cap.out, rcp_unit(exp2_unit(2.f * kLog2e * x) + 1.f), cap.out);
      };
      s[c] = fabsf(x.x) <= 0.6f ? q.x : far(x.x), s[c + 1] = fabsf(x.y) <= 0.6f ? q.y : far(x.y);
    }
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Rows of a packed output before the first document and past the last (q_offsets' ends): zeros, and a log-sum-exp
// of -infinity. One warp of every block of the grid takes its share.
__device__ __forceinline__ void clear_outside(const AttentionParams& p, long long block, long long blocks, int lane) {
  const int first = min(max(p.q_offsets[0], 0), p.q_tokens);
  const int last = min(max(p.q_offsets[p.documents], 0), p.q_tokens);
  const int rows = first + p.q_tokens - last, units = p.heads * (p.dim / 8);
  if (rows == 0 || last < first) return;
  const long long step = blocks * 32, n = static_cast<long long>(rows) * units;
  for (long long i = block * 32 + lane; i < n; i += step) {
    const int r = static_cast<int>(i / units), u = static_cast<int>(i - static_cast<long long>(r) * units);
    const int h = u / (p.dim / 8), d = u - h * (p.dim / 8);
    const long long row = r < first ? r : last + (r - first);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.o_token + h * p.o_head + d * 8) =
        make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr && d == 0) p.lse[row * p.heads + h] = -INFINITY;
  }
}

}  // namespace ctmr
