// Root-mean-square norm of rows, with the residual's addition before it and an output in 8 bits where wanted:
//   h = x + r,  s = h / sqrt(mean(h^2) + eps) * w,
// h rounded to x's type beside it, where it is kept (the residual stream of a block).
//
// One pass over memory: a row's values stay in registers between the sum and the scaling. What bounds it is memory, 7
// bytes a channel for 16-bit rows with a residual and an 8-bit output: 8,192 rows of 4,096 take 50 us, 4.7 TB/s
// (without a weight 49, with a 16-bit output, which is 32 MB more to write, 46). Between that and the memory's 36 stand
// latencies: a quarter of an SM's warps, which issue 0.53 instructions a clock and scheduler. The squares are added in 64
// bits: at 3 channels a clock and SM the conversions take a fifth of their unit's time, and the 8-bit rounding gets a
// mean that its 64-bit recomputation can rely on. The norm is taken of the unrounded sum h, so that it does not see
// the stream's rounding.
#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"
#include "launch.cuh"

namespace ctmr {
namespace {

// In units of 2^-24: the sum, the factor, two products and the scaling. (The factor is a normal number for rows of a root
// mean square up to 2^126; h times it may be none, but only weights above 2^15 bring such a value back to what is kept.)
constexpr int kNormUnits = 6;

// What the squares of h lack of those of h + low, but for 2^-44 of them. In 32 bits, which cost a row of 4,096 fp32
// channels 2 % where 64 cost 7 %, as long as `total`, the sum of the squares of h, says that no product leaves them.
// Nothing beside an infinity.
template <int V>
__device__ __forceinline__ double squares_rest(const float (&h)[V][kEach], const float (&low)[V][kEach], double total) {
  if (total > 0x1p100 || (total < 0x1p-60 && total > 0.0)) {
    double rest = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll 1
      for (int e = 0; e < kEach; ++e)
        rest = fma(static_cast<double>(pick(h[i], e)), static_cast<double>(pick(low[i], e)), rest);
    return rest == rest ? 2.0 * rest : 0.0;
  }
  float2 rest = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < kEach; e += 2)
      rest = fma2(make_float2(h[i][e], h[i][e + 1]), make_float2(low[i][e], low[i][e + 1]), rest);
  return 2.0 * (static_cast<double>(rest.x) + static_cast<double>(rest.y));
}

// LANES lanes to a row: 8, 16 or 32 of a warp, or (0) a block. V: groups of channels to eight lanes. LOOP (of blocks):
// a block goes on to another row, whose loads it starts before this row's sum is known, with the weight in registers.
template <typename T, int V, int LANES, bool LOOP, bool EIGHT, bool WIDE>
__global__ void __launch_bounds__(LANES ? 256 : LOOP ? 512 : 1024, 1) row_norm_kernel(const __grid_constant__ RowNormParams p) {
  constexpr bool BLOCK = LANES == 0;
  // Sums of 16-bit numbers are exact in 32 bits but where one is 2^13 times the other, and h is then that sum; 32-bit
  // ones keep the rest.
  constexpr bool kLow = EIGHT && sizeof(T) == 4;
  __shared__ double part[2][BLOCK ? 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane8 = lane & 7;
  const int span = BLOCK ? blockDim.x : LANES;
  // A thread's first group; the next is span / 8 further.
  const int first = (BLOCK ? threadIdx.x : threadIdx.x & (span - 1)) / kGroupLanes, step = span / kGroupLanes;
  const long long rows = static_cast<long long>(p.tokens) * p.heads;
  long long row = BLOCK ? blockIdx.x : (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  griddep_wait();
  griddep_launch_dependents();
  const bool idle = row >= rows;  // part of a warp may be: it stays for the shuffles
  if (idle) row = rows - 1;
  const int channels = idle ? 0 : p.channels;

  int token, head;
  const T *x, *r;
  float h[V][kEach], w[V][kEach], low[kLow ? V : 1][kEach];
  auto at_row = [&](long long i) {
    token = p.heads == 1 ? static_cast<int>(i) : static_cast<int>(i / p.heads);
    head = p.heads == 1 ? 0 : static_cast<int>(i - static_cast<long long>(token) * p.heads);
    x = static_cast<const T*>(p.x) + token * p.x_token + head * p.x_head;
    r = static_cast<const T*>(p.residual) + (p.residual ? token * p.r_token + head * p.r_head : 0);
  };
  auto load_row = [&](Loaded<T, WIDE>(&a)[V], Loaded<T, WIDE>(&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i].load(x, channels, first + i * step, lane8);
    if (p.residual != nullptr)
#pragma unroll
      for (int i = 0; i < V; ++i) b[i].load(r, channels, first + i * step, lane8);
  };
  auto load_weight = [&](int i) {
    if (p.weight_f32) load16<float, WIDE>(static_cast<const float*>(p.weight), channels, first + i * step, lane8, w[i]);
    else load16<T, WIDE>(static_cast<const T*>(p.weight), channels, first + i * step, lane8, w[i]);
  };

  Loaded<T, WIDE> x_in[V], r_in[V];
  at_row(row);
  load_row(x_in, r_in);
  if (LOOP && p.weight != nullptr)
#pragma unroll
    for (int i = 0; i < V; ++i) load_weight(i);
  for (int turn = 0;; turn ^= 1) {
    double sums[4] = {0.0, 0.0, 0.0, 0.0};  // four chains
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x_in[i].values(h[i], channels, first + i * step, lane8);
      if (p.residual != nullptr) {
        float add[kEach];
        r_in[i].values(add, channels, first + i * step, lane8);
        if constexpr (kLow) {  // what the sum's rounding cuts off, exactly
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const float sum = h[i][e] + add[e], back = sum - h[i][e];
            low[i][e] = (h[i][e] - (sum - back)) + (add[e] - back);
          }
        }
        add16(h[i], add);
      } else if constexpr (kLow) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) low[i][e] = 0.f;
      }
    }
    const int token_now = token, head_now = head;
    const bool more = LOOP && row + gridDim.x < rows;
    if (more) {
      row += gridDim.x;
      at_row(row);
      load_row(x_in, r_in);
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        sums[e % 4] = fma(static_cast<double>(h[i][e]), static_cast<double>(h[i][e]), sums[e % 4]);
    double total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    if constexpr (kLow)
      if (p.residual != nullptr) total += squares_rest<V>(h, low, total);
#pragma unroll
    for (int i = (BLOCK ? 32 : LANES) / 2; i > 0; i /= 2) total += __shfl_xor_sync(0xffffffffu, total, i);
    if constexpr (BLOCK) {
      if (lane == 0) part[turn][warp] = total;
      __syncthreads();
      const int warps = blockDim.x >> 5;
      total = part[turn][0];
      for (int i = 1; i < warps; ++i) total += part[turn][i];
    }
    // 1 / sqrt(mean + eps): 32 bits' root and a step of Newton's in 64, good to 2^-43.
    const double mean = fma(total, p.per_channel, static_cast<double>(p.eps));
    double by64;
    if (mean < 0x1p120 && mean > 0x1p-120) {
      by64 = static_cast<double>(rsqrtf(static_cast<float>(mean)));
      by64 = fma(0.5 * by64, fma(-mean * by64, by64, 1.0), by64);
    } else {
      by64 = 1.0 / sqrt(mean);
    }
    const float by = static_cast<float>(by64);

#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int group = first + i * step;
      float s[kEach];
      mul16(s, h[i], by);
      if (p.weight != nullptr) {
        if (!LOOP) load_weight(i);
        mul16(s, s, w[i]);
      }
      if constexpr (EIGHT) {
        if (__any_sync(0xffffffffu, channel_of<WIDE>(group, lane8, kEach - 1) >= channels))  // nothing past the row's end, whatever the factor
#pragma unroll
          for (int e = 0; e < kEach; ++e) s[e] = channel_of<WIDE>(group, lane8, e) < channels ? s[e] : 0.f;
        uint32_t q[4];
        float scale, by8;
        auto exact = [&](int e) {
          double v = static_cast<double>(pick(h[i], e));
          if (kLow) v += static_cast<double>(pick(low[i], e));
          if (p.weight != nullptr) v *= static_cast<double>(pick(w[i], e));
          return v * by64;
        };
        auto top64 = [&]() {
          double most = 0.0;
#pragma unroll 1
          for (int e = 0; e < kEach; ++e) most = fmax(most, fabs(exact(e)));
          return most;
        };
        // From registers: a reload would keep the warp, and the block that waits for it, some microseconds.
        uint32_t differ = quantize_group<kNormUnits, false>(s, false, top64, q, scale, by8);
#pragma unroll 1
        for (; differ != 0; differ &= differ - 1) {
          const int e = __ffs(differ) - 1, bit = (e & 3) * 8;
          const uint32_t byte = e4m3_exact(exact(e) * by8);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j == e >> 2) q[j] = (q[j] & ~(0xffu << bit)) | byte << bit;
        }
        store_bytes<WIDE>(static_cast<uint8_t*>(p.y) + token_now * p.y_token, channels, group, lane8, q);
        if (lane8 == 0 && group * kScaleGroup < channels)
          p.scale[token_now * p.scale_token + group * p.scale_group] = scale;
      } else {
        store16<T, WIDE>(static_cast<T*>(p.y) + token_now * p.y_token + head_now * p.y_head, channels, group, lane8, s);
      }
      // Last, as it may lie where x or r did.
      if (p.sum != nullptr)
        store16<T, WIDE>(static_cast<T*>(p.sum) + token_now * p.s_token + head_now * p.s_head, channels, group, lane8,
                         h[i]);
    }
    if (!more) break;
  }
}

template <typename T, int V, int LANES, bool LOOP, bool EIGHT>
cudaError_t launch(const RowNormParams& p, bool wide, long long grid, int threads, cudaStream_t stream) {
  auto go = [&](auto kern) {
    return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, p);
  };
  return wide ? go(row_norm_kernel<T, V, LANES, LOOP, EIGHT, true>) : go(row_norm_kernel<T, V, LANES, LOOP, EIGHT, false>);
}

template <typename T, bool EIGHT>
cudaError_t launch_rows(const RowNormParams& p, cudaStream_t stream) {
  // 16-byte accesses where every row allows them.
  constexpr int kAlign = 16 / sizeof(T);
  auto row_ok = [](const void* at, long long token, long long head) {
    return at == nullptr || (reinterpret_cast<uintptr_t>(at) % 16 == 0 && token % kAlign == 0 && head % kAlign == 0);
  };
  const bool wide = p.channels % 8 == 0 && row_ok(p.x, p.x_token, p.x_head) && row_ok(p.residual, p.r_token, p.r_head) &&
                    row_ok(p.sum, p.s_token, p.s_head) &&
                    (EIGHT ? reinterpret_cast<uintptr_t>(p.y) % 8 == 0 && p.y_token % 8 == 0
                           : row_ok(p.y, p.y_token, p.y_head)) &&
                    (p.weight == nullptr || reinterpret_cast<uintptr_t>(p.weight) % 16 == 0);
  const long long rows = static_cast<long long>(p.tokens) * p.heads;
  const int groups = (p.channels + kScaleGroup - 1) / kScaleGroup;
  // Lanes to a row: 8, 16 or 32 of a warp, two groups to eight lanes up to 1,024 channels; with few rows a block of one
  // group to eight lanes even there (1,777 rows of 1,001 fp32 channels 7.4 us, by warps 10.7; 300 of 1,024 in bf16 2.8
  // and 3.6; 20,000 rows keep all warps busy either way). Longer rows: blocks that go on from row to row, of up
  // to 128 registers, where these fill their SMs and accesses are wide (8,192 rows of 4,096: 49 us, a block of 64
  // registers to each row 57; of 4,224, whose 288 threads fit once: 90 and 68; of 4,097: 190 and 146), or where there
  // are few rows and a row's own time counts (1,777 rows of 1,001: 7.4 and 10.5; 600 of 2,048: 4.0 and 4.4). The blocks
  // of 64 registers, to which that leaves many rows of 4,097 to 7,040 channels, and all rows above 8,192, are far from
  // the memory's rate and spill: 8,192 rows of 5,120 take 72 us (bytes: 45), of 6,144 100
  // (54), 2,000 of 16,384 97 (35).
  auto grid = [&](int lanes) { return (rows * lanes + 255) / 256; };
  if (groups == 1) return launch<T, 1, 8, false, EIGHT>(p, wide, grid(8), 256, stream);
  if (groups == 2) return launch<T, 1, 16, false, EIGHT>(p, wide, grid(16), 256, stream);
  if (groups <= 4) return launch<T, 1, 32, false, EIGHT>(p, wide, grid(32), 256, stream);
  if (groups <= 8 && rows > 16 * device_sm_count()) return launch<T, 2, 32, false, EIGHT>(p, wide, grid(32), 256, stream);
  auto threads = [&](int v) { return (groups + 4 * v - 1) / (4 * v) * 32; };
  const int at_once = 512 / threads(1);  // blocks on an SM at 128 registers
  const long long resident = static_cast<long long>(device_sm_count()) * at_once;
  if (threads(1) <= 512 && (rows <= 2 * resident || (wide && at_once * threads(1) >= 448)))
    return launch<T, 1, 0, true, EIGHT>(p, wide, rows < resident ? rows : resident, threads(1), stream);
  if (threads(1) <= 512) return launch<T, 1, 0, false, EIGHT>(p, wide, rows, threads(1), stream);
  return launch<T, 2, 0, false, EIGHT>(p, wide, rows, threads(2), stream);
}

}  // namespace

cudaError_t launch_row_norm(const RowNormParams& p_, int dtype, cudaStream_t stream) {
  RowNormParams p = p_;
  p.per_channel = 1.0 / p.channels;
  const bool eight = p.scale != nullptr;
  switch (dtype) {
    case CTMR_DTYPE_F32: return eight ? launch_rows<float, true>(p, stream) : launch_rows<float, false>(p, stream);
    case CTMR_DTYPE_BF16:
      return eight ? launch_rows<__nv_bfloat16, true>(p, stream) : launch_rows<__nv_bfloat16, false>(p, stream);
    default: return eight ? launch_rows<__half, true>(p, stream) : launch_rows<__half, false>(p, stream);
  }
}

}  // namespace ctmr
