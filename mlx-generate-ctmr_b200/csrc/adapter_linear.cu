// A projection shared by all rows, beside it a low-rank adapter for each segment of rows:
//   y_i = W x_i + b + scale_a up_a (down_a x_i),  a = index[segment of i], no adapter where a < 0.
//
// Two launches. adapter_inner_kernel computes t_i = scale_a down_a x_i (fp32 sums, rounded once to the
// operands' type: it becomes a tensor-core operand, and its rounding is that of y's own adapter part).
// The product kernel then computes y^T tiles, 128 (or a CTA pair's 256) outputs as TMEM lanes by a
// tile of rows as columns: D = W x^T over the input in blocks of 128, and for every segment that
// meets the tile one further block of K = rank, up_a t^T, into the same accumulator. An
// adapter thus costs its own bytes and rank / in of the product, and y is rounded and written once.
//
// t is stored by blocks: block tile + segment for each pair of a row tile and a segment that meet (both
// grow along the rows, so the numbers are distinct and at most tiles + segments - 1), `tile` rows each,
// zeros in the rows of other segments. A block is a TMA box and needs no mask in the product.
//
// The product kernel starts (programmatic launch) while the inner products run: it reads x and W at
// once, whose producers finished before the inner kernel let it start, and waits only for t.
//
// Outputs as lanes: a warp stores 32 adjacent outputs of a row, and few rows (serving) use few
// columns: the tensor core then streams W at the memory's rate.
#include <cmath>

#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "launch.cuh"
#include "tokens.cuh"

namespace ctmr {
namespace {

// Inputs per block: two halves of one 128-byte swizzled row each. (With one half to a block the issuing
// warp's own instructions, some 600 clocks a block, took longer than a pair's products, 512.)
constexpr int kHalf = 64, kK = 2 * kHalf;
constexpr uint32_t kAHalf = 128 * 128;     // 128 outputs x 64 inputs

struct LinearMaps {
  CUtensorMap x, w, up, inner;
};

// What the two product kernels and the inner kernel have to agree on.
struct LinearPlan {
  int tile;      // rows per tile
  int row_tiles, out_tiles;
  int split;     // CTAs (a cluster) that share a tile's blocks; 0: CTA pairs of 256 outputs
  int blocks;    // blocks of t
  int rank_pad;  // t's row length: rank rounded up to the 16 of one product step
};

// ---------------------------------------------------------------- segments of a row tile
// The last s with offsets[s] <= row (0 if none), by a warp.
__device__ __forceinline__ int segment_at_row(const int* offsets, int segments, int row, int lane) {
  return last_segment(segments, lane, [&](int s) { return offsets[s] <= row; });
}

// The segments with an adapter that meet rows [r0, r1), in order; used by a whole warp. The first 32 are
// read at once when the scan begins, ahead of their use.
struct AdapterScan {
  int r0, r1, base, lane;
  unsigned hits;
  bool more;
  int my_adapter, my_lo, my_hi;

  __device__ __forceinline__ void fill(const LinearParams& p) {
    const int s = base + lane;
    bool hit = false, beyond = true;
    if (s < p.segments) {
      const int begin = p.offsets[s], end = min(p.offsets[s + 1], p.rows);
      my_adapter = p.index[s];
      my_lo = max(begin, r0), my_hi = min(end, r1);
      hit = my_lo < my_hi && my_adapter >= 0 && my_adapter < p.adapters;
      beyond = begin >= r1;
    }
    hits = __ballot_sync(0xffffffffu, hit);
    more = __ballot_sync(0xffffffffu, beyond) == 0;
  }
  __device__ __forceinline__ void begin(const LinearParams& p, int row0, int row1, int lane_) {
    r0 = row0, r1 = row1, lane = lane_, hits = 0, more = false, my_adapter = -1, my_lo = my_hi = 0;
    if (p.segments == 0) return;
    base = segment_at_row(p.offsets, p.segments, r0, lane);
    fill(p);
  }
  __device__ __forceinline__ bool next(const LinearParams& p, int& segment, int& adapter, int& lo, int& hi) {
    while (hits == 0) {
      if (!more) return false;
      base += 32;
      fill(p);
    }
    const int src = __ffs(hits) - 1;
    hits &= hits - 1;
    segment = base + src;
    adapter = __shfl_sync(0xffffffffu, my_adapter, src);
    lo = __shfl_sync(0xffffffffu, my_lo, src);
    hi = __shfl_sync(0xffffffffu, my_hi, src);
    return true;
  }
};

// ---------------------------------------------------------------- inner products
// One CTA: 16 rows of one block of t, all ranks (at most NT * 8). Its sixteen warps take the input in turn,
// 32 inputs at a time, and add up in shared memory. Both operands come straight from memory, 16 bytes a
// thread: a thread's eight inputs are dealt to two product steps, the same way for x and down, which
// permutes the sum's order and nothing else. Memory-bound (x once, down once per 16 rows from L2), and
// for few rows bound by latency, which is why so many warps share a sum;
// tcgen05 would want 128 rows and a trip through shared memory for the same bytes.
constexpr int kInnerWarps = 16;

template <bool BF16, int NT>
__global__ void __launch_bounds__(kInnerWarps * 32) adapter_inner_kernel(const LinearParams p, const LinearPlan plan) {
  constexpr int kParts = NT <= 4 ? 16 : (NT == 8 ? 8 : 4);  // sums held at once, within 48 KB
  __shared__ float part[kParts][16][NT * 8 + 1];
  griddep_wait();
  griddep_launch_dependents();  // after the wait: what starts now may read all that came before this kernel
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block = blockIdx.x;
  if (block == plan.blocks) {  // one more than there are
    if (blockIdx.y > 0) return;
    report_offsets(p.offsets, p.segments, p.rows);
    for (int i = threadIdx.x; i < p.segments; i += blockDim.x)
      if (p.index[i] >= p.adapters) flag_error(kErrBadOffsets);
    return;
  }
  int s, begin, end, adapter;
  if (p.segments <= 32) {  // all of them in one round of loads
    const bool is = lane < p.segments;
    const int a = is ? p.offsets[lane] : 0, b = is ? p.offsets[lane + 1] : 0, mine = is ? p.index[lane] : -1;
    const bool ok = lane == 0 || (is && max(a, 0) / plan.tile + lane <= block);
    s = 31 - __clz(__ballot_sync(0xffffffffu, ok));
    const int a_s = __shfl_sync(0xffffffffu, a, s), b_s = __shfl_sync(0xffffffffu, b, s);
    adapter = __shfl_sync(0xffffffffu, mine, s);
    begin = min(max(a_s, 0), p.rows), end = min(max(b_s, begin), p.rows);
  } else {
    s = segment_of_tile(p.offsets, p.segments, plan.tile, block, lane);
    segment_range(p.offsets, s, p.rows, begin, end);
    adapter = p.index[s];
  }
  const int tile = block - s, row0 = tile * plan.tile + blockIdx.y * 16;
  const int lo = max(begin, tile * plan.tile), hi = min(end, (tile + 1) * plan.tile);
  if (tile < 0 || lo >= hi || adapter < 0 || adapter >= p.adapters) return;  // no such block, or none is read
  uint16_t* inner = static_cast<uint16_t*>(p.inner) +
                    (static_cast<long long>(block) * plan.tile + blockIdx.y * 16) * plan.rank_pad;
  if (row0 >= hi || row0 + 16 <= lo) {
    if (plan.split == 0)  // a pair's product takes the whole tile of rows
      for (int i = threadIdx.x; i < 16 * plan.rank_pad / 8; i += kInnerWarps * 32)
        reinterpret_cast<uint4*>(inner)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int g = lane >> 2, c = lane & 3;
  const bool in0 = row0 + g >= lo && row0 + g < hi, in1 = row0 + g + 8 >= lo && row0 + g + 8 < hi;
  const uint16_t* x0 = static_cast<const uint16_t*>(p.x) + (row0 + g) * p.x_stride;
  const uint16_t* x1 = x0 + 8 * p.x_stride;
  const uint16_t* d = static_cast<const uint16_t*>(p.down) + static_cast<long long>(adapter) * p.rank * p.in;
  const float scale = p.scale[adapter];
  float acc[NT][4] = {};
  // Loads of kDepth turns are started before the first one's products.
  constexpr int kDepth = NT <= 2 ? 5 : (NT <= 4 ? 2 : 1), kTurn = kInnerWarps * 32;
  for (int k0 = warp * 32; k0 < p.in; k0 += kTurn * kDepth) {
    uint4 a0[kDepth], a1[kDepth], b[kDepth][NT];
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int k = k0 + i * kTurn + c * 8;
      const bool in = k < p.in;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      a0[i] = in && in0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero;
      a1[i] = in && in1 ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        b[i][n] = in && n * 8 + g < p.rank
                      ? __ldg(reinterpret_cast<const uint4*>(d + static_cast<long long>(n * 8 + g) * p.in + k)) : zero;
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const uint32_t u0[4] = {a0[i].x, a1[i].x, a0[i].y, a1[i].y}, u1[4] = {a0[i].z, a1[i].z, a0[i].w, a1[i].w};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_16816<BF16>(acc[n], u0, b[i][n].x, b[i][n].y);
        mma_16816<BF16>(acc[n], u1, b[i][n].z, b[i][n].w);
      }
    }
  }
  // Groups of kParts warps, the last first: each adds what the one after it left in its place.
#pragma unroll
  for (int turn = kInnerWarps / kParts - 1; turn >= 0; --turn) {
    if (warp / kParts == turn) {
      float(*mine)[NT * 8 + 1] = part[warp % kParts];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& at = mine[g + (i >> 1) * 8][n * 8 + 2 * c + (i & 1)];
          at = turn == kInnerWarps / kParts - 1 ? acc[n][i] : at + acc[n][i];
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 16 * plan.rank_pad; i += kInnerWarps * 32) {
    const int r = i / plan.rank_pad, n = i - r * plan.rank_pad;
    float v = 0.f;
    if (n < p.rank && row0 + r >= lo && row0 + r < hi) {  // zeros elsewhere, whatever this adapter makes of a zero
#pragma unroll
      for (int q = 0; q < kParts; ++q) v += part[q][r][n];
      v *= scale;
    }
    if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(inner)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(inner)[i] = __float2half_rn(v);
  }
}

// ---------------------------------------------------------------- product, one CTA (or a cluster) per tile
constexpr int kSmallThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue

template <int BN>
struct SmallSmem {
  static constexpr uint32_t kBHalf = BN * 128, kOffB = 2 * kAHalf;
  static constexpr uint32_t kStageBytes = kOffB + 2 * kBHalf;
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr uint32_t kOffBar = kStages * kStageBytes;
  static constexpr uint32_t kBytes = kOffBar + 512 + 1024;  // + barriers + alignment slack
  // (A warp reads columns in batches that span BN / 4: at a split of eight the last share's reach past the tile.)
  static_assert((BN + BN / 8) * 512u <= kOffBar, "the partial sums and what is read past them lie in the stages");
};

// A block as the producer hands it to the MMA thread beside its data: product steps (16 inputs each),
// first column and columns of the product, and whether it is the last.
__device__ __forceinline__ uint32_t pack_block(int steps, int col, int cols, bool last) {
  return static_cast<uint32_t>(steps) | static_cast<uint32_t>(col) << 4 | static_cast<uint32_t>(cols) << 16 |
         (last ? 1u << 31 : 0u);
}

__device__ __forceinline__ float bias_of(const LinearParams& p, bool bf16, int o) {
  if (p.bias == nullptr || o >= p.out) return 0.f;
  if (p.bias_f32) return static_cast<const float*>(p.bias)[o];
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[o])
              : __half2float(static_cast<const __half*>(p.bias)[o]);
}

template <bool BF16>
__device__ __forceinline__ void store16(void* y, long long i, float v) {
  if constexpr (BF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(y)[i] = __float2half_rn(v);
}

// ---------------------------------------------------------------- outputs that are not finite
// An adapter's block meets every row of its tile, with t = 0 in those of other segments, and zero times an
// infinity in `up` is NaN: one request's broken adapter would spoil its neighbours. So an accumulator that is not
// finite is not taken at its word: that output is computed by itself, from its own row and its own adapter.
// (Finite calls pay one operation an output for the test: 617 rows of 512 -> 1,536 went from 9.9 to 10.3 us. 8,192
// rows of 4,096 -> 4,096, 203 us: 11 ms beside one row whose adapter is all NaN, 77 ms with all of W NaN.)
template <bool BF16>
__device__ __forceinline__ float dot8(const void* a, const void* b) {
  const uint4 ua = *static_cast<const uint4*>(a), ub = *static_cast<const uint4*>(b);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t wa = (&ua.x)[i], wb = (&ub.x)[i];
    float2 fa, fb;
    if constexpr (BF16) {
      fa = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wa));
      fb = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wb));
    } else {
      fa = __half22float2(*reinterpret_cast<const __half2*>(&wa));
      fb = __half22float2(*reinterpret_cast<const __half2*>(&wb));
    }
    sum = fmaf(fa.x, fb.x, sum), sum = fmaf(fa.y, fb.y, sum);
  }
  return sum;
}

// By a whole warp: bit e of a lane's `bad` names row row0 + e / OUTS * step and output o + e % OUTS of this lane.
template <bool BF16, int OUTS>
__device__ __noinline__ void alone(const LinearParams& p, const LinearPlan& plan, unsigned bad, int row0, int step, int o) {
  griddep_wait();  // t is complete
  const int lane = threadIdx.x & 31;
  const uint16_t *x = static_cast<const uint16_t*>(p.x), *w = static_cast<const uint16_t*>(p.weight);
  const uint16_t *up = static_cast<const uint16_t*>(p.up), *inner = static_cast<const uint16_t*>(p.inner);
  while (const unsigned who = __ballot_sync(0xffffffffu, bad != 0)) {
    const int src = __ffs(who) - 1, e = __ffs(__shfl_sync(0xffffffffu, bad, src)) - 1;
    const int row = row0 + e / OUTS * step, out = __shfl_sync(0xffffffffu, o, src) + e % OUTS;
    float sum = 0.f;
    for (int k = lane * 8; k < p.in; k += 256) sum += dot8<BF16>(x + row * p.x_stride + k, w + out * p.weight_stride + k);
    const int s = segment_at_row(p.offsets, p.segments, row, lane), a = p.index[s];
    if (row >= p.offsets[s] && row < p.offsets[s + 1] && a >= 0 && a < p.adapters && lane * 8 < p.rank) {
      const long long t = static_cast<long long>(row / plan.tile + s) * plan.tile + row % plan.tile;
      sum += dot8<BF16>(inner + t * plan.rank_pad + lane * 8, up + (static_cast<long long>(a) * p.out + out) * p.rank + lane * 8);
    }
#pragma unroll
    for (int i = 16; i > 0; i /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if (lane == src) {
      store16<BF16>(p.y, row * p.y_stride + out, sum + bias_of(p, BF16, out));
      bad &= bad - 1;
    }
  }
}

// z, zero, as long as all of the values are finite; NaN once one is not.
template <int N>
__device__ __forceinline__ float test_finite(const float (&v)[N], float z) {
#pragma unroll
  for (int e = 0; e < N; ++e) z = fmaf(v[e], 0.f, z);
  return z;
}

__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) <= 3.402823466e38f; }

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"  // volatile: in order with the barriers
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// blockIdx.x = (row tile * out tiles + out tile) * split + rank. Rank r of a cluster takes its share of the
// input blocks and every split-th adapter block; the partial tiles meet through distributed shared
// memory, each CTA adding up and writing its share of the columns.
template <int BN, bool BF16>
__global__ void __launch_bounds__(kSmallThreads, 1)
    linear_small_kernel(const __grid_constant__ LinearMaps maps, const __grid_constant__ LinearParams p,
                        const __grid_constant__ LinearPlan plan) {
  using L = SmallSmem<BN>;
  constexpr int S = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* info = tmem_slot + 2;  // [S]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % plan.split, unit = static_cast<int>(blockIdx.x) / plan.split;
  const int row_tile = unit / plan.out_tiles, m0 = (unit - row_tile * plan.out_tiles) * 128, r0 = row_tile * BN;
  constexpr uint32_t kCols = BN < 32 ? 32 : BN;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (p.segments == 0) griddep_wait();  // otherwise x, W and the segments are complete already
  griddep_launch_dependents();

  const int kb = (p.in + kK - 1) / kK, k_begin = rank * kb / plan.split, k_end = (rank + 1) * kb / plan.split;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    int it = 0;
    bool ok = true;
    auto stage = [&](int s) {
      return it < S || mbar_wait_warp(&empty[s], static_cast<uint32_t>(it / S - 1) & 1u, kErrWaitEmpty);
    };
    // Adapter blocks known from the start, so that the last input block knows whether more follow.
    AdapterScan scan;
    scan.begin(p, r0, min(r0 + BN, p.rows), lane);
    int ordinal = 0, seg = 0, adapter = 0, lo = 0, hi = 0;
    auto next_mine = [&]() {
      while (scan.next(p, seg, adapter, lo, hi))
        if (ordinal++ % plan.split == rank) return true;
      return false;
    };
    bool more = next_mine();
    for (int k = k_begin; ok && k < k_end; ++k, ++it) {
      const int s = it % S, left = p.in - k * kK, halves = left > kHalf ? 2 : 1;
      ok = stage(s);
      if (ok && lane == 0) {
        uint8_t* at = smem + s * L::kStageBytes;
        info[s] = pack_block(min(kK, left + 15) / 16, 0, BN, k + 1 == k_end && !more);
        mbar_arrive_expect_tx(&full[s], halves * (kAHalf + L::kBHalf));
        for (int h = 0; h < halves; ++h) {
          tma_load_2d(at + h * kAHalf, &maps.w, &full[s], k * kK + h * kHalf, m0);
          tma_load_2d(at + L::kOffB + h * L::kBHalf, &maps.x, &full[s], k * kK + h * kHalf, r0);
        }
      }
      __syncwarp();
    }
    // Adapter blocks, up to a ring of them at a time: up's part at once, t's after the inner products. Every
    // CTA waits for those, adapters or not, so this grid cannot end before theirs does.
    const int halves = plan.rank_pad > kHalf ? 2 : 1;
    bool waited = p.segments == 0;
    while (ok && more) {
      const int first = it;
      int my_block = 0;  // lane i: the block of t of stage first + i
      while (ok && more && it < first + S) {
        const int s = it % S;
        ok = stage(s);
        if (!ok) break;
        if (lane == it - first) my_block = row_tile + seg;
        const int a = adapter, c0 = (lo - r0) & ~15, c1 = (hi - r0 + 15) & ~15;
        more = next_mine();
        if (lane == 0) {
          info[s] = pack_block(plan.rank_pad / 16, c0, c1 - c0, !more);
          mbar_arrive_expect_tx(&full[s], halves * (kAHalf + L::kBHalf));
          for (int h = 0; h < halves; ++h)
            tma_load_3d(smem + s * L::kStageBytes + h * kAHalf, &maps.up, &full[s], h * kHalf, m0, a);
        }
        __syncwarp();
        ++it;
      }
      if (!waited) griddep_wait();
      waited = true;
      for (int i = first; i < it; ++i) {
        const int block = __shfl_sync(0xffffffffu, my_block, i - first), s = i % S;
        if (lane == 0)
          for (int h = 0; h < halves; ++h)
            tma_load_2d(smem + s * L::kStageBytes + L::kOffB + h * L::kBHalf, &maps.inner, &full[s], h * kHalf,
                        block * BN);
        __syncwarp();
      }
    }
    if (!waited) griddep_wait();
    if (lane == 0) {
      if (!ok) *abort_flag = 1;
      for (int i = max(0, it - S); i < it; ++i)  // every issued load lands before the CTA goes on
        mbar_wait_bounded(&full[i % S], static_cast<uint32_t>(i / S) & 1u, kErrWaitDrain);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer: a warp that stays together
    const uint32_t tm = warp_value(tmem), base = warp_value(smem_u32(smem));
    const uint64_t d0 = smem_desc_kmajor(base, 128);
    const int plain = warp_value(k_end - k_begin) - 1;  // whole blocks that need no word from the producer
    bool ok = true, last = false;
    for (int it = 0; ok && !last; ++it) {
      const int s = it % S;
      ok = mbar_wait_warp(&full[s], static_cast<uint32_t>(it / S) & 1u, kErrWaitFull);
      if (!ok) break;
      tc_fence_after();
      uint32_t steps = 8, col = 0, cols = BN;
      if (it >= plain) {
        const uint32_t b = warp_value(static_cast<uint32_t>(info[s]));
        steps = b & 15u, col = (b >> 4) & 0xfffu, cols = (b >> 16) & 0x7fffu, last = b >> 31;
      }
      const uint64_t ad = desc_advance(d0, static_cast<uint32_t>(s) * L::kStageBytes);
      const uint64_t bd = desc_advance(ad, L::kOffB + col * 128u);
      const uint32_t id = idesc_f16(BF16, 128, cols);
      if (elect_one()) {
        if (steps == 8) {
#pragma unroll
          for (uint32_t k = 0; k < 8; ++k)
            umma_f16(tm + col, desc_advance(ad, (k >> 2) * kAHalf + (k & 3) * 32u),
                     desc_advance(bd, (k >> 2) * L::kBHalf + (k & 3) * 32u), id, it > 0 || k > 0 ? 1u : 0u);
        } else {
#pragma unroll 1
          for (uint32_t k = 0; k < steps; ++k)
            umma_f16(tm + col, desc_advance(ad, (k >> 2) * kAHalf + (k & 3) * 32u),
                     desc_advance(bd, (k >> 2) * L::kBHalf + (k & 3) * 32u), id, it > 0 || k > 0 ? 1u : 0u);
        }
        umma_commit(&empty[s]);
        if (last) umma_commit(done);
      }
      __syncwarp();
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, o = m0 + quarter * 32 + lane;
    const float bias = bias_of(p, BF16, o);
    const bool ok = mbar_wait_warp(done, 0, kErrWaitAcc) && __all_sync(0xffffffffu, !*abort_flag);
    tc_fence_after();
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    float z = 0.f;
    for (int c = 0; c < BN; c += 16) {
      float v[16];
      tmem_ld16(tmem + lanes + c, v);
      if (plan.split > 1) {
        // The stages' data are consumed: they hold the partial tile now, [column][output].
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int e = 0; e < 16; ++e) part[(c + e) * 128 + quarter * 32 + lane] = v[e];
      } else if (ok && o < p.out) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (r0 + c + e < p.rows) store16<BF16>(p.y, static_cast<long long>(r0 + c + e) * p.y_stride + o, v[e] + bias);
      }
      z = test_finite(v, z);
    }
    if (plan.split == 1 && ok && p.segments > 0 && __any_sync(0xffffffffu, z != 0.f)) {
      for (int c = 0; c < BN; c += 16) {
        float v[16];
        tmem_ld16(tmem + lanes + c, v);
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (o < p.out && r0 + c + e < p.rows && !is_finite(v[e])) bad |= 1u << e;
        alone<BF16, 1>(p, plan, bad, r0 + c, 1, o);
      }
    }
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (plan.split > 1) {
    cluster_sync();
    if (warp >= 2 && !*abort_flag) {
      // Four outputs a thread, a column a warp.
      const int o = m0 + lane * 4;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = bias_of(p, BF16, o + e);
      const bool wide = o + 4 <= p.out && p.y_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % 8 == 0;
      const int c_end = min((rank + 1) * BN / plan.split, p.rows - r0);
      constexpr int kBatch = BN / 16;  // columns read together, a warp's share of them at a split of four
      for (int c = rank * BN / plan.split + warp - 2; c < c_end; c += 4 * kBatch) {
        float4 v[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) v[e] = make_float4(bias[0], bias[1], bias[2], bias[3]);
#pragma unroll 4
        for (int z = 0; z < plan.split; ++z) {
          const uint32_t at = cluster_addr(smem, z) + (c * 128 + lane * 4) * 4;
#pragma unroll
          for (int e = 0; e < kBatch; ++e) {
            const float4 t = ld_cluster4(at + e * 4 * 512);  // past the share: anything, and not used
            v[e].x += t.x, v[e].y += t.y, v[e].z += t.z, v[e].w += t.w;
          }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          if (c + 4 * e >= c_end) break;
          const long long at = static_cast<long long>(r0 + c + 4 * e) * p.y_stride + o;
          if (wide) {
            uint2 h;
            if constexpr (BF16) {
              const __nv_bfloat162 h0 = __floats2bfloat162_rn(v[e].x, v[e].y);
              const __nv_bfloat162 h1 = __floats2bfloat162_rn(v[e].z, v[e].w);
              h = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
            } else {
              const __half2 h0 = __floats2half2_rn(v[e].x, v[e].y), h1 = __floats2half2_rn(v[e].z, v[e].w);
              h = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
            }
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) = h;
          } else {
            const float u[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (o + i < p.out) store16<BF16>(p.y, at + i, u[i]);
          }
        }
        if (p.segments > 0) {
          float z = 0.f;
#pragma unroll
          for (int e = 0; e < kBatch; ++e)
            if (c + 4 * e < c_end) z = fmaf(v[e].x, 0.f, fmaf(v[e].y, 0.f, fmaf(v[e].z, 0.f, fmaf(v[e].w, 0.f, z))));
          if (__any_sync(0xffffffffu, z != 0.f)) {
            unsigned bad = 0;
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
              const float u[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (c + 4 * e < c_end && o + i < p.out && !is_finite(u[i])) bad |= 1u << (e * 4 + i);
            }
            alone<BF16, 4>(p, plan, bad, r0 + c, 4, o);
          }
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its partial tile
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

// ---------------------------------------------------------------- product, CTA pairs
constexpr int kPairThreads = 320;  // warp 0 TMA, warp 1 MMA (first CTA), warps 2-9 epilogue
constexpr int kPairRows = 256;
constexpr int kPairStages = 3;
constexpr uint32_t kPairOffB = 2 * kAHalf, kPairStageBytes = 4 * kAHalf;  // this CTA's 128 outputs and 128 rows
constexpr uint32_t kPairOffBar = kPairStages * kPairStageBytes;
constexpr uint32_t kPairBytes = kPairOffBar + 512 + 1024;
constexpr int kRaster = 8;  // row tiles that are walked together, so that W's and x's tiles meet in L2

// 256 outputs x 256 rows per pair of CTAs (tcgen05.mma.cta_group::2): each CTA loads half of W's rows and
// half of x's, i.e. 64 bytes per clock and SM at the tensor cores' full rate where one CTA's own
// 128 x 256 tile would take 96. Two accumulators in TMEM: a tile is written while the next is computed.
template <bool BF16>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ LinearMaps maps, const __grid_constant__ LinearParams p,
                       const __grid_constant__ LinearPlan plan) {
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairOffBar);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;      // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2] read out by both CTAs (first CTA's barriers)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* info = tmem_slot + 2;  // [S]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
  const int tiles = plan.row_tiles * plan.out_tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before anything crosses the pair
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (p.segments == 0) griddep_wait();
  griddep_launch_dependents();

  auto place = [&](int t, int& row_tile, int& m0) {
    const int per = kRaster * plan.out_tiles, group = t / per, in_group = t - group * per;
    const int height = min(kRaster, plan.row_tiles - group * kRaster);
    row_tile = group * kRaster + in_group % height;
    m0 = in_group / height * 256;
  };

  const int kb = (p.in + kK - 1) / kK;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t full0 = cluster_addr(full, 0);
    int it = 0;
    bool ok = true, waited = p.segments == 0;
    auto stage = [&](int s) {
      return it < S || mbar_wait_warp(&empty[s], static_cast<uint32_t>(it / S - 1) & 1u, kErrWaitEmpty);
    };
    const int rank_halves = plan.rank_pad > kHalf ? 2 : 1;
    for (int t = pair; ok && t < tiles; t += pairs) {
      int row_tile, m0;
      place(t, row_tile, m0);
      const int r0 = row_tile * kPairRows, my_m = m0 + static_cast<int>(rank) * 128;
      const int my_r = r0 + static_cast<int>(rank) * 128;
      AdapterScan scan;
      scan.begin(p, r0, min(r0 + kPairRows, p.rows), lane);
      int seg, adapter, lo, hi;
      bool more = scan.next(p, seg, adapter, lo, hi);
      for (int k = 0; ok && k < kb; ++k, ++it) {
        const int s = it % S, left = p.in - k * kK, halves = left > kHalf ? 2 : 1;
        ok = stage(s);
        if (ok && lane == 0) {
          uint8_t* at = smem + s * kPairStageBytes;
          if (rank == 0) {
            info[s] = pack_block(min(kK, left + 15) / 16, 0, kPairRows, k + 1 == kb && !more);
            mbar_arrive_expect_tx(&full[s], halves * 4u * kAHalf);
          }
          for (int h = 0; h < halves; ++h) {
            tma_load_2d_pair(at + h * kAHalf, &maps.w, full0 + 8u * s, k * kK + h * kHalf, my_m);
            tma_load_2d_pair(at + kPairOffB + h * kAHalf, &maps.x, full0 + 8u * s, k * kK + h * kHalf, my_r);
          }
        }
        __syncwarp();
      }
      if (!waited) {
        griddep_wait();
        waited = true;
      }
      while (ok && more) {
        const int row = (row_tile + seg) * kPairRows + static_cast<int>(rank) * 128, a = adapter, s = it % S;
        more = scan.next(p, seg, adapter, lo, hi);
        ok = stage(s);
        if (ok && lane == 0) {
          uint8_t* at = smem + s * kPairStageBytes;
          if (rank == 0) {
            info[s] = pack_block(plan.rank_pad / 16, 0, kPairRows, !more);
            mbar_arrive_expect_tx(&full[s], rank_halves * 4u * kAHalf);
          }
          for (int h = 0; h < rank_halves; ++h) {
            tma_load_3d_pair(at + h * kAHalf, &maps.up, full0 + 8u * s, h * kHalf, my_m, a);
            tma_load_2d_pair(at + kPairOffB + h * kAHalf, &maps.inner, full0 + 8u * s, h * kHalf, row);
          }
        }
        __syncwarp();
        ++it;
      }
    }
    if (!waited) griddep_wait();
    if (lane == 0) {
      if (!ok) *abort_flag = 1;
      // The first CTA's barriers count both CTAs' bytes: all land before the closing cluster barrier.
      if (rank == 0)
        for (int i = max(0, it - S); i < it; ++i)
          if (!mbar_wait_bounded(&full[i % S], static_cast<uint32_t>(i / S) & 1u, kErrWaitDrain)) break;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (first CTA): a warp that stays together
    if (rank == 0) {
      const uint32_t id = idesc_f16(BF16, 256, kPairRows);
      const uint32_t tm = warp_value(tmem), base = warp_value(smem_u32(smem));
      const uint64_t d0 = smem_desc_kmajor(base, 128);
      const int plain = warp_value(kb) - 1;  // whole blocks that need no word from the producer
      int it = 0, lt = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs, ++lt) {
        const int buf = lt & 1;
        if (lt >= 2) ok = mbar_wait_warp(&acc_empty[buf], static_cast<uint32_t>((lt >> 1) - 1) & 1u, kErrWaitAcc);
        bool last = false;
        for (int k = 0; ok && !last; ++k, ++it) {
          const int s = it % S;
          ok = mbar_wait_warp(&full[s], static_cast<uint32_t>(it / S) & 1u, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          uint32_t steps = 8;
          if (k >= plain) {
            const uint32_t b = warp_value(static_cast<uint32_t>(info[s]));
            steps = b & 15u, last = b >> 31;
          }
          const uint64_t ad = desc_advance(d0, static_cast<uint32_t>(s) * kPairStageBytes);
          const uint64_t bd = desc_advance(ad, kPairOffB);
          if (elect_one()) {
            if (steps == 8) {
#pragma unroll
              for (uint32_t i = 0; i < 8; ++i)
                umma_f16_pair(tm + buf * 256, desc_advance(ad, (i >> 2) * kAHalf + (i & 3) * 32u),
                              desc_advance(bd, (i >> 2) * kAHalf + (i & 3) * 32u), id, k > 0 || i > 0 ? 1u : 0u);
            } else {
#pragma unroll 1
              for (uint32_t i = 0; i < steps; ++i)
                umma_f16_pair(tm + buf * 256, desc_advance(ad, (i >> 2) * kAHalf + (i & 3) * 32u),
                              desc_advance(bd, (i >> 2) * kAHalf + (i & 3) * 32u), id, k > 0 || i > 0 ? 1u : 0u);
            }
            umma_commit_pair(&empty[s]);
            if (last) umma_commit_pair(&acc_full[buf]);
          }
          __syncwarp();
        }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t release0 = cluster_addr(acc_empty, 0);
    int lt = 0;
    for (int t = pair; t < tiles; t += pairs, ++lt) {
      int row_tile, m0;
      place(t, row_tile, m0);
      const int o = m0 + static_cast<int>(rank) * 128 + quarter * 32 + lane, buf = lt & 1;
      const float bias = bias_of(p, BF16, o);
      if (!mbar_wait_warp(&acc_full[buf], static_cast<uint32_t>(lt >> 1) & 1u, kErrWaitAcc) ||
          __any_sync(0xffffffffu, *abort_flag)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      for (int c = half * 128; c < half * 128 + 128; c += 32) {
        float v[32];
        tmem_ld32(lanes + buf * 256 + c, v);
        tmem_ld_wait();
        tmem_ld_fence(v);
        if (c == half * 128 + 96) {  // all read: the next tile but one may overwrite it
          tc_fence_before();
          if (lane == 0) mbar_arrive_cluster(release0 + 8u * buf);
        }
        const int row = row_tile * kPairRows + c;
        if (o < p.out) {
          long long at = static_cast<long long>(row) * p.y_stride + o;
#pragma unroll
          for (int e = 0; e < 32; ++e, at += p.y_stride)
            if (row + e < p.rows) store16<BF16>(p.y, at, v[e] + bias);
        }
        if (p.segments > 0 && __any_sync(0xffffffffu, test_finite(v, 0.f) != 0.f)) {
          unsigned bad = 0;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (o < p.out && row + e < p.rows && !is_finite(v[e])) bad |= 1u << e;
          alone<BF16, 1>(p, plan, bad, row, 1, o);
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA exits while the other's products, copies or arrivals may reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------- host
// CTA pairs that are resident at once: one pair more would run alone after all the others.
int resident_pairs() {
  static ResidentClusters resident;
  return resident.count(linear_pair_kernel<true>, 2, kPairThreads, kPairBytes);
}

int encode(CUtensorMap* map, const void* base, bool bf16, int rank, long long d0, long long d1, long long d2,
           long long s1, long long s2, int box_rows, const char* what) {
  auto enc = api_tensor_map_encoder();
  if (enc == nullptr) return api_fail(CTMR_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d0), static_cast<cuuint64_t>(d1), static_cast<cuuint64_t>(d2)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(s1 * 2), static_cast<cuuint64_t>(s2 * 2)};
  const cuuint32_t box[3] = {kHalf, static_cast<cuuint32_t>(box_rows), 1}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return api_fail(CTMR_ERR_INVALID, "%s: tensor map rejected (CUresult %d)", what, int(r));
  return CTMR_OK;
}

// Which kernel, tile and split: the least of these estimates (microseconds), fitted to runs of 1 to 1,300 rows
// with 256 to 4,096 inputs and outputs, which they meet within some 20 %. One CTA per tile: a wave of them takes
// 2.8 + 0.032 tile, plus 0.8 + 0.01 tile where a cluster splits the input, plus 0.32 + 0.0011 tile per block of 128
// inputs. CTA pairs of 256 x 256, which overlap a tile's stores with the next one's products: 8 in all and 0.62 per
// block. (617 rows of 512 -> 1,536: tiles of 64 rows 6.0, of 128 8.2, of 32 9.1, pairs 10.6; 617 rows of
// 4,096 -> 4,096: pairs 29, tiles of 128 41.)
// Adapters, fitted to 64 to 8,192 rows in segments of 1 to 256 with ranks of 16 to 128: a block of one CTA's tile 0.45
// (0.65 for two halves of rank), a pair's 0.27 (0.52), and 0.012 per CTA of the inner products, of which there are
// tile / 16 to every block of t, most of them idle where segments are short. The best plan was taken within 5 %.
// (4,096 one-row segments of rank 16: 4,096 -> 4,096 tiles of 64 rows 1,048, pairs 1,274; 512 -> 1,536 tiles of 16
// rows 382, pairs 872. With rank 128 their t takes 68 and 17 MB where a pair's takes 270.)
LinearPlan plan_linear(const LinearParams& p) {
  LinearPlan plan{};
  const int sms = device_sm_count(), kb = (p.in + kK - 1) / kK;
  auto waves = [](long long n, int at_once) { return static_cast<float>((n + at_once - 1) / at_once); };
  const bool wide = p.rank > kHalf;
  // Adapter blocks that a tile meets, if the segments' borders lie evenly; and what the inner products add.
  auto blocks = [&](int tile) {
    const float per = 1.f + static_cast<float>(p.segments - 1) / static_cast<float>((p.rows + tile - 1) / tile);
    return p.segments > 0 ? fminf(per, static_cast<float>(tile)) : 0.f;
  };
  auto inner = [&](int tile) {
    return p.segments > 0 ? 0.012f * (tile / 16) * static_cast<float>((p.rows + tile - 1) / tile + p.segments - 1) : 0.f;
  };
  const long long pair_tiles = ((p.out + 255LL) / 256) * ((p.rows + 255LL) / 256);
  float best = 8.f + inner(256) + waves(pair_tiles, sms / 2) * (kb * 0.62f + blocks(256) * (wide ? 0.52f : 0.27f));
  plan.tile = kPairRows, plan.split = 0, plan.out_tiles = (p.out + 255) / 256;
  for (int tile = 16; tile <= 128; tile *= 2) {
    if (tile > 16 && tile / 2 >= p.rows) break;
    const long long tiles = ((p.out + 127LL) / 128) * ((p.rows + tile - 1LL) / tile);
    for (int split = 1; split <= 8 && split <= kb; split *= 2) {
      const float adapters = p.segments > 0 ? fmaxf(blocks(tile) / split, 1.f) * (wide ? 0.65f : 0.45f) : 0.f;
      const float one = 2.8f + 0.032f * tile + (split > 1 ? 0.8f + 0.01f * tile : 0.f) +
                        static_cast<float>(kb) / split * (0.32f + 0.0011f * tile) + adapters;
      const float t = waves(tiles * split, sms) * one + inner(tile);
      if (t < best) best = t, plan.tile = tile, plan.split = split, plan.out_tiles = (p.out + 127) / 128;
    }
  }
  plan.row_tiles = (p.rows + plan.tile - 1) / plan.tile;
  plan.blocks = p.segments > 0 ? plan.row_tiles + p.segments - 1 : 0;
  plan.rank_pad = (p.rank + 15) / 16 * 16;
  return plan;
}

template <bool BF16, int NT>
cudaError_t launch_inner(const LinearParams& p, const LinearPlan& plan, cudaStream_t stream) {
  return launch_kernel(adapter_inner_kernel<BF16, NT>, dim3(plan.blocks + 1, plan.tile / 16), dim3(kInnerWarps * 32),
                       0, stream, p, plan);
}

template <int BN, bool BF16>
cudaError_t launch_small(const LinearMaps& maps, const LinearParams& p, const LinearPlan& plan, unsigned grid,
                         cudaStream_t stream) {
  static SharedMemoryGrant grant;
  return launch_cluster(grant, linear_small_kernel<BN, BF16>, grid, kSmallThreads, SmallSmem<BN>::kBytes, plan.split,
                        stream, maps, p, plan);
}

template <bool BF16>
int launch(const LinearParams& p, const LinearPlan& plan, cudaStream_t stream) {
  LinearMaps maps;
  const int box_rows = plan.split == 0 ? 128 : plan.tile;
  int st = encode(&maps.x, p.x, BF16, 2, p.in, p.rows, 1, p.x_stride, 0, box_rows, "x");
  if (st == CTMR_OK) st = encode(&maps.w, p.weight, BF16, 2, p.in, p.out, 1, p.weight_stride, 0, 128, "weight");
  if (st != CTMR_OK) return st;
  maps.up = maps.inner = maps.w;  // not read without adapters
  cudaError_t e = cudaSuccess;
  if (p.segments > 0) {
    st = encode(&maps.up, p.up, BF16, 3, p.rank, p.out, p.adapters, p.rank, static_cast<long long>(p.rank) * p.out, 128,
                "up");
    if (st == CTMR_OK)
      st = encode(&maps.inner, p.inner, BF16, 2, plan.rank_pad, static_cast<long long>(plan.blocks) * plan.tile, 1,
                  plan.rank_pad, 0, box_rows, "workspace");
    if (st != CTMR_OK) return st;
    if (p.rank <= 16) e = launch_inner<BF16, 2>(p, plan, stream);
    else if (p.rank <= 32) e = launch_inner<BF16, 4>(p, plan, stream);
    else if (p.rank <= 64) e = launch_inner<BF16, 8>(p, plan, stream);
    else e = launch_inner<BF16, 16>(p, plan, stream);
    if (e != cudaSuccess) return api_fail(CTMR_ERR_CUDA, "adapter_linear launch: %s", cudaGetErrorString(e));
  }
  const long long tiles = static_cast<long long>(plan.row_tiles) * plan.out_tiles;
  if (plan.split == 0) {
    const long long pairs = resident_pairs();
    static SharedMemoryGrant grant;
    e = launch_cluster(grant, linear_pair_kernel<BF16>, static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)),
                       kPairThreads, kPairBytes, 2, stream, maps, p, plan);
  } else {
    const unsigned grid = static_cast<unsigned>(tiles * plan.split);
    if (plan.tile == 16) e = launch_small<16, BF16>(maps, p, plan, grid, stream);
    else if (plan.tile == 32) e = launch_small<32, BF16>(maps, p, plan, grid, stream);
    else if (plan.tile == 64) e = launch_small<64, BF16>(maps, p, plan, grid, stream);
    else e = launch_small<128, BF16>(maps, p, plan, grid, stream);
  }
  return e == cudaSuccess ? CTMR_OK : api_fail(CTMR_ERR_CUDA, "adapter_linear launch: %s", cudaGetErrorString(e));
}

}  // namespace

size_t adapter_linear_workspace(const LinearParams& p) {
  const LinearPlan plan = plan_linear(p);
  return static_cast<size_t>(plan.blocks) * plan.tile * plan.rank_pad * 2;
}

int launch_adapter_linear(const LinearParams& p, bool bf16, cudaStream_t stream) {
  const LinearPlan plan = plan_linear(p);
  if (plan.blocks > 0x3fffff) return api_fail(CTMR_ERR_UNSUPPORTED, "too many segments");
  return bf16 ? launch<true>(p, plan, stream) : launch<false>(p, plan, stream);
}

}  // namespace ctmr
