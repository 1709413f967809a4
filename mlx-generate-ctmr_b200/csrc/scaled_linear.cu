// The product of 8-bit rows with an 8-bit weight, both with scales along blocks of 128 inputs:
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] (sum_{k in block b} x[m, k] w[n, k]) + bias[n].
//
// tcgen05 products of kind::f8f6f4 make each block's sum in TMEM; a block is one 128-byte swizzled row of shared memory
// and four products. The scales change with every block, so the epilogue's warps take each block's sums out of
// TMEM and add them, scaled, to sums that they keep in fp32 registers, while the next blocks' products run. That also
// bounds how long a sum stays inside the tensor core.
//
// Two forms. Pairs of CTAs take 256 rows x 256 outputs, rows as TMEM lanes: a thread then has one row scale and one
// weight scale a block, and 128 products and additions. Few rows take tiles of 128 outputs as lanes by 16 to
// 128 rows as columns, with the inputs split over a cluster: all SMs stream the weight at the memory's rate, and the
// partial sums meet through distributed shared memory, in the order of the ranks.
//
// 8,191 rows of 4,096 -> 12,288: 394 us in short runs (2,090 TFLOP/s), 427 to 436 back to back, where the power cap
// holds the clock near 1.48 GHz. A block takes a pair some 930 clocks, its products 512. The way from the products' end
// to the sums' warps (250), through their loads (320) and back (300) is longer than the other buffer's products, and two
// buffers fill TMEM; but by these figures two blocks would take 512 + 870 clocks, 691 each: the other 240 are not
// accounted for. (Halves of 128 outputs with four buffers, one CTA to a tile of 128 x 256, and sixteen warps for the sums were slower.)
// 32 rows of 4,096 -> 4,096: 8.1 us, one of 11,264 -> 4,096 11.7 (3.9 TB/s of weight): a launch, the first loads and the
// exchange take 4 to 5 us of both.
#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "eight_bit.cuh"
#include "launch.cuh"

namespace ctmr {
namespace {

constexpr int kK = kScaleGroup;
constexpr uint32_t kHalfTile = 128 * 128;  // 128 rows of 128 bytes

struct ScaledMaps {
  CUtensorMap x, w, y;  // y: CTA pairs only, and where rows of y allow it
};

struct ScaledPlan {
  int tile, row_tiles, out_tiles;
  int split;   // CTAs (a cluster) that share a tile's blocks; 0: CTA pairs
  int copied;  // y's map is there
};

template <typename T>
__device__ __forceinline__ float bias_at(const ScaledLinearParams& p, int o) {
  if (p.bias == nullptr || o >= p.out) return 0.f;
  return p.bias_f32 ? static_cast<const float*>(p.bias)[o] : to_float(static_cast<const T*>(p.bias)[o]);
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"  // volatile: in order with the barriers
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// N values of a row from output o on; WIDE: the address allows 16-byte accesses and all of them are the row's.
template <typename T, int N>
__device__ __forceinline__ void store_outputs(T* at, const float* v, bool wide, int left) {
  if (wide && left >= N) {
    constexpr int kEach = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
    struct alignas(kEach * sizeof(T)) Pack {
      T e[kEach];
    };
#pragma unroll
    for (int i = 0; i < N; i += kEach) {
      Pack pack;
#pragma unroll
      for (int e = 0; e < kEach; ++e) pack.e[e] = from_float<T>(v[i + e]);
      *reinterpret_cast<Pack*>(at + i) = pack;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) at[i] = from_float<T>(v[i]);
  }
}

// ---------------------------------------------------------------- few rows
constexpr int kFewThreads = 224;  // warp 0 TMA, warp 1 MMA, warps 2-5 sums, warp 6 scales

// A stage holds two blocks: waiting for a barrier costs a warp some 100 clocks, the products of a block of few rows less.
// A tile of 16 rows leaves room for two CTAs on an SM. (Of 32 rows only with two stages each, which is slower.)
template <int BN>
struct FewSmem {
  static constexpr int kCtas = BN <= 16 ? 2 : 1;
  static constexpr uint32_t kBlockBytes = kHalfTile + BN * 128, kStageBytes = 2 * kBlockBytes;
  static constexpr int kStages = (kCtas == 2 ? 112640 : 200704) / kStageBytes;
  static constexpr int kAcc = 2;      // stages whose sums are in TMEM
  static constexpr int kFactors = 2;  // fours of blocks whose scales are in shared memory
  static constexpr uint32_t kCols = 2 * kAcc * BN;
  static constexpr uint32_t kOffFactors = kStages * kStageBytes;
  static constexpr uint32_t kOffBar = kOffFactors + kFactors * 4 * BN * 4;
  static constexpr uint32_t kBytes = kOffBar + 256 + 1024;  // + barriers + alignment slack
  static_assert(BN * 512u <= kOffFactors, "the partial sums lie in the stages");
  static_assert((2 * kStages + 2 * kAcc + 2 * kFactors) * 8 + 16 <= 256, "barriers");
  static_assert(kCtas * (kBytes + 1024) <= 228 * 1024, "shared memory of an SM");
};

// blockIdx.x = (row tile * out tiles + out tile) * split + rank.
template <int BN, typename T>
__global__ void __launch_bounds__(kFewThreads, FewSmem<BN>::kCtas)
    scaled_few_kernel(const __grid_constant__ ScaledMaps maps, const __grid_constant__ ScaledLinearParams p,
                      const __grid_constant__ ScaledPlan plan) {
  using L = FewSmem<BN>;
  constexpr int S = L::kStages, A = L::kAcc, F = L::kFactors;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* factors = reinterpret_cast<float*>(smem + L::kOffFactors);  // [F][BN]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_empty = acc_full + A;
  uint64_t* factor_full = acc_empty + A;
  uint64_t* factor_empty = factor_full + F;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(factor_empty + F);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % plan.split, unit = static_cast<int>(blockIdx.x) / plan.split;
  const int row_tile = unit / plan.out_tiles, m0 = (unit - row_tile * plan.out_tiles) * 128, r0 = row_tile * BN;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < A; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    for (int i = 0; i < F; ++i) {
      mbar_init(&factor_full[i], 1);
      mbar_init(&factor_empty[i], 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int kb = (p.in + kK - 1) / kK, k_begin = rank * kb / plan.split, k_end = (rank + 1) * kb / plan.split;
  griddep_wait();
  griddep_launch_dependents();

  const int n = k_end - k_begin, stages = (n + 1) / 2;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    bool ok = true;
    int it = 0;
    for (; ok && it < stages; ++it) {
      const int s = it % S, blocks = min(2, n - 2 * it);
      if (it >= S) ok = mbar_wait_warp(&empty[s], static_cast<uint32_t>(it / S - 1) & 1u, kErrWaitEmpty);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[s], blocks * L::kBlockBytes);
        for (int h = 0; h < blocks; ++h) {
          uint8_t* at = smem + s * L::kStageBytes + h * L::kBlockBytes;
          tma_load_2d(at, &maps.w, &full[s], (k_begin + 2 * it + h) * kK, m0);
          tma_load_2d(at + kHalfTile, &maps.x, &full[s], (k_begin + 2 * it + h) * kK, r0);
        }
      }
      __syncwarp();
    }
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
    constexpr uint32_t id = idesc_e4m3(128, BN);
    bool ok = true;
    for (int it = 0; it < stages; ++it) {
      const int s = it % S, a = it % A;
      ok = mbar_wait_warp(&full[s], static_cast<uint32_t>(it / S) & 1u, kErrWaitFull);
      if (it >= A) ok = ok && mbar_wait_warp(&acc_empty[a], static_cast<uint32_t>(it / A - 1) & 1u, kErrWaitAcc);
      if (!ok) break;
      tc_fence_after();
      const uint64_t ad = desc_advance(d0, static_cast<uint32_t>(s) * L::kStageBytes);
      const bool both = 2 * it + 1 < n;
      if (elect_one()) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
          if (h == 0 || both)
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
              umma_f8(tm + (2 * a + h) * BN, desc_advance(ad, h * L::kBlockBytes + k * 32u),
                      desc_advance(ad, h * L::kBlockBytes + kHalfTile + k * 32u), id, k > 0 ? 1u : 0u);
        umma_commit(&empty[s]);
        umma_commit(&acc_full[a]);
      }
      __syncwarp();
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
  } else if (warp == 6) {
    // ------------------------------------------------------------ scales, four blocks at a time
    constexpr int kEach = (BN + 31) / 32;
    const float* xs[kEach];
    bool in[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int c = j * 32 + lane;
      in[j] = c < BN && r0 + c < p.rows;
      xs[j] = p.x_scale + (in[j] ? (r0 + c) * p.xs_row : 0);
    }
    const float* ws = p.w_scale + (m0 / kScaleGroup) * p.ws_row;
    bool ok = true;
    for (int it = 0; ok && 4 * it < n; ++it) {
      float v[4][kEach], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k_begin + 4 * it + i;
        w[i] = 4 * it + i < n ? ws[k * p.ws_block] : 0.f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[i][j] = 4 * it + i < n && in[j] ? xs[j][k * p.xs_block] : 0.f;
      }
      const int f = it % F;
      if (it >= F) ok = mbar_wait_warp(&factor_empty[f], static_cast<uint32_t>(it / F - 1) & 1u, kErrWaitEmpty);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (j * 32 + lane < BN) factors[(f * 4 + i) * BN + j * 32 + lane] = v[i][j] * w[i];
      __syncwarp();
      if (lane == 0) mbar_arrive(&factor_full[f]);
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
  } else {
    // ------------------------------------------------------------ sums
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    float sum[BN];
#pragma unroll
    for (int c = 0; c < BN; ++c) sum[c] = 0.f;
    bool ok = true;
    for (int it = 0; it < stages; ++it) {
      const int a = it % A, f = it / 2 % F;
      if (it % 2 == 0) ok = mbar_wait_warp(&factor_full[f], static_cast<uint32_t>(it / 2 / F) & 1u, kErrWaitFull);
      ok = ok && mbar_wait_warp(&acc_full[a], static_cast<uint32_t>(it / A) & 1u, kErrWaitAcc);
      if (!ok) break;
      tc_fence_after();
      const int blocks = min(2, n - 2 * it);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == blocks) break;
        const float4* by = reinterpret_cast<const float4*>(factors + (f * 4 + it % 2 * 2 + h) * BN);
        const uint32_t at = lanes + (2 * a + h) * BN;
        float v[2][16];
        tmem_ld16_start(at, v[0]);
#pragma unroll
        for (int c = 0; c < BN; c += 16) {
          float(&now)[16] = v[(c / 16) & 1];
          tmem_ld_wait();
          tmem_ld_fence16(now);
          if (c + 16 < BN) {
            tmem_ld16_start(at + c + 16, v[(c / 16 + 1) & 1]);
          } else if (h + 1 == blocks) {  // all read
            tc_fence_before();
            if (lane == 0) mbar_arrive(&acc_empty[a]);
          }
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 s = by[(c + e) / 4];
            sum[c + e] = fmaf(now[e], s.x, sum[c + e]);
            sum[c + e + 1] = fmaf(now[e + 1], s.y, sum[c + e + 1]);
            sum[c + e + 2] = fmaf(now[e + 2], s.z, sum[c + e + 2]);
            sum[c + e + 3] = fmaf(now[e + 3], s.w, sum[c + e + 3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0 && (it % 2 == 1 || it + 1 == stages)) mbar_arrive(&factor_empty[f]);
    }
    if (!ok) *abort_flag = 1;
    const int o = m0 + quarter * 32 + lane;
    if (plan.split > 1) {
      // The stages' data are consumed: they hold the partial tile now, [column][output].
      float* part = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int c = 0; c < BN; ++c) part[c * 128 + quarter * 32 + lane] = sum[c];
    } else if (ok && o < p.out) {
      const float bias = bias_at<T>(p, o);
      T* y = static_cast<T*>(p.y) + r0 * p.y_stride + o;
#pragma unroll
      for (int c = 0; c < BN; ++c)
        if (r0 + c < p.rows) y[c * p.y_stride] = from_float<T>(sum[c] + bias);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (plan.split > 1) {
    cluster_sync();
    if (!*abort_flag) {
      // Each CTA adds up its share of the columns: four outputs a thread, a column a warp.
      const int o = m0 + lane * 4;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = bias_at<T>(p, o + e);
      const bool wide = p.y_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % (4 * sizeof(T)) == 0;
      const int c_begin = rank * BN / plan.split, c_end = min((rank + 1) * BN / plan.split, p.rows - r0);
      constexpr int kBatch = 4, kWarps = kFewThreads / 32;
      for (int c = c_begin + warp; c < c_end; c += kWarps * kBatch) {
        float v[kBatch][4];
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[e][i] = 0.f;
#pragma unroll 2
        for (int z = 0; z < plan.split; ++z) {
          const uint32_t at = cluster_addr(smem, z) + lane * 16;
#pragma unroll
          for (int e = 0; e < kBatch; ++e) {
            const float4 t = ld_cluster4(at + min(c + e * kWarps, c_end - 1) * 512);
            v[e][0] += t.x, v[e][1] += t.y, v[e][2] += t.z, v[e][3] += t.w;
          }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int column = c + e * kWarps;
          if (column >= c_end) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[e][i] += bias[i];
          store_outputs<T, 4>(static_cast<T*>(p.y) + (r0 + column) * p.y_stride + o, v[e], wide, p.out - o);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its partial tile
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

// By a warp: 32 rows (a lane's sums are one) of COLUMNS outputs, 64 bytes of each row at a time by way of shared memory;
// for rows of y that TMA does not take (not 16-byte aligned). A lane then holds 16 bytes of a row and stores them element
// by element, 16 bytes from its neighbour's: slow where the outputs are many and the products few (8,191 x 4,096 ->
// 12,287: 747 us, 12,288: 378 to 423; 16,000 x 64 -> 12,289: 890, 12,288: 72; 8,968 x 512 -> 1,537: 117, 1,536: 35).
template <typename T, int COLUMNS>
__device__ __forceinline__ void write_rows(const ScaledLinearParams& p, uint8_t* store, const float* sum, int row0, int o0,
                                           int lane) {
  constexpr int kPer = 16 / sizeof(T), kWide = 4 * kPer;  // outputs in 16 bytes, in 64
#pragma unroll
  for (int c = 0; c < COLUMNS; c += kWide) {
    if (o0 + c >= p.out) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // 16 bytes each, in an order by which neither side meets a bank twice
      alignas(16) T e[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) e[i] = from_float<T>(sum[c + j * kPer + i]);
      *reinterpret_cast<uint4*>(store + lane * 64 + (j ^ (lane >> 1 & 3)) * 16) = *reinterpret_cast<const uint4*>(e);
    }
    __syncwarp();
    const int chunk = lane & 3, o = o0 + c + chunk * kPer;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + lane / 4;
      const uint4 v = *reinterpret_cast<const uint4*>(store + r * 64 + (chunk ^ (r >> 1 & 3)) * 16);
      if (row0 + r >= p.rows) continue;
      T* y = static_cast<T*>(p.y) + (row0 + r) * p.y_stride + o;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int x = 0; x < kPer; ++x)
        if (o + x < p.out) y[x] = e[x];
    }
    __syncwarp();
  }
}

// The same by TMA, 128 bytes of each row at a time from two boxes in turn: the warp goes on to the next tile while they
// are written. (8,191 x 4,096 -> 12,288: 473 us with stores by the warps, 13 % of them waiting for the stores of
// all SMs at once.)
template <typename T, int COLUMNS>
__device__ __forceinline__ void copy_rows(const CUtensorMap& map, const ScaledLinearParams& p, uint8_t* store,
                                          const float* sum, int row0, int o0, int lane) {
  constexpr int kPer = 16 / sizeof(T), kBox = 8 * kPer;  // outputs in 16 bytes, in 128
#pragma unroll
  for (int c = 0; c < COLUMNS; c += kBox) {
    uint8_t* box = store + (c / kBox & 1) * 4096;
    if (lane == 0) bulk_groups_read<1>();  // the box's last copy, two groups ago, has read it
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      alignas(16) T e[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) e[i] = from_float<T>(sum[c + j * kPer + i]);
      *reinterpret_cast<uint4*>(box + lane * 128 + (j ^ (lane & 7)) * 16) = *reinterpret_cast<const uint4*>(e);
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) {
      if (row0 < p.rows && o0 + c < p.out) tma_store_2d(&map, box, o0 + c, row0);
      bulk_group_end();
    }
  }
}

// sum += v by, 16 of them, two to an instruction.
__device__ __forceinline__ void add_scaled(float* sum, const float (&v)[16], float by) {
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%0, %1};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "+f"(sum[i]), "+f"(sum[i + 1])
        : "f"(v[i]), "f"(v[i + 1]), "f"(by));
}

// ---------------------------------------------------------------- CTA pairs
constexpr int kSumWarps = 8, kColumns = 1024 / kSumWarps;
constexpr int kPairThreads = 96 + 32 * kSumWarps;  // warp 0 TMA, warp 1 MMA (first CTA), warp 2 scales, the others sums
constexpr int kPairTile = 256;
constexpr int kPairStages = 4;
constexpr uint32_t kPairStageBytes = 2 * kHalfTile;  // this CTA's 128 rows and 128 outputs
constexpr int kPairFactors = 3;  // fours of blocks whose scales are in shared memory: [block][half of the outputs][row]
constexpr uint32_t kStoreBytes = 2 * 4096;  // a warp's two boxes of 32 rows of 128 bytes
constexpr uint32_t kPairOffStore = kPairStages * kPairStageBytes;
constexpr uint32_t kPairOffFactors = kPairOffStore + kSumWarps * kStoreBytes;
constexpr uint32_t kPairOffBar = kPairOffFactors + kPairFactors * 4 * 256 * 4;
constexpr uint32_t kPairBytes = kPairOffBar + 512 + 1024;
constexpr int kRaster = 8;  // row tiles that are walked together, so that the weight's and x's tiles meet in L2

// 256 rows x 256 outputs per pair (tcgen05.mma.cta_group::2), persistent. A CTA's 128 x 256 sums of a block are
// half its TMEM: the products of one block run while the other's sums are taken out, 128 of a row to a thread.
template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    scaled_pair_kernel(const __grid_constant__ ScaledMaps maps, const __grid_constant__ ScaledLinearParams p,
                       const __grid_constant__ ScaledPlan plan) {
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairOffBar);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;      // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2] read out by both CTAs (first CTA's barriers)
  uint64_t* factor_full = acc_empty + 2;
  uint64_t* factor_empty = factor_full + kPairFactors;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(factor_empty + kPairFactors);
  float* factors = reinterpret_cast<float*>(smem + kPairOffFactors);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

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
      mbar_init(&acc_empty[i], 2 * kSumWarps);
    }
    for (int i = 0; i < kPairFactors; ++i) {
      mbar_init(&factor_full[i], 1);
      mbar_init(&factor_empty[i], kSumWarps);
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
  griddep_wait();
  griddep_launch_dependents();

  auto place = [&](int t, int& r0, int& n0) {
    const int per = kRaster * plan.out_tiles, group = t / per, in_group = t - group * per;
    const int height = min(kRaster, plan.row_tiles - group * kRaster);
    r0 = (group * kRaster + in_group % height) * kPairTile + static_cast<int>(rank) * 128;  // this CTA's rows
    n0 = in_group / height * kPairTile;
  };

  const int kb = (p.in + kK - 1) / kK;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t full0 = cluster_addr(full, 0);
    int it = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      int r0, n0;
      place(t, r0, n0);
      for (int k = 0; k < kb; ++k, ++it) {
        const int s = it % S;
        if (it >= S) ok = mbar_wait_warp(&empty[s], static_cast<uint32_t>(it / S - 1) & 1u, kErrWaitEmpty);
        if (!ok) break;
        if (lane == 0) {
          uint8_t* at = smem + s * kPairStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStageBytes);
          tma_load_2d_pair(at, &maps.x, full0 + 8u * s, k * kK, r0);
          tma_load_2d_pair(at + kHalfTile, &maps.w, full0 + 8u * s, k * kK, n0 + static_cast<int>(rank) * 128);
        }
        __syncwarp();
      }
    }
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
      constexpr uint32_t id = idesc_e4m3(256, kPairTile);
      const uint32_t tm = warp_value(tmem), base = warp_value(smem_u32(smem));
      const uint64_t d0 = smem_desc_kmajor(base, 128);
      const int my_tiles = warp_value(pair < tiles ? (tiles - pair + pairs - 1) / pairs : 0), blocks = my_tiles * kb;
      bool ok = true;
      for (int it = 0; it < blocks; ++it) {
        const int s = it % S, a = it & 1;
        ok = mbar_wait_warp(&full[s], static_cast<uint32_t>(it / S) & 1u, kErrWaitFull);
        // Last, as it is the one that others wait behind.
        if (it >= 2) ok = ok && mbar_wait_warp(&acc_empty[a], static_cast<uint32_t>((it >> 1) - 1) & 1u, kErrWaitAcc);
        if (!ok) break;
        tc_fence_after();
        const uint64_t ad = desc_advance(d0, static_cast<uint32_t>(s) * kPairStageBytes), bd = desc_advance(ad, kHalfTile);
        if (elect_one()) {
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)
            umma_f8_pair(tm + a * 256, desc_advance(ad, k * 32u), desc_advance(bd, k * 32u), id, k > 0 ? 1u : 0u);
          umma_commit_pair(&empty[s]);
          umma_commit_pair(&acc_full[a]);
        }
        __syncwarp();
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales (both CTAs), four blocks' loads at a time.
    // (In the registers of the warps that use them there is no room to have them loaded ahead.)
    int it = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      int r0, n0;
      place(t, r0, n0);
      const float* xs[4];
      const float* ws[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) xs[j] = r0 + j * 32 + lane < p.rows ? p.x_scale + (r0 + j * 32 + lane) * p.xs_row : nullptr;
#pragma unroll
      for (int j = 0; j < 2; ++j) ws[j] = n0 + j * 128 < p.out ? p.w_scale + (n0 / kScaleGroup + j) * p.ws_row : nullptr;
      for (int k0 = 0; ok && k0 < kb; k0 += 4) {
        float x[4][4], w[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = k0 + i < kb;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] = in && xs[j] != nullptr ? xs[j][(k0 + i) * p.xs_block] : 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) w[i][j] = in && ws[j] != nullptr ? ws[j][(k0 + i) * p.ws_block] : 0.f;
        }
        const int f = it % kPairFactors;
        if (it >= kPairFactors)
          ok = mbar_wait_warp(&factor_empty[f], static_cast<uint32_t>(it / kPairFactors - 1) & 1u, kErrWaitEmpty);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) factors[(f * 4 + i) * 256 + j * 32 + lane] = x[i][j & 3] * w[i][j >> 2];
        __syncwarp();
        if (lane == 0) mbar_arrive(&factor_full[f]);
        ++it;
      }
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
  } else {
    // ------------------------------------------------------------ sums (both CTAs)
    const int quarter = warp & 3, columns = (warp - 3) / 4 * kColumns;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + columns;
    const uint32_t release0 = cluster_addr(acc_empty, 0);
    const float* my_factor = factors + columns / 128 * 128 + quarter * 32 + lane;
    int it = 0, group = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      int r0, n0;
      float sum[kColumns];
#pragma unroll
      for (int c = 0; c < kColumns; ++c) sum[c] = 0.f;
      if (p.bias != nullptr) {
        place(t, r0, n0);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) sum[c] = bias_at<T>(p, n0 + columns + c);
      }
      for (int k = 0; k < kb; ++k, ++it) {
        const int a = it & 1, f = group % kPairFactors;
        if ((k & 3) == 0) {
          ok = mbar_wait_warp(&factor_full[f], static_cast<uint32_t>(group / kPairFactors) & 1u, kErrWaitFull);
          // All lanes are past the four before.
          if (lane == 0 && group > 0) mbar_arrive(&factor_empty[(group - 1) % kPairFactors]);
        }
        const float by = my_factor[(f * 4 + (k & 3)) * 256];
        ok = ok && mbar_wait_warp(&acc_full[a], static_cast<uint32_t>(it >> 1) & 1u, kErrWaitAcc);
        if (!ok) break;
        tc_fence_after();
        // 16 sums at a time, waited for and then added: a second array, for loads ahead, would be 16 registers more, which
        // the sums do not leave.
        float v[16];
#pragma unroll
        for (int c = 0; c < kColumns; c += 16) {
          tmem_ld16_start(lanes + a * 256 + c, v);
          tmem_ld_wait();
          tmem_ld_fence16(v);
          if (c + 16 == kColumns) {  // all read: the next block but one may overwrite it
            tc_fence_before();
            if (lane == 0) mbar_arrive_remote(release0 + 8u * a);
          }
          add_scaled(sum + c, v, by);
        }
        group += (k & 3) == 3 || k + 1 == kb;
      }
      ok = ok && __all_sync(0xffffffffu, !*abort_flag);
      if (!ok) break;
      // The tile's place once more: kept over the loop it would cost registers that the sums need.
      int tile = t, thread = threadIdx.x;
      asm volatile("" : "+r"(tile), "+r"(thread));
      place(tile, r0, n0);
      const int at_lane = thread & 31, at_warp = thread >> 5;
      r0 += (at_warp & 3) * 32, n0 += (at_warp - 3) / 4 * kColumns;
      uint8_t* store = smem + kPairOffStore + (at_warp - 3) * kStoreBytes;
      if (plan.copied) copy_rows<T, kColumns>(maps.y, p, store, sum, r0, n0, at_lane);
      else write_rows<T, kColumns>(p, store, sum, r0, n0, at_lane);
    }
    if (lane == 0) bulk_groups_done();
    __syncwarp();
    if (!ok) *abort_flag = 1;
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
int encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long columns, long long rows,
           long long row_bytes, int box_columns, int box_rows, const char* what) {
  auto enc = api_tensor_map_encoder();
  if (enc == nullptr) return api_fail(CTMR_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_columns), static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
  const CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return api_fail(CTMR_ERR_INVALID, "%s: tensor map rejected (CUresult %d)", what, int(r));
  return CTMR_OK;
}

// Which form, tile and split: the least of these estimates (microseconds), fitted to runs of 1 to 1,000 rows with 512
// to 11,264 inputs and 512 to 4,096 outputs, which they meet within some 15 %. The output's bytes are not in them, nor
// whether TMA writes its rows: wide outputs of few inputs take longer (16,000 x 64 -> 12,288: 51 estimated, 72 measured;
// 8,968 x 512 -> 1,536: 13 and 34). One CTA to a tile: 2.2 + 0.052 tile for
// the start, the first loads and the stores, 0.185 + 0.001 tile a block of 128 inputs. Split over a cluster, the partial
// sums' way takes longer the more columns there are. CTA pairs: 4.5, and 0.53 a block and 0.6 a tile, whose stores fall
// between the next one's products. (1 row of 4,096 -> 4,096: tiles of 16 rows split four ways 6.5, two ways 7.5, not
// 9.4; 32 rows: tiles of 32 split two ways 8.0, four ways 9.0; 128 rows: of 64 split two ways 10.6, of 128 four ways
// 11.7; 300 rows: of 128 19.8, pairs 19.4; 1,000 rows: pairs 20.6, tiles of 128 38.5.)
ScaledPlan plan_scaled(const ScaledLinearParams& p) {
  ScaledPlan plan{};
  const int sms = device_sm_count(), kb = (p.in + kK - 1) / kK;
  auto waves = [](long long n, int at_once) { return static_cast<float>((n + at_once - 1) / at_once); };
  const long long pair_tiles = ((p.out + 255LL) / 256) * ((p.rows + 255LL) / 256);
  float best = 4.5f + waves(pair_tiles, sms / 2) * (0.6f + kb * 0.53f);
  plan.tile = kPairTile, plan.split = 0, plan.out_tiles = (p.out + 255) / 256;
  for (int tile = 16; tile <= 128; tile *= 2) {
    if (tile > 16 && tile / 2 >= p.rows) break;
    const long long tiles = ((p.out + 127LL) / 128) * ((p.rows + tile - 1LL) / tile);
    const float columns = static_cast<float>(tile < p.rows ? tile : p.rows);
    for (int split = 1; split <= 8 && split <= kb; split *= 2) {
      const float start = split == 1 ? 2.2f + 0.052f * tile
                          : split == 2 ? 4.2f + 0.027f * tile : 4.2f + 0.1f * split + 0.08f * columns;
      // (Clusters that are resident at once: of the 148 SMs, four's take 132 and eight's 120.)
      const int clusters = split <= 2 ? sms / split : split == 4 ? sms * 33 / 148 : sms * 15 / 148;
      // A tile of 16 rows shares its SM with another, which then takes half as long again.
      const float rounds = waves(tiles, clusters), t =
          (tile == 16 ? 0.55f + 0.45f * rounds : rounds) *
          (start + static_cast<float>(kb) / split * (0.185f + 0.001f * tile));
      if (t < best) best = t, plan.tile = tile, plan.split = split, plan.out_tiles = (p.out + 127) / 128;
    }
  }
  plan.row_tiles = (p.rows + plan.tile - 1) / plan.tile;
  return plan;
}

template <int BN, typename T>
cudaError_t launch_few(const ScaledMaps& maps, const ScaledLinearParams& p, const ScaledPlan& plan, unsigned grid,
                       cudaStream_t stream) {
  static SharedMemoryGrant grant;
  return launch_cluster(grant, scaled_few_kernel<BN, T>, grid, kFewThreads, FewSmem<BN>::kBytes, plan.split, stream, maps,
                        p, plan);
}

template <typename T>
int launch(const ScaledLinearParams& p, cudaStream_t stream) {
  ScaledPlan plan = plan_scaled(p);
  ScaledMaps maps;
  constexpr CUtensorMapDataType kByte = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int st = encode(&maps.x, kByte, p.x, p.in, p.rows, p.x_stride, kK, plan.split == 0 ? 128 : plan.tile, "x");
  if (st == CTMR_OK) st = encode(&maps.w, kByte, p.weight, p.in, p.out, p.weight_stride, kK, 128, "weight");
  const long long y_bytes = p.y_stride * static_cast<long long>(sizeof(T));
  plan.copied = plan.split == 0 && y_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  maps.y = maps.w;  // not read otherwise
  if (st == CTMR_OK && plan.copied)
    st = encode(&maps.y, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, p.y, p.out,
                p.rows, y_bytes, 128 / sizeof(T), 32, "y");
  if (st != CTMR_OK) return st;
  const long long tiles = static_cast<long long>(plan.row_tiles) * plan.out_tiles;
  if (tiles * (plan.split > 0 ? plan.split : 1) > 0x3fffffffLL)
    return api_fail(CTMR_ERR_UNSUPPORTED, "scaled_linear: too many tiles");
  cudaError_t e;
  if (plan.split == 0) {
    static ResidentClusters resident;
    static SharedMemoryGrant grant;
    const long long pairs = resident.count(scaled_pair_kernel<T>, 2, kPairThreads, kPairBytes);
    e = launch_cluster(grant, scaled_pair_kernel<T>, static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)),
                       kPairThreads, kPairBytes, 2, stream, maps, p, plan);
  } else {
    const unsigned grid = static_cast<unsigned>(tiles * plan.split);
    if (plan.tile == 16) e = launch_few<16, T>(maps, p, plan, grid, stream);
    else if (plan.tile == 32) e = launch_few<32, T>(maps, p, plan, grid, stream);
    else if (plan.tile == 64) e = launch_few<64, T>(maps, p, plan, grid, stream);
    else e = launch_few<128, T>(maps, p, plan, grid, stream);
  }
  return e == cudaSuccess ? CTMR_OK : api_fail(CTMR_ERR_CUDA, "scaled_linear launch: %s", cudaGetErrorString(e));
}

}  // namespace

int launch_scaled_linear(const ScaledLinearParams& p, int y_dtype, cudaStream_t stream) {
  switch (y_dtype) {
    case CTMR_DTYPE_F32: return launch<float>(p, stream);
    case CTMR_DTYPE_BF16: return launch<__nv_bfloat16>(p, stream);
    default: return launch<__half>(p, stream);
  }
}

}  // namespace ctmr
