// The attention of attention_packed.cu for documents of few queries (serving: one new token per request
// over a cache): group x queries rows share each key head's keys, up to 32 to a CTA. The cache is read once and
// that read is the time, so all of the GPU has to read at once: the keys of a (document, key head) are split
// over a cluster of up to 16 CTAs, in steps of 64 that TMA brings into a ring in shared memory (96 KB a CTA, two
// CTAs an SM: 192 KB in flight); each of four warps takes 16 keys of a step. The partial softmaxes meet in
// shared memory and, across the cluster, in distributed shared memory, in one launch.
//
// The products are mma.sync m16n8k16, whose 16 rows fit: tcgen05 would want 128 where there are few. With
// the loads in registers instead of a ring (eight warps an SM, a step's loads then its products) the same
// kernel took 72 us for 16 requests of 4,096 to 8,192 keys, four key heads of 128.
#include <cooperative_groups.h>

#include "ctmr_b200.h"
#include "launch.cuh"
#include "softmax.cuh"

namespace ctmr {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32 + 32;  // four warps compute, one loads
// P and its sum are held 2^15 larger: fp16 rounds numbers below 2^-14 ever more coarsely.
constexpr float kLift = 15.f, kDrop = 1.f / 32768.f;
constexpr int kKeys = 16, kStep = kWarps * kKeys;         // keys per warp and per step

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// MT: row tiles of 16. DC: channel chunks of 64.
template <int MT, int DC>
struct FewSmem {
  static constexpr int kRows = MT * 16, kD = DC * 64;
  static constexpr int kStages = 6 / DC;
  static constexpr uint32_t kChunk = kStep * 128, kStage = 2 * DC * kChunk;  // K then V, chunks of 64 channels
  static constexpr int kPitch = kD + 8;                                      // of Q, 16-bit
  static constexpr uint32_t kOffQ = kStages * kStage, kOffBar = kOffQ + kRows * kPitch * 2;
  static constexpr uint32_t kBytes = kOffBar + 128 + 1024;  // + barriers + alignment slack
  // After the last step the ring holds the warps' sums: [kWarps][kRows][kD], then their (m, l).
  static constexpr uint32_t kOffStat = kWarps * kRows * kD * 4;
  static_assert(kOffStat + kWarps * kRows * 8 <= kOffQ, "the sums fit in the ring");
};

template <int MT, int DC, bool BF16>
__global__ void __launch_bounds__(kThreads, 2)
    attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const AttentionParams p, int splits) {
  using L = FewSmem<MT, DC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint16_t* q_s = reinterpret_cast<uint16_t*>(smem + L::kOffQ);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* empty = full + L::kStages;
  float* o_s = reinterpret_cast<float*>(smem);                   // [kWarps][kRows][kD]
  float* stat_s = reinterpret_cast<float*>(smem + L::kOffStat);  // [kWarps][kRows][2]
  griddep_wait();
  griddep_launch_dependents();
  const int rank = static_cast<int>(blockIdx.x) % splits, doc = static_cast<int>(blockIdx.x) / splits, hk = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    fence_barrier_init();
  }
  const int group = p.heads / p.kv_heads;

  // The document's rows. (All threads of the cluster agree on them.)
  int q_len = p.q_tokens, k_len = p.k_tokens, k_row = 0, map_doc = 0;
  long long q_at = 0, o_at = 0, lse_at = 0;
  if (p.q_offsets != nullptr) {
    int qb, qe, kb, ke;
    segment_range(p.q_offsets, doc, p.q_tokens, qb, qe);
    segment_range(p.k_offsets, doc, p.k_tokens, kb, ke);
    q_len = qe - qb, k_len = ke - kb;
    if (q_len > p.max_q) flag_error(kErrBadOffsets);
    q_at = qb * p.q_token, o_at = qb * p.o_token, lse_at = qb, k_row = kb;
    const long long block = (static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    if (warp == kWarps)  // the one that loads; the queries are loaded by all
      clear_outside(p, block, static_cast<long long>(gridDim.x) * gridDim.y * gridDim.z, lane);
  } else {
    if (p.k_lengths != nullptr) {
      const int n = p.k_lengths[doc];
      k_len = min(max(n, 0), p.k_tokens);
      if (n != k_len) flag_error(kErrBadOffsets);
    }
    q_at = doc * p.q_doc, o_at = doc * p.o_doc, map_doc = doc;
    lse_at = static_cast<long long>(doc) * p.q_tokens;
  }
  const int prefix = p.prefix != nullptr ? p.prefix[doc] : 0, shift = k_len - q_len;
  // Row base + r of the key head's: query (base + r) / group, head (base + r) % group. Calls of more rows than a
  // CTA holds read the keys again for each further kRows of them (blockIdx.z).
  const int queries = min(q_len, p.max_q), base = blockIdx.z * L::kRows;
  const int rows = min(max(queries * group - base, 0), L::kRows);
  auto limit_of = [&](int i) { return p.causal ? min(k_len, max(max(i + shift + 1, prefix), 0)) : k_len; };
  const uint16_t* qp = static_cast<const uint16_t*>(p.q) + q_at;

  // This CTA's keys: a share of those that any row sees, in whole steps.
  const int seen = rows > 0 ? limit_of((base + rows - 1) / group) : 0;
  const int share = (seen + splits * kStep - 1) / (splits * kStep) * kStep;
  const int k0 = min(rank * share, seen), k1 = min(k0 + share, seen), steps = (k1 - k0 + kStep - 1) / kStep;

  for (int i = threadIdx.x; i < L::kRows * (L::kD / 8); i += kThreads) {
    const int r = i / (L::kD / 8), d = (i - r * (L::kD / 8)) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows && d < p.dim)
      v = *reinterpret_cast<const uint4*>(qp + ((base + r) / group) * p.q_token +
                                          (hk * group + (base + r) % group) * p.q_head + d);
    *reinterpret_cast<uint4*>(q_s + r * L::kPitch + d) = v;
  }
  __syncthreads();

  float o[MT][DC * 8][4] = {};
  float m[MT][2], l[MT][2] = {};
  if (warp == kWarps) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      for (int j = 0; j < steps; ++j) {
        const int st = j % L::kStages, use = j / L::kStages;
        if (use > 0 && !mbar_wait_bounded(&empty[st], static_cast<uint32_t>(use - 1) & 1u, kErrWaitEmpty)) {
          for (int i = max(0, j - L::kStages); i < j; ++i)  // what is in flight lands before anything else
            mbar_wait_bounded(&full[i % L::kStages], static_cast<uint32_t>(i / L::kStages) & 1u, kErrWaitDrain);
          break;
        }
        mbar_arrive_expect_tx(&full[st], L::kStage);
#pragma unroll
        for (int w = 0; w < DC; ++w) {
          uint8_t* to = smem + st * L::kStage + w * L::kChunk;
          tma_load_4d(to, &map_k, &full[st], w * 64, hk, k_row + k0 + j * kStep, map_doc);
          tma_load_4d(to + DC * L::kChunk, &map_v, &full[st], w * 64, hk, k_row + k0 + j * kStep, map_doc);
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ 16 keys of each step
    float slope[MT][2];
    int lim[MT][2], place[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = t * 16 + g + 8 * e;
        m[t][e] = -INFINITY;
        lim[t][e] = r < rows ? min(limit_of((base + r) / group), k1) : 0;
        place[t][e] = (base + r) / group + shift;
        slope[t][e] = p.slopes != nullptr && r < rows ? p.slopes[hk * group + (base + r) % group] * kLog2e : 0.f;
      }
    const float scale = p.scale * kLog2e;
    const bool capped = p.cap > 0.f;
    const ScoreCap cap = capped ? score_cap(p.scale, p.cap) : ScoreCap{};
    // ldmatrix rows: lanes 8 i .. 8 i + 7 give the rows of matrix i. K: four 16-byte units of 8 keys; V: the
    // warp's keys 0-7 and 8-15 of one unit, then of the next; Q: rows 0-7 and 8-15 of one unit, then the next.
    const int mat = lane >> 3, in = lane & 7;
    const uint32_t ring = smem_u32(smem);
    const uint32_t k_lane = (warp * kKeys + in) * 128, v_lane = (warp * kKeys + (mat & 1) * 8 + in) * 128;
    const uint32_t q_lane = smem_u32(q_s) + (((mat & 1) * 8 + in) * L::kPitch + (mat >> 1) * 8) * 2;

    for (int j = 0; j < steps; ++j) {
      const int st = j % L::kStages, kb = k0 + j * kStep + warp * kKeys;
      if (!mbar_wait_warp(&full[st], static_cast<uint32_t>(j / L::kStages) & 1u, kErrWaitFull)) break;
      const uint32_t k_at = ring + st * L::kStage + k_lane, v_at = ring + st * L::kStage + DC * L::kChunk + v_lane;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float s[2][4] = {};
#pragma unroll
        for (int w = 0; w < DC * 2; ++w) {  // 32 channels: two product steps
          if (w * 32 >= p.dim) break;
          uint32_t a0[4], a1[4];
          ldmatrix4(a0, q_lane + (t * 16 * L::kPitch + w * 32) * 2);
          ldmatrix4(a1, q_lane + (t * 16 * L::kPitch + w * 32 + 16) * 2);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t b[4];
            ldmatrix4(b, k_at + (w >> 1) * L::kChunk + n * 8 * 128 + (((w & 1) * 4 + mat) ^ in) * 16);
            mma_16816<BF16>(s[n], a0, b[0], b[1]);
            mma_16816<BF16>(s[n], a1, b[2], b[3]);
          }
        }
        if (capped) cap_scores(reinterpret_cast<float(&)[8]>(s), cap);
        // Base-2 scores; s[n][2 e + i] belongs to row g + 8 e and key kb + 8 n + 2 c + i.
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = i >> 1, key = kb + n * 8 + 2 * c + (i & 1);
            float x = capped ? s[n][i] : s[n][i] * scale;
            x = fmaf(-slope[t][e], fabsf(static_cast<float>(place[t][e] - key)), x);
            x = key < lim[t][e] ? x : -INFINITY;
            s[n][i] = x;
            top[e] = fmaxf(top[e], x);
          }
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
          top[e] = fmaxf(top[e], m[t][e]);
          f[e] = m[t][e] == top[e] ? 1.f : exp2_unit(m[t][e] - top[e]);
          m[t][e] = top[e];
        }
        uint32_t a[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float from = m[t][e] == -INFINITY ? 0.f : m[t][e] - kLift;
            const float x0 = exp2_unit(s[n][2 * e] - from), x1 = exp2_unit(s[n][2 * e + 1] - from);
            l[t][e] = n == 0 ? fmaf(l[t][e], f[e], x0 + x1) : l[t][e] + (x0 + x1);
            a[n * 2 + e] = pack2<BF16>(x0, x1);
          }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < DC * 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][n][i] *= f[i >> 1];
        }
#pragma unroll
        for (int u = 0; u < DC * 8; u += 2) {  // 16 channels: two output tiles
          if (u * 8 >= p.dim) break;
          uint32_t b[4];
          ldmatrix4_trans(b, v_at + (u >> 3) * L::kChunk + (((u & 7) + (mat >> 1)) ^ in) * 16);
          if (kb + kKeys > k1) {  // keys that are not this document's or this CTA's: anything at all, so zeros
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = kb + (i & 1) * 8 + 2 * c;
              b[i] &= (key < k1 ? 0xffffu : 0u) | (key + 1 < k1 ? 0xffff0000u : 0u);
            }
          }
          mma_16816<BF16>(o[t][u], a, b[0], b[1]);
          mma_16816<BF16>(o[t][u + 1], a, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
  }

  // Each warp's sums to shared memory, where the ring was: every step has been read.
  __syncthreads();
  if (warp < kWarps) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 1);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 2);
        const int r = t * 16 + g + 8 * e;
        if (c == 0) {
          stat_s[(warp * L::kRows + r) * 2] = m[t][e];
          stat_s[(warp * L::kRows + r) * 2 + 1] = l[t][e];
        }
        float* to = o_s + (warp * L::kRows + r) * L::kD + 2 * c;
#pragma unroll
        for (int u = 0; u < DC * 8; ++u)
          *reinterpret_cast<float2*>(to + u * 8) = make_float2(o[t][u][2 * e], o[t][u][2 * e + 1]);
      }
  }
  __syncthreads();
  auto merge = [&](int r, int d, float& big, float& total) {  // relative to the largest m, 4 channels from d
    big = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) big = fmaxf(big, stat_s[(w * L::kRows + r) * 2]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const float from = big == -INFINITY ? 0.f : big;  // no maximum: nothing was seen, or NaN, which the sums hold
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_unit(stat_s[(w * L::kRows + r) * 2] - from);
      total = fmaf(f, stat_s[(w * L::kRows + r) * 2 + 1], total);
      const float4 v = *reinterpret_cast<const float4*>(o_s + (w * L::kRows + r) * L::kD + d);
      sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y);
      sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
    }
    return sum;
  };
  auto finish = [&](int r, int d, float4 sum, float big, float total) {
    const int i = (base + r) / group, h = hk * group + (base + r) % group;
    if (total == 0.f) sum = make_float4(0.f, 0.f, 0.f, 0.f);  // a query that saw nothing gets zeros
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint16_t* out = static_cast<uint16_t*>(p.out) + o_at + i * p.o_token + h * p.o_head;
    *reinterpret_cast<uint2*>(out + d) =
        make_uint2(pack2<BF16>(sum.x * inv, sum.y * inv), pack2<BF16>(sum.z * inv, sum.w * inv));
    if (p.lse != nullptr && d == 0)
      p.lse[(lse_at + i) * p.heads + h] = total == 0.f ? -INFINITY : (big + log2f(total * kDrop)) * 0.6931471805599453f;
  };
  const int quads = p.dim / 4, work = rows * quads;
  if (splits == 1) {
    for (int i = threadIdx.x; i < work; i += kThreads) {
      const int r = i / quads, d = (i - r * quads) * 4;
      float big, total;
      const float4 sum = merge(r, d, big, total);
      finish(r, d, sum, big, total);
    }
    return;
  }
  // The CTA's sums take the first warp's place: every thread merges into registers first.
  constexpr int kEach = (L::kRows * L::kD / 4 + kThreads - 1) / kThreads;
  float4 mine[kEach];
  float2 st[kEach];
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int i = threadIdx.x + n * kThreads;
    if (i < work) mine[n] = merge(i / quads, i % quads * 4, st[n].x, st[n].y);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int i = threadIdx.x + n * kThreads;
    if (i < work) {
      const int r = i / quads, d = i % quads * 4;
      *reinterpret_cast<float4*>(o_s + r * L::kD + d) = mine[n];
      if (d == 0) stat_s[r * 2] = st[n].x, stat_s[r * 2 + 1] = st[n].y;
    }
  }
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  for (int i = rank * kThreads + threadIdx.x; i < work; i += splits * kThreads) {
    const int r = i / quads, d = (i - r * quads) * 4;
    float big = -INFINITY, total = 0.f;
    for (int z = 0; z < splits; ++z) big = fmaxf(big, cluster.map_shared_rank(stat_s, z)[r * 2]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const float from = big == -INFINITY ? 0.f : big;
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
      const float2 other = *reinterpret_cast<const float2*>(cluster.map_shared_rank(stat_s, z) + r * 2);
      const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(o_s, z) + r * L::kD + d);
      const float f = exp2_unit(other.x - from);
      total = fmaf(f, other.y, total);
      sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y);
      sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
    }
    finish(r, d, sum, big, total);
  }
  cluster.sync();  // no CTA leaves while another reads its sums
}

template <int MT, int DC, bool BF16>
cudaError_t launch(const CUtensorMap& k, const CUtensorMap& v, const AttentionParams& p, int splits,
                   cudaStream_t stream) {
  auto kern = attention_few_kernel<MT, DC, BF16>;
  constexpr int bytes = static_cast<int>(FewSmem<MT, DC>::kBytes);
  static SharedMemoryGrant grant;
  const cudaError_t e = grant.ensure(kern, bytes, true);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  const int rows = p.heads / p.kv_heads * p.max_q;
  cfg.gridDim = dim3(static_cast<unsigned>(p.documents) * splits, static_cast<unsigned>(p.kv_heads),
                     static_cast<unsigned>((rows + MT * 16 - 1) / (MT * 16)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, k, v, p, splits);
}

template <bool BF16>
cudaError_t launch_type(const CUtensorMap& k, const CUtensorMap& v, const AttentionParams& p, int splits,
                        cudaStream_t stream) {
  const int rows = p.heads / p.kv_heads * p.max_q;
  if (p.dim <= 64)
    return rows <= 16 ? launch<1, 1, BF16>(k, v, p, splits, stream) : launch<2, 1, BF16>(k, v, p, splits, stream);
  return rows <= 16 ? launch<1, 2, BF16>(k, v, p, splits, stream) : launch<2, 2, BF16>(k, v, p, splits, stream);
}

}  // namespace

// How many CTAs share the keys of a unit (document, key head, group of rows): up to two CTAs for every SM, as
// long as each keeps two steps or more.
static int few_splits(long long units, int keys) {
  int splits = 1;
  while (splits < 16 && units * splits <= device_sm_count() && keys >= splits * 2 * 2 * kStep) splits *= 2;
  return splits;
}

// Whether this form takes the call: up to 128 rows of a key head, where the lesser of two estimates (microseconds,
// fitted to 1 to 32 requests of 5 to 128 queries over 256 to 16,000 keys). This one: 6 for 16 rows, 10 for more, and
// per step of 64 keys of a CTA 0.8 to 1.2 (head sizes to 64, above), 1.4 to 2.8. The tile kernel's CTAs take all
// keys of one head's queries: 3.5 a wave and 0.57 to 0.65 a step. (16 heads on 2 of
// 128: 5 queries of one request over 16,000 keys 43 us here and 170 there, 16 queries of 8 over 2,000 35 and 26.)
bool attention_few_takes(const AttentionParams& p) {
  const long long rows = static_cast<long long>(p.heads / p.kv_heads) * p.max_q;
  if (rows > 128 || p.documents > (1 << 24)) return false;
  const int keys = p.q_offsets != nullptr ? p.k_tokens / p.documents : p.k_tokens, sms = device_sm_count();
  const bool wide = p.dim > 64, many = rows > 16;
  const long long units = static_cast<long long>(p.documents) * p.kv_heads * ((rows + 31) / 32);
  const int splits = few_splits(units, keys);
  auto waves = [](long long n, long long at_once) { return static_cast<float>((n + at_once - 1) / at_once); };
  const float steps = static_cast<float>((keys + kStep - 1) / kStep);
  const float few = (many ? 10.f : 6.f) + waves(units * splits, 2 * sms) * steps / splits *
                                              (many ? (wide ? 2.8f : 1.4f) : (wide ? 1.2f : 0.8f));
  const float tiles = 3.f + waves(static_cast<long long>(p.documents) * p.heads, wide ? sms : 2 * sms) *
                                (3.5f + steps * (wide ? 0.65f : 0.57f));
  return few <= tiles;
}

cudaError_t launch_attention_few(const CUtensorMap& k, const CUtensorMap& v, const AttentionParams& p, bool bf16,
                                 cudaStream_t stream) {
  const int rows = p.heads / p.kv_heads * p.max_q;
  const int splits = few_splits(static_cast<long long>(p.documents) * p.kv_heads * ((rows + 31) / 32),
                                p.q_offsets != nullptr ? p.k_tokens / p.documents : p.k_tokens);
  return bf16 ? launch_type<true>(k, v, p, splits, stream) : launch_type<false>(k, v, p, splits, stream);
}

}  // namespace ctmr
