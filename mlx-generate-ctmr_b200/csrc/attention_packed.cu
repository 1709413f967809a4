// Attention over packed documents: softmax over the keys of a query's own document, with causal and
// prefix masks, capped scores and a bias that falls with distance, grouped heads.
//   s_ij = cap(scale q_i . k_j) - slope_h |p_i - j|,  p_i = i + Lk - Lq,  cap(x) = c tanh(x / c)
// Every mask leaves a query the keys [0, lim_i): lim_i = Lk, or min(Lk, max(p_i + 1, prefix)) when causal.
//
// Queries come in tiles of 128 of a document and head. Head sizes up to 64: a CTA takes one tile and two CTAs
// share an SM; above: a CTA takes two tiles, which share its K and V in shared memory. A query has two
// softmax threads of 32 keys a step each (with one thread of 64 keys the schedulers had two warps to choose
// from and issued in 47 % of the clocks). Keys come in steps of 64: S = Q K^T (128 x 64 fp32)
// lands in TMEM, a thread reads its half row into registers, turns it into base-2 scores, takes the maximum,
// exchanges it with the other half's through shared memory, and writes P = 2^(s - m) as 16-bit pairs over S's
// own columns, and the tensor core reads P from TMEM for O += P V (V is MN-major in shared memory, as
// loaded). Each tile has two S buffers, S(j + 1) is ready while the threads work on S(j), and a warp for each
// tile issues
//   S(0) S(1) | PV(0) S(2) | PV(1) S(3) | ...
// O stays in TMEM; it is
// rescaled (by the softmax threads, which hold m) only where a row's maximum has grown by more than 2^8
// since the last time: until then P may exceed one, up to 2^8 (2^15 as it is held), which neither 16-bit type
// minds, and the sum of P is kept in fp32 with the same m.
//
// With a distance bias the steps are visited from the queries' own place outwards, first towards the first
// key, then towards the last: in order of keys the maximum grew with every step that came nearer, and the
// tiles at the end of 8,192 tokens took 205 us where those at the start took 131.
#include <cmath>

#include "capi_internal.cuh"
#include "ctmr_b200.h"
#include "launch.cuh"
#include "softmax.cuh"

namespace ctmr {
namespace {

constexpr int kTile = 128;     // queries per tile
constexpr int kStep = 64;      // keys per step
constexpr int kPart = 32;      // of them per softmax thread
constexpr uint32_t kQChunk = kTile * 128, kKChunk = kStep * 128;  // rows of 64 16-bit channels
constexpr float kRescale = 8.f;  // log2 of the growth that O and the sum are rescaled for
// P and its sum are held 2^7 larger: fp16 rounds numbers below 2^-14 ever more coarsely (weights of 2^-20 to one
// part in 32), and 2^(8 + 7) is the most that it holds.
constexpr float kLift = 7.f, kDrop = 1.f / 128.f;

// NC chunks of 64 channels per row (two above 64 channels), as many query tiles. V in a ring of four steps, K,
// which runs two steps ahead, in one of five: K(j + 2) takes the place of K(j - 3), V(j) of V(j - 4); both are
// read when step j - 3 is done.
template <int NC>
struct Layout {
  static constexpr int kTiles = NC, kBlock = kTiles * kTile;
  // Softmax warps by tile, half of the keys and quarter of the queries; then TMA; then each tile's products.
  static constexpr int kTmaWarp = 8 * kTiles, kThreads = (kTmaWarp + 1 + kTiles) * 32;
  static constexpr int kCtas = NC == 1 ? 2 : 1;              // per SM
  static constexpr uint32_t kTmem = 256 * kTiles, kTmemO = 128 * kTiles;  // S of each tile, then O of each
  static constexpr int kStages = 4, kKSlots = 5;
  static constexpr uint32_t kQBytes = NC * kQChunk, kKBytes = NC * kKChunk;
  static constexpr uint32_t kOffK = kTiles * kQBytes;
  static constexpr uint32_t kOffV = kOffK + kKSlots * kKBytes;
  static constexpr uint32_t kOffBar = kOffV + kStages * kKBytes;
  static constexpr uint32_t kOffMax = kOffBar + 256;  // [step parity][tile][half][query] maxima
  static constexpr uint32_t kBytes = kOffMax + 2048 * kTiles + 1024;  // + alignment slack
  static_assert(kCtas * (kBytes + 1024) <= 228 * 1024, "shared memory of an SM");
};

struct Maps {
  CUtensorMap q, k, v;
};

// The larger, NaN if either is: a NaN score must not become a weight of zero (the integer addition below makes it the
// largest number, which is infinity to the product).
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// 2^x of a pair, x <= 15, on the FMA pipe: x = n + f with n the nearest integer (the low bits of x plus
// 1.5 * 2^23) and |f| <= 1/2, 2^f by a quartic (least maximum relative error on that interval, 2.6e-6, mean
// error 4e-8: far below P's rounding, and small enough for the log-sum-exp, whose sum it enters; a cubic's
// 7.5e-5 would show there), n added to the exponent. Zero below 2^-127, where that leaves no positive bits: a clamp
// at 2^-125 gave masked keys that weight, and with values near bf16's lowest a share of the output.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = max_or_nan(x.x, -250.f), x.y = max_or_nan(x.y, -250.f);  // (n fits the nine bits above the mantissa)
  const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
  const float2 j = add2(x, magic), n = add2(j, back);
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 p = fma2(make_float2(0.009567703887021797f, 0.009567703887021797f), f,
                  make_float2(0.05591834983019358f, 0.05591834983019358f));
  p = fma2(p, f, make_float2(0.24024836877206313f, 0.24024836877206313f));
  p = fma2(p, f, make_float2(0.6931217761894134f, 0.6931217761894134f));
  p = fma2(p, f, make_float2(0.9999991951706715f, 0.9999991951706715f));
  p.x = __int_as_float(__viaddmax_s32(__float_as_int(p.x), __float_as_int(j.x) << 23, 0));
  p.y = __int_as_float(__viaddmax_s32(__float_as_int(p.y), __float_as_int(j.y) << 23, 0));
  return p;
}

// The document and rows of one CTA.
struct Place {
  int doc, q_row, k_row;  // rows of the TMA maps where the document's queries and keys start
  int map_doc;            // document coordinate of the maps
  int q_len, k_len, first;  // first: the CTA's first query inside the document
  int prefix;
  long long row0;         // the document's first row of lse
};

// Keys [0, lim) that query i of the document sees.
__device__ __forceinline__ int limit_of(const AttentionParams& p, const Place& w, int i) {
  if (!p.causal) return w.k_len;
  return min(w.k_len, max(max(i + w.k_len - w.q_len + 1, w.prefix), 0));
}

// Up to 32 documents: their tiles in order of falling key counts, each document's heads together, so that no
// long one starts when the others are done (seven volumes of 105 to 2,048 tokens, 8 heads of 32: 61 us in order
// of documents, 55 us so; four causal ones of 1 to 2,300 tokens, 16 heads of 128: 101 and 83 us). More documents
// than a warp has lanes keep their order (four of 2,048 tokens and 28 of 64, and the same with an empty one more: 65
// and 80 us with 8 heads of 32, 152 and 171 with 16 of 128). By a whole warp; false where `id` is past the last tile.
template <int kBlock>
__device__ __forceinline__ bool longest_first(const AttentionParams& p, int id, int lane, int& doc, int& head,
                                              int& tile) {
  int tiles = 0, keys = -1;
  if (lane < p.documents) {
    const int qb = min(max(p.q_offsets[lane], 0), p.q_tokens), qe = min(max(p.q_offsets[lane + 1], qb), p.q_tokens);
    tiles = (qe - qb + kBlock - 1) / kBlock;
    keys = max(p.k_offsets[lane + 1] - p.k_offsets[lane], 0);
  }
  int before = 0;
  for (int d = 0; d < p.documents; ++d) {
    const int other = __shfl_sync(0xffffffffu, keys, d), n = __shfl_sync(0xffffffffu, tiles, d);
    if (other > keys || (other == keys && d < lane)) before += n;
  }
  const int start = before * p.heads, in = id - start;
  const unsigned mine = __ballot_sync(0xffffffffu, in >= 0 && in < tiles * p.heads);
  if (mine == 0) return false;
  doc = __ffs(mine) - 1;
  const int n = __shfl_sync(0xffffffffu, tiles, doc), at = __shfl_sync(0xffffffffu, in, doc);
  head = at / n, tile = at - head * n;
  return true;
}

template <int kBlock>
__device__ __forceinline__ bool find_place(const AttentionParams& p, int id, int lane, Place& w, int& head) {
  int tile;
  if (p.q_offsets != nullptr) {
    if (p.documents <= 32) {
      if (!longest_first<kBlock>(p, id, lane, w.doc, head, tile)) return false;
    } else {
      const int per = p.q_tokens / kBlock + p.documents;
      head = id / per, id -= head * per;
      w.doc = segment_of_tile(p.q_offsets, p.documents, kBlock, id, lane);
      tile = id - (max(p.q_offsets[w.doc], 0) / kBlock + w.doc);
    }
    int qe, ke;
    segment_range(p.q_offsets, w.doc, p.q_tokens, w.q_row, qe);
    segment_range(p.k_offsets, w.doc, p.k_tokens, w.k_row, ke);
    w.q_len = qe - w.q_row, w.k_len = ke - w.k_row;
    w.map_doc = 0;
    w.row0 = w.q_row;
  } else {
    const int per = (p.q_tokens + kBlock - 1) / kBlock;
    head = id / per % p.heads, w.doc = id / (per * p.heads), tile = id % per;
    w.q_row = w.k_row = 0, w.map_doc = w.doc, w.q_len = p.q_tokens, w.k_len = p.k_tokens;
    if (p.k_lengths != nullptr) {
      const int n = p.k_lengths[w.doc];
      w.k_len = min(max(n, 0), p.k_tokens);
      if (n != w.k_len) flag_error(kErrBadOffsets);
    }
    w.row0 = static_cast<long long>(w.doc) * p.q_tokens;
  }
  if (w.q_len > p.max_q) flag_error(kErrBadOffsets);
  const int tiles = (w.q_len + kBlock - 1) / kBlock;
  if (tile < 0 || tile >= tiles) return false;
  // Later queries see more keys: the longest tiles of a causal document start first.
  w.first = (p.causal ? tiles - 1 - tile : tile) * kBlock;
  w.prefix = p.prefix != nullptr ? p.prefix[w.doc] : 0;
  return true;
}

template <int NC, bool CAP, bool BIAS, bool BF16>
__global__ void __launch_bounds__(Layout<NC>::kThreads, Layout<NC>::kCtas)
    attention_tile_kernel(const __grid_constant__ Maps maps, const AttentionParams p) {
  using L = Layout<NC>;
  constexpr int kTiles = L::kTiles, kTmaWarp = L::kTmaWarp;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_full = bar;                  // [2]
  // [tile][buffer]: S(j) is done, and with it PV(j - 2); both also for the two steps after the last.
  uint64_t* s_full = bar + 2;
  uint64_t* p_full = bar + 6;              // [tile][buffer]: P(j) is written, S(j) read
  uint64_t* k_first = bar + 10;            // [2] K(0), K(1)
  uint64_t* full = bar + 12;               // [kStages] V(j) and K(j + 2)
  uint64_t* empty = full + L::kStages;     // [kStages] both read by both tiles
  uint64_t* v_fixed = empty + L::kStages;  // the last V step has zeros past the document
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_fixed + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  Place w;
  int h;
  if (p.q_offsets != nullptr && blockIdx.x == gridDim.x - 1) {  // one block more than the tiles may need
    report_offsets(p.q_offsets, p.documents, p.q_tokens);
    report_offsets(p.k_offsets, p.documents, p.k_tokens);
    if (warp == 0) clear_outside(p, blockIdx.x, gridDim.x, lane);
    return;
  }
  if (!find_place<L::kBlock>(p, blockIdx.x, lane, w, h)) {  // the same answer in every warp
    if (p.q_offsets != nullptr && warp == 0) clear_outside(p, blockIdx.x, gridDim.x, lane);
    return;
  }
  const int hk = h / (p.heads / p.kv_heads);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&k_first[i], 1);
    }
    for (int i = 0; i < 2 * kTiles; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 2 * kTile);
    }
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kTiles);
    }
    mbar_init(v_fixed, 1);
    fence_barrier_init();
  }
  if (warp == kTmaWarp + 1) {
    tmem_alloc(tmem_slot, L::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Dependents are released once this block holds its columns: one that allocates ahead of its own wait could take
  // them otherwise. (A block without a tile releases them by its end.)
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;  // tile t: S at columns 128 t and 128 t + 64 (P over them), O at kTmemO + 128 t

  // Steps of each query tile: the keys that its last query sees. (With a bias all take the longest's, and
  // find the rest masked: the order below starts at the far end of it.)
  auto steps_of = [&](int t) {
    const int last = min(w.q_len - 1, w.first + (t + 1) * kTile - 1);
    return last < w.first + t * kTile ? 0 : (limit_of(p, w, last) + kStep - 1) / kStep;
  };
  int n0 = steps_of(0), n1 = kTiles == 2 ? steps_of(1) : 0;
  const int n_max = max(n0, n1);
  if (BIAS) n0 = n_max, n1 = n1 > 0 ? n_max : 0;
  // The step of keys that is visited as the j-th.
  const int own = (w.first + min(L::kBlock, w.q_len - w.first) / 2 + w.k_len - w.q_len) / kStep;
  const int centre = BIAS ? min(max(own, 0), max(n_max - 1, 0)) : 0;
  auto step_at = [&](int j) { return !BIAS || j > centre ? j : centre - j; };
  // The document's keys in its last step, if fewer than 64, and when that is visited.
  const int tail = w.k_len - (n_max - 1) * kStep, tail_at = BIAS && centre == n_max - 1 ? 0 : n_max - 1;

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ TMA producer: lane 0 issues
    if (n_max > 0) {
      if (lane == 0) {
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        for (int t = 0; t < kTiles; ++t) {
          if ((t == 0 ? n0 : n1) == 0) continue;
          mbar_arrive_expect_tx(&q_full[t], L::kQBytes);
#pragma unroll
          for (int c = 0; c < NC; ++c)
            tma_load_4d(smem + t * L::kQBytes + c * kQChunk, &maps.q, &q_full[t], c * 64, h,
                        w.q_row + w.first + t * kTile, w.map_doc);
        }
      }
      auto load = [&](const CUtensorMap* map, uint32_t off, uint64_t* bar, int j) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          tma_load_4d(smem + off + c * kKChunk, map, bar, c * 64, hk, w.k_row + step_at(j) * kStep, w.map_doc);
      };
      const int firsts = min(n_max, 2);
      if (lane == 0)
        for (int j = 0; j < firsts; ++j) {
          mbar_arrive_expect_tx(&k_first[j], L::kKBytes);
          load(&maps.k, L::kOffK + j * L::kKBytes, &k_first[j], j);
        }
      __syncwarp();
      int j = 0;
      for (; j < n_max; ++j) {
        const int s = j % L::kStages, done = j - 3;
        if (done >= 0 && !mbar_wait_warp(&empty[done % L::kStages], static_cast<uint32_t>(done / L::kStages) & 1u,
                                         kErrWaitEmpty))
          break;
        if (lane == 0) {
          const bool more = j + 2 < n_max;
          mbar_arrive_expect_tx(&full[s], more ? 2 * L::kKBytes : L::kKBytes);
          load(&maps.v, L::kOffV + s * L::kKBytes, &full[s], j);
          if (more) load(&maps.k, L::kOffK + (j + 2) % L::kKSlots * L::kKBytes, &full[s], j + 2);
        }
        __syncwarp();
        if (j == tail_at && tail < kStep) {
          // Rows past the document hold another's values, whose product with P = 0 must still be 0.
          if (!mbar_wait_warp(&full[s], static_cast<uint32_t>(j / L::kStages) & 1u, kErrWaitFull)) {
            ++j;
            break;
          }
          uint8_t* vt = smem + L::kOffV + s * L::kKBytes;
          for (int i = lane; i < (kStep - tail) * 8; i += 32)
#pragma unroll
            for (int c = 0; c < NC; ++c)
              *reinterpret_cast<uint4*>(vt + c * kKChunk + tail * 128 + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(v_fixed);
        }
      }
      if (lane == 0) {
        // Drain: every issued load lands before the CTA can exit.
        if (n0 > 0) mbar_wait_bounded(&q_full[0], 0, kErrWaitDrain);
        if (n1 > 0) mbar_wait_bounded(&q_full[1], 0, kErrWaitDrain);
        for (int i = 0; i < firsts; ++i) mbar_wait_bounded(&k_first[i], 0, kErrWaitDrain);
        for (int i = max(0, j - L::kStages); i < j; ++i)
          mbar_wait_bounded(&full[i % L::kStages], static_cast<uint32_t>(i / L::kStages) & 1u, kErrWaitDrain);
      }
      __syncwarp();
    }
  } else if (warp > kTmaWarp) {
    // ------------------------------------------------------------ MMA issuer of tile t: a warp that stays together
    const int t = warp - kTmaWarp - 1;
    // (While the first loads are on their way: ahead of the tile's own work it took 1 us of 54.)
    if (t == kTiles - 1 && p.q_offsets != nullptr) clear_outside(p, blockIdx.x, gridDim.x, lane);
    __syncwarp();
    const int dk = warp_value((p.dim + 15) / 16), n = warp_value(t == 0 ? n0 : n1), last = warp_value(n_max);
    const int fix_at = warp_value(tail < kStep ? tail_at : -1);
    const uint32_t tm_s = warp_value(tmem + t * 128), tm_o = tm_s + L::kTmemO;
    const uint32_t base = warp_value(smem_u32(smem));
    const uint32_t id_s = idesc_f16(BF16, kTile, kStep);
    const uint32_t id_o = idesc_f16(BF16, kTile, static_cast<uint32_t>(dk) * 16u) | (1u << 16);  // V MN-major
    const uint64_t d_q = smem_desc_kmajor(base + t * L::kQBytes, 128);
    const uint64_t d_k = smem_desc_kmajor(base + L::kOffK, 128);
    const uint64_t d_v = smem_desc_mnmajor(base + L::kOffV, kKChunk);
    bool ok = true;
    // S(j). The last chunk of channels may have fewer than four products: those are a loop.
    auto issue_s = [&](int j) {
      const uint64_t b = desc_advance(d_k, static_cast<uint32_t>(j % L::kKSlots) * L::kKBytes);
      const uint32_t d = tm_s + (j & 1) * 64;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int steps = dk - c * 4;
        const uint64_t ac = desc_advance(d_q, c * kQChunk), bc = desc_advance(b, c * kKChunk);
        if (steps >= 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(d, desc_advance(ac, k * 32u), desc_advance(bc, k * 32u), id_s, c > 0 || k > 0 ? 1u : 0u);
        } else {
#pragma unroll 1
          for (int k = 0; k < steps; ++k)
            umma_f16(d, desc_advance(ac, k * 32u), desc_advance(bc, k * 32u), id_s, c > 0 || k > 0 ? 1u : 0u);
        }
      }
    };
    if (n > 0) ok = mbar_wait_warp(&q_full[t], 0, kErrWaitFull);
    for (int j = 0; ok && j < 2 && j < n; ++j) {
      ok = mbar_wait_warp(&k_first[j], 0, kErrWaitFull);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        issue_s(j);
        umma_commit(&s_full[t * 2 + j]);
      }
      __syncwarp();
    }
    for (int j = 0; ok && j < n; ++j) {
      const int s = j % L::kStages;
      // One lane to a barrier: V(j) with K(j + 2), P(j), and where there are any V's zeros.
      bool got = true;
      if (lane == 0) got = mbar_wait_bounded(&full[s], static_cast<uint32_t>(j / L::kStages) & 1u, kErrWaitFull);
      if (lane == 1)
        got = mbar_wait_bounded(&p_full[t * 2 + (j & 1)], static_cast<uint32_t>(j >> 1) & 1u, kErrWaitFull);
      if (lane == 2 && j == fix_at) got = mbar_wait_bounded(v_fixed, 0, kErrWaitFull);
      ok = __all_sync(0xffffffffu, got);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t b = desc_advance(d_v, static_cast<uint32_t>(s) * L::kKBytes);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          umma_f16_ts(tm_o, tm_s + (j & 1) * 64 + k * 8, desc_advance(b, k * 2048u), id_o, j > 0 || k > 0 ? 1u : 0u);
        if (j + 2 < n) issue_s(j + 2);
        umma_commit(&s_full[t * 2 + (j & 1)]);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    // The other tile may see more keys: this one frees their stages as they come.
    for (int j = n; ok && j < last; ++j) {
      ok = mbar_wait_warp(&full[j % L::kStages], static_cast<uint32_t>(j / L::kStages) & 1u, kErrWaitFull);
      if (ok && lane == 0) mbar_arrive(&empty[j % L::kStages]);
      __syncwarp();
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax, two threads per query
    const int t = warp >> 3, half = (warp >> 2) & 1;
    const int row = (warp & 3) * 32 + lane, i = w.first + t * kTile + row;  // the query inside the document
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + L::kTmemO + t * 128;
    const int n = t == 0 ? n0 : n1;
    constexpr int kParity = kTiles * 2 * kTile;
    float* maxima = reinterpret_cast<float*>(smem + L::kOffMax) + t * 2 * kTile + row;  // + parity, + half * 128
    const int pair_bar = 1 + t * 4 + (warp & 3);  // the two warps of these queries
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
    bool ok = true;
    auto wait_s = [&](int j) {  // (after a failure without waiting: the other half meets here)
      // By the whole warp: tcgen05.ld wants its lanes together, and each would leave a wait by itself. (One try ahead
      // of the loop, 8,192 tokens of 8 heads of 32, and of 128 causal: 222 and 171 us; the loop alone: 225 and 184.)
      uint64_t* bar = &s_full[t * 2 + (j & 1)];
      const uint32_t parity = static_cast<uint32_t>(j >> 1) & 1u;
      if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) ok = ok && mbar_wait_warp(bar, parity, kErrWaitAcc);
      tc_fence_after();
    };
    const int lim = limit_of(p, w, i) - half * kPart, place = i + w.k_len - w.q_len - half * kPart;
    const float scale = p.scale * kLog2e;
    const ScoreCap cap = CAP ? score_cap(p.scale, p.cap) : ScoreCap{};
    const float slope = BIAS ? p.slopes[h] * kLog2e : 0.f;
    const float unit = CAP || BIAS ? 1.f : scale;  // what turns s below into base-2 scores
    float m = -INFINITY, l = 0.f;  // m: what P is relative to; the maximum or up to 2^8 below; l: of this half
    for (int j = 0; j < n; ++j) {
      wait_s(j);
      const uint32_t t_s = tmem + lanes + t * 128 + (j & 1) * 64;
      const int key0 = step_at(j) * kStep;
      float s[kPart];
      tmem_ld32(t_s + half * kPart, s);
      tmem_ld_wait();
      tmem_ld_fence(s);
      if constexpr (CAP) cap_scores(s, cap);
      if constexpr (BIAS) {
        // s - slope |at - c|: away from the query's own place the distance is linear in c.
        const int at = place - key0;
        const float mul = CAP ? 1.f : scale;
        if (__all_sync(0xffffffffu, at >= kPart - 1 || at <= 0)) {
          const float step = at > 0 ? slope : -slope, from = -step * static_cast<float>(at);
#pragma unroll
          for (int c = 0; c < kPart; ++c) s[c] = fmaf(s[c], mul, fmaf(static_cast<float>(c), step, from));
        } else {
#pragma unroll
          for (int c = 0; c < kPart; ++c) s[c] = fmaf(-slope, fabsf(static_cast<float>(at - c)), s[c] * mul);
        }
      }
      const int left = lim - key0;
      if (left < kPart) {
#pragma unroll
        for (int c = 0; c < kPart; ++c) s[c] = c < left ? s[c] : -INFINITY;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) mx[c] = s[c];
#pragma unroll
      for (int c = 4; c < kPart; ++c) mx[c & 3] = fmaxf(mx[c & 3], s[c]);
      const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // The halves meet: the maximum of both, and P may take the place of S, which both have read.
      maxima[(j & 1) * kParity + half * kTile] = mine;
      meet();
      const float top = unit * fmaxf(mine, maxima[(j & 1) * kParity + (half ^ 1) * kTile]);
      const bool grow = top > m + kRescale || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? exp2_unit(m - top) : 1.f;
        if (grow) m = top;
        l *= f;
        if (j > 0) {  // PV(j - 1) has to be done; nothing writes O then until P(j) is handed over
          wait_s(j + 1);
          for (int c = half * 32; c < p.dim; c += 64) {
            float o[32];
            tmem_ld32(t_o + c, o);
            tmem_ld_wait();
            tmem_ld_fence(o);
            uint32_t r[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(o[e] * f);
            tmem_st32(t_o + c, r);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : kLift - m;
      const float2 u2 = make_float2(unit, unit), b2 = make_float2(base, base);
      float2 sum[2] = {};
      uint32_t r[kPart / 2];
#pragma unroll
      for (int e = 0; e < kPart / 2; ++e) {
        float2 x = fma2(make_float2(s[2 * e], s[2 * e + 1]), u2, b2);
        // One pair in four on the FMA pipe, the others on the exponential unit (16 a clock per SM,
        // half of the time of a step's two products at head size 128 and more below it).
        if ((e & 3) == 3) x = exp2_poly(x);
        else x = make_float2(exp2_unit(x.x), exp2_unit(x.y));
        sum[e & 1] = add2(sum[e & 1], x);
        r[e] = pack2<BF16>(x.x, x.y);
      }
      tmem_st16(t_s + half * (kPart / 2), r);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t * 2 + (j & 1)]);
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
    }
    if (n > 0) {
      wait_s(n + 1);  // PV(n - 1)
      maxima[(n & 1) * kParity + half * kTile] = l;
      meet();
      l += maxima[(n & 1) * kParity + (half ^ 1) * kTile];
    }
    // A query that saw nothing gets zeros; one whose scores are NaN has no maximum either, but NaN for a sum.
    const bool some = m != -INFINITY || l != l;
    const float inv = some ? 1.f / l : 0.f;
    uint16_t* out = static_cast<uint16_t*>(p.out) + w.map_doc * p.o_doc + (w.q_row + i) * p.o_token + h * p.o_head;
    for (int c = half * 32; c < p.dim; c += 64) {
      float o[32];
      if (n > 0) {
        tmem_ld32(t_o + c, o);
        tmem_ld_wait();
        tmem_ld_fence(o);
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        if (c + e >= p.dim || i >= w.q_len) break;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (some)
          v = make_uint4(pack2<BF16>(o[e] * inv, o[e + 1] * inv), pack2<BF16>(o[e + 2] * inv, o[e + 3] * inv),
                         pack2<BF16>(o[e + 4] * inv, o[e + 5] * inv), pack2<BF16>(o[e + 6] * inv, o[e + 7] * inv));
        *reinterpret_cast<uint4*>(out + c + e) = v;
      }
    }
    if (p.lse != nullptr && half == 0 && i < w.q_len)
      p.lse[(w.row0 + i) * p.heads + h] = some ? (m + log2f(l * kDrop)) * 0.6931471805599453f : -INFINITY;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kTmaWarp + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmem);
  }
}

template <int NC, bool CAP, bool BIAS, bool BF16>
cudaError_t launch_tiles(const Maps& maps, const AttentionParams& p, dim3 grid, cudaStream_t stream) {
  auto kern = attention_tile_kernel<NC, CAP, BIAS, BF16>;
  constexpr int bytes = static_cast<int>(Layout<NC>::kBytes);
  static SharedMemoryGrant grant;
  const cudaError_t e = grant.ensure(kern, bytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kern, grid, dim3(Layout<NC>::kThreads), bytes, stream, maps, p);
}

template <int NC, bool BF16>
cudaError_t launch_variant(const Maps& maps, const AttentionParams& p, dim3 grid, cudaStream_t stream) {
  if (p.cap > 0.f)
    return p.slopes != nullptr ? launch_tiles<NC, true, true, BF16>(maps, p, grid, stream)
                               : launch_tiles<NC, true, false, BF16>(maps, p, grid, stream);
  return p.slopes != nullptr ? launch_tiles<NC, false, true, BF16>(maps, p, grid, stream)
                             : launch_tiles<NC, false, false, BF16>(maps, p, grid, stream);
}

}  // namespace

// (channel, head, token, document) view of one operand, a box of 64 channels x box_tokens tokens.
int encode_tokens_map(CUtensorMap* map, const void* base, bool bf16, int dim, int heads, long long tokens,
                      long long docs, long long s_head, long long s_token, long long s_doc, int box_tokens,
                      const char* what) {
  auto enc = api_tensor_map_encoder();
  if (enc == nullptr) return api_fail(CTMR_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(docs)};
  // A stride that addresses nothing (an extent of one) may be anything the encoder takes.
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(heads > 1 ? s_head * 2 : 16),
                                 static_cast<cuuint64_t>(tokens > 1 ? s_token * 2 : 16),
                                 static_cast<cuuint64_t>(docs > 1 ? s_doc * 2 : 16)};
  const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(box_tokens), 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return api_fail(CTMR_ERR_INVALID, "%s's strides cannot be read by TMA (CUresult %d)", what, int(r));
  return CTMR_OK;
}

int launch_attention_packed(const AttentionParams& p, bool bf16, cudaStream_t stream) {
  const bool packed = p.q_offsets != nullptr;
  const int docs = packed ? 1 : p.documents;
  Maps maps{};
  int st = CTMR_OK;
  const bool few = attention_few_takes(p);
  if (!few)
    st = encode_tokens_map(&maps.q, p.q, bf16, p.dim, p.heads, p.q_tokens, docs, p.q_head, p.q_token, p.q_doc, kTile,
                           "q");
  if (st == CTMR_OK && p.k_tokens > 0)  // not read where there are no keys
    st = encode_tokens_map(&maps.k, p.k, bf16, p.dim, p.kv_heads, p.k_tokens, docs, p.k_head, p.k_token, p.k_doc, kStep,
                           "k");
  if (st == CTMR_OK && p.k_tokens > 0)
    st = encode_tokens_map(&maps.v, p.v, bf16, p.dim, p.kv_heads, p.k_tokens, docs, p.v_head, p.v_token, p.v_doc, kStep,
                           "v");
  if (st != CTMR_OK) return st;
  cudaError_t e;
  if (few) {
    e = launch_attention_few(maps.k, maps.v, p, bf16, stream);
  } else {
    const int block = p.dim <= 64 ? Layout<1>::kBlock : Layout<2>::kBlock;
    const long long tiles = packed ? p.q_tokens / block + static_cast<long long>(p.documents)
                                   : static_cast<long long>(p.documents) * ((p.q_tokens + block - 1) / block);
    if (tiles * p.heads >= 0x7fffffffLL) return api_fail(CTMR_ERR_UNSUPPORTED, "too many documents and heads");
    const dim3 grid(static_cast<unsigned>(tiles * p.heads + packed));
    if (p.dim <= 64)
      e = bf16 ? launch_variant<1, true>(maps, p, grid, stream) : launch_variant<1, false>(maps, p, grid, stream);
    else
      e = bf16 ? launch_variant<2, true>(maps, p, grid, stream) : launch_variant<2, false>(maps, p, grid, stream);
  }
  return e == cudaSuccess ? CTMR_OK : api_fail(CTMR_ERR_CUDA, "attention launch: %s", cudaGetErrorString(e));
}

}  // namespace ctmr
