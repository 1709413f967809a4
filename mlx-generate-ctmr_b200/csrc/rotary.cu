// Rotary positions along several axes (depth, height, width of a latent grid, or any others): pair c of
// a head belongs to one axis, its angle is position[token][axis] * inv_freq[c], and
// (a, b) -> (a cos - b sin, b cos + a sin); the inverse takes the opposite angle. Channels past the
// pairs are copied. The pairs are (2c, 2c + 1), or (c, c + pairs).
//
// Angles: an fp32 position times an fp32 frequency is exact in 64 bits; it is turned into a fraction of
// a turn there (the only lossy step, 2^-53 relative) and sincospi takes that fraction in 32 bits. A
// product in 32 bits would be off by 2^-24 of the angle itself, i.e. by 6e-3 at a position of 1e5,
// more than the rounding of a 16-bit output.
//
// Bound by memory: x is read and y written once. A block takes a few tokens, computes their
// (cos, sin) table once in shared memory (the table serves every head: heads * pairs rotations for
// pairs sines) and then streams the heads past it, each thread one unit of up to 16 bytes (or one from
// each half) at a time; its first loads are on their way while the table is computed. 23,209 tokens of 24
// heads of 128 in bf16 (285 MB): 54 us, 5.3 TB/s, with six blocks an SM and six units a thread. More units
// in flight per thread cost blocks per SM and more time: two 64 us, four 95 us.
#include "launch.cuh"
#include "tokens.cuh"

namespace ctmr {
namespace {

constexpr int kThreads = 256, kBlocks = 6;  // six blocks an SM: 40 registers a thread

// V elements moved by one load or store of V * sizeof(T) bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// One unit of work of a token's head. HALVES: units [0, pairs / V) rotate V pairs (c, c + pairs), then
// the (dim - 2 pairs) / V others copy. Interleaved (V >= 2): dim / V units of V / 2 pairs, the table
// continued past the pairs by the identity. Interleaved with V = 1: units [0, pairs) are pairs moved
// element by element (for strides that allow no wider access), the others copy one element.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads, kBlocks) rotary_kernel(const RotaryParams p, int per_block, int units) {
  extern __shared__ __align__(16) float2 table[];  // [per_block][tab]
  griddep_wait();
  griddep_launch_dependents();
  const int tab = (!HALVES && V > 1) ? max(p.pairs, (p.dim + 1) / 2) : p.pairs;
  const long long t0 = static_cast<long long>(blockIdx.x) * per_block;
  const int n = static_cast<int>(min(static_cast<long long>(per_block), p.tokens - t0));

  using P = Vec<T, V>;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const int rotated = HALVES ? p.pairs / V : (V > 1 ? units : p.pairs);
  // Element offsets of a unit's first load and, where it has one, its second.
  auto first = [&](int u) {
    if (HALVES) return u < rotated ? u * V : 2 * p.pairs + (u - rotated) * V;
    return V > 1 ? u * V : (u < rotated ? 2 * u : 2 * p.pairs + (u - rotated));
  };
  const int second = HALVES ? p.pairs : 1;
  constexpr bool kTwo = HALVES || V == 1;
  // Unit i of the block is (token, head, unit of the head); a thread walks them kThreads apart, which is a
  // fixed step in each of the three with carries.
  const int per_token = p.heads * units;
  int t = threadIdx.x / per_token, u = threadIdx.x - t * per_token, h = u / units;
  u -= h * units;
  const int dt = kThreads / per_token, du0 = kThreads - dt * per_token, dh = du0 / units, du = du0 - dh * units;
  P a, b;
  auto load = [&]() {
    const T* in = x + (t0 + t) * p.x_token + h * p.x_head + first(u);
    a = *reinterpret_cast<const P*>(in);
    if (kTwo && u < rotated) b = *reinterpret_cast<const P*>(in + second);
  };
  if (t < n) load();  // on its way while the table is computed

  for (int i = threadIdx.x; i < n * tab; i += kThreads) {
    const int t = i / tab, c = i - t * tab;
    float2 cs = make_float2(1.f, 0.f);
    if (c < p.pairs) {
      int axis = 0;
      while (axis + 1 < p.axes && c >= p.section_end[axis]) ++axis;
      const long long at = (t0 + t) * p.pos_stride + axis;
      const double pos = p.positions_f32 ? static_cast<double>(static_cast<const float*>(p.positions)[at])
                                         : static_cast<double>(static_cast<const int*>(p.positions)[at]);
      constexpr double kInvTwoPi = 0.15915494309189533577;
      const double turns = pos * static_cast<double>(p.inv_freq[c]) * kInvTwoPi;
      const float f = static_cast<float>(turns - rint(turns));
      sincospif(2.f * f, &cs.y, &cs.x);
      if (p.inverse) cs.y = -cs.y;
    }
    table[i] = cs;
  }
  __syncthreads();

  while (t < n) {
    T* out = y + (t0 + t) * p.y_token + h * p.y_head + first(u);
    if (u < rotated) {
      if constexpr (kTwo) {
        const float2* cs = table + t * tab + u * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float p0 = to_float(a.e[e]), p1 = to_float(b.e[e]);
          a.e[e] = from_float<T>(p0 * cs[e].x - p1 * cs[e].y);
          b.e[e] = from_float<T>(p1 * cs[e].x + p0 * cs[e].y);
        }
        *reinterpret_cast<P*>(out + second) = b;
      } else {
        const float2* cs = table + t * tab + u * (V / 2);
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
          // Past the pairs the table holds the identity, but a copy must stay a copy for infinities too.
          if (u * V + e >= 2 * p.pairs) break;
          const float p0 = to_float(a.e[e]), p1 = to_float(a.e[e + 1]);
          a.e[e] = from_float<T>(p0 * cs[e / 2].x - p1 * cs[e / 2].y);
          a.e[e + 1] = from_float<T>(p1 * cs[e / 2].x + p0 * cs[e / 2].y);
        }
      }
    }
    *reinterpret_cast<P*>(out) = a;
    u += du;
    const int cu = u >= units;
    u -= cu ? units : 0, h += dh + cu;
    const int ch = h >= p.heads;
    h -= ch ? p.heads : 0, t += dt + ch;
    if (t < n) load();
  }
}

// The widest access, in elements, that every stride, both base addresses and (halves) the place of the
// second half allow.
int widest(const RotaryParams& p, int size, bool halves) {
  for (int v = 16 / size; v > 1; v /= 2) {
    const uintptr_t bytes = static_cast<uintptr_t>(v * size);
    bool ok = reinterpret_cast<uintptr_t>(p.x) % bytes == 0 && reinterpret_cast<uintptr_t>(p.y) % bytes == 0;
    ok = ok && p.dim % v == 0 && (!halves || p.pairs % v == 0);
    ok = ok && p.x_token % v == 0 && p.x_head % v == 0 && p.y_token % v == 0 && p.y_head % v == 0;
    if (ok) return v;
  }
  return 1;
}

template <typename T, int V>
cudaError_t launch(const RotaryParams& p, cudaStream_t stream) {
  const int units = p.interleaved ? (V > 1 ? p.dim / V : p.dim - p.pairs) : p.pairs / V + (p.dim - 2 * p.pairs) / V;
  const int tab = (p.interleaved && V > 1) ? (p.dim + 1) / 2 : p.pairs;
  // Six units a thread where the call is large enough to fill the GPU twice over, fewer otherwise;
  // the table stays within the 48 KB of shared memory that need no opt-in.
  long long per = (6LL * kThreads + p.heads * units - 1) / (static_cast<long long>(p.heads) * units);
  per = per < 1 ? 1 : (per > 32 ? 32 : per);
  const long long spread = p.tokens / (2LL * device_sm_count());
  if (per > spread) per = spread < 1 ? 1 : spread;
  const long long room = 49152 / (static_cast<long long>(sizeof(float2)) * (tab < 1 ? 1 : tab));
  if (per > room) per = room;
  const long long blocks = (p.tokens + per - 1) / per;
  if (per < 1 || blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  auto kern = p.interleaved ? rotary_kernel<T, V, false> : rotary_kernel<T, V, true>;
  return launch_kernel(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), per * tab * sizeof(float2), stream, p,
                       static_cast<int>(per), units);
}

template <typename T>
cudaError_t launch_type(const RotaryParams& p, cudaStream_t stream) {
  switch (widest(p, sizeof(T), !p.interleaved)) {
    case 8: if constexpr (sizeof(T) == 2) return launch<T, 8>(p, stream); [[fallthrough]];
    case 4: return launch<T, 4>(p, stream);
    case 2: return launch<T, 2>(p, stream);
    default: return launch<T, 1>(p, stream);
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream) {
  if (dtype == 0) return launch_type<float>(p, stream);
  return dtype == 1 ? launch_type<__nv_bfloat16>(p, stream) : launch_type<__half>(p, stream);
}

}  // namespace ctmr
