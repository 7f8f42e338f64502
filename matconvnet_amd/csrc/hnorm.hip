// The heads of queries and keys, each divided by the root of its mean square, scaled per channel, and turned pair by pair by angles made of
// its position.
//   sigma = sqrt(mean_d x^2 + epsilon), xh = x/sigma, u = g xh;  angle_j = sum_a position[n][a] frequency[a][j]
//   (y_lo, y_hi) = (u_lo cos - u_hi sin, u_hi cos + u_lo sin) for the two channels of pair j; channels of no pair stay u
//   backward: du = the pairs of dzdy turned back, dzdg = sum over positions and heads of du xh, a = g du,
//             dzdx = (a - xh mean_d(a xh))/sigma
// Bound by memory: a head's channels stay in the registers of T lanes between the sum of squares and the output.  A wavefront takes
// the heads of one position, so that the angles of a position are made once: lane by lane one pair each, the cosines and sines
// then pass through local memory to the lanes that hold the pair in each head.  Angles are products and sums of doubles, brought to a
// revolution in double, which the sine takes in two parts: position 10^6 times frequency 1 keeps all of a single-precision sine.
//
// A lane holds VP pairs, 2 VP channels: the pairs' first channels and their second ones a run of pairs apart, or neighbours.  Channels of
// no pair are held likewise and not turned.  Heads of any size and address are read four values at a time from wherever they start, what is
// left over value by value.
#include "mcn_internal.hpp"

#include <algorithm>

namespace mcn {
namespace {

typedef unsigned short bf16;
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
template <class V> __device__ __forceinline__ V from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __builtin_bit_cast(bf16, (__bf16)v); }
template <class V, int N> struct alignas(sizeof(V) * N) Pack { V v[N]; };

constexpr int kMostD = 512, kWaves = 4;

struct HeadsP {        // one of the two sets
  const void *x, *dy;  // (dy: backward)
  void* out;
  long long xPos, xHead, dyPos, dyHead, outPos, outHead;
  const float* g;
  int heads;
};

struct HnormP {
  HeadsP set[2];
  const double *positions, *frequencies;
  float* partials;     // backward: [workgroups][2][D], or null
  int D, N, pairs, axes, normalise;
  int slices, perSlice;   // of the two sets' heads one behind the other: a wavefront's share of a position
  FastDiv bySlices;
  float epsilon;
};

// Where a chunk of VP pairs lies: its first channels from lo on and the others from hi on (neighbours: the first VP of its channels, and the
// rest); nLo and nHi of them are there.  Chunks of pairs that turn come first, then those of channels of no pair.  WHOLE: nothing is left over in
// either, and everything starts at a multiple of 16 bytes.
template <int VP, bool NEIGHBOURS, bool WHOLE>
struct Place {
  int lo, hi, nLo, nHi, pair;
  bool turned;
  __device__ __forceinline__ Place(int chunk, int D, int pairs) {
    const int turning = (pairs + VP - 1) / VP;
    turned = chunk < turning;
    pair = chunk * VP;
    int left;   // channels from lo on, neighbours and channels of no pair
    if (turned && !NEIGHBOURS) {
      lo = pair;
      hi = pair + pairs;
      nLo = nHi = WHOLE ? VP : std::min(VP, pairs - pair);
      return;
    }
    if (turned) {
      lo = 2 * pair;
      left = 2 * (pairs - pair);
    } else {
      lo = 2 * pairs + 2 * VP * (chunk - turning);
      left = D - lo;
    }
    hi = lo + VP;
    nLo = std::min(VP, left);
    nHi = std::min(VP, left - VP);
    if (WHOLE) nLo = nHi = left > 0 ? VP : 0;
  }
};

// Channels of a lane's pairs: w[0..VP) are those at lo, w[VP..2 VP) those at hi.  Pair e: its two channels' indices in w.
template <int VP, bool NEIGHBOURS> __device__ __forceinline__ constexpr int first_of(int e) { return NEIGHBOURS ? 2 * e : e; }
template <int VP, bool NEIGHBOURS> __device__ __forceinline__ constexpr int second_of(int e) { return NEIGHBOURS ? 2 * e + 1 : VP + e; }

template <class V, int VP>
struct Raw {
  Pack<V, VP> lo, hi;
};
// VP values that may start anywhere
template <class V, int VP> struct Loose;
template <> struct Loose<float, 4> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Loose<bf16, 4> { typedef unsigned short type __attribute__((ext_vector_type(4), aligned(2))); };
template <class V, int VP, bool WHOLE>
__device__ __forceinline__ Pack<V, VP> load_some(const V* at, int n) {
  Pack<V, VP> r = {};
  if constexpr (WHOLE) {
    if (n > 0) r = *(const Pack<V, VP>*)at;
  } else {
    if (n == VP) {
      const typename Loose<V, VP>::type v = *(const typename Loose<V, VP>::type*)at;
#pragma unroll
      for (int e = 0; e < VP; ++e) r.v[e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < VP - 1; ++e)
        if (e < n) r.v[e] = at[e];
    }
  }
  return r;
}
template <class V, int VP, bool WHOLE>
__device__ __forceinline__ void store_some(V* at, int n, const Pack<V, VP>& r) {
  if constexpr (WHOLE) {
    if (n > 0) *(Pack<V, VP>*)at = r;
  } else {
    if (n == VP) {
      typename Loose<V, VP>::type v;
#pragma unroll
      for (int e = 0; e < VP; ++e) v[e] = r.v[e];
      *(typename Loose<V, VP>::type*)at = v;
    } else {
#pragma unroll
      for (int e = 0; e < VP - 1; ++e)
        if (e < n) at[e] = r.v[e];
    }
  }
}
template <class V, int VP>
__device__ __forceinline__ void unpack(float (&w)[2 * VP], const Raw<V, VP>& r) {
#pragma unroll
  for (int e = 0; e < VP; ++e) {
    w[e] = to_float(r.lo.v[e]);
    w[VP + e] = to_float(r.hi.v[e]);
  }
}
template <class V, int VP, bool WHOLE>
__device__ __forceinline__ void store(V* head, int lo, int hi, int nLo, int nHi, const float (&w)[2 * VP]) {
  Raw<V, VP> r;
#pragma unroll
  for (int e = 0; e < VP; ++e) {
    r.lo.v[e] = from_float<V>(w[e]);
    r.hi.v[e] = from_float<V>(w[VP + e]);
  }
  store_some<V, VP, WHOLE>(head + lo, nLo, r.lo);
  store_some<V, VP, WHOLE>(head + hi, nHi, r.hi);
}

// The sum over a group's lanes, in each of them: within 16 lanes by the vector instructions' own lane exchange (through LDS, as shuffles go, the
// four exchanges of each of the backward pass's two sums are waited for: 16384 x 40 heads of 128, bfloat16: 140 us, 120 so)
template <int CONTROL>
__device__ __forceinline__ float exchanged(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
template <int T>
__device__ __forceinline__ float group_sum(float v) {
  v += exchanged<0xB1>(v);                // lane ^ 1
  v += exchanged<0x4E>(v);                // lane ^ 2
  if (T >= 8) v += exchanged<0x141>(v);   // the other four of eight, mirrored
  if (T >= 16) v += exchanged<0x140>(v);  // the other eight of sixteen, mirrored
#pragma unroll
  for (int o = 16; o < T; o *= 2) v += __shfl_xor(v, o, kWave);
  return v;
}

// The cosines and sines of position n's pairs, [2][kMostD / 2] in this wavefront's local memory.
// (LDS accesses of a wavefront are in order; the fences keep the compiler to it.)
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
constexpr int kAxes = 3;   // of so many axes and up to 64 pairs a lane keeps its pair's frequencies
struct Turns {
  double frequency[kAxes], position[kAxes];
};
__device__ __forceinline__ bool kept(const HnormP& p) { return p.axes <= kAxes && p.pairs <= 64; }
__device__ __forceinline__ void angles(float (*lds)[kMostD / 2], const HnormP& p, const Turns& turns, int n, int lane) {
  wave_order();
  for (int j = lane; j < p.pairs; j += 64) {
    double angle = 0.0;
    if (kept(p)) {
#pragma unroll
      for (int a = 0; a < kAxes; ++a) angle += turns.position[a] * turns.frequency[a];
    } else {
      for (int a = 0; a < p.axes; ++a) angle += p.positions[(size_t)n * p.axes + a] * p.frequencies[(size_t)a * p.pairs + j];
    }
    double r = angle * 0.15915494309189533577;   // revolutions
    r -= rint(r);
    // (half revolutions in two parts: rounded to one the sine near a whole one would be off by up to 9e-8, whatever is left of it)
    const float half = (float)(2.0 * r), rest = (float)((2.0 * r - (double)half) * 3.14159265358979323846);
    float s, c;
    sincospif(half, &s, &c);
    lds[0][j] = c - rest * s;
    lds[1][j] = s + rest * c;
  }
  wave_order();
}

// A wavefront's place in its work: kGroups * HB heads of a set from `first` on, of position n
struct Cursor {
  int unit, n, which, first, to;
};

// T lanes to a head, NCH chunks of VP pairs a lane, HB heads a lane at a time; the next HB are on their way meanwhile, the next position's
// too (16384 x 40 heads of 128, bfloat16: forward and backward 109 and 183 us with a position's loads behind its angles, 72 and 120 so).
template <class V, int VP, int T, int NCH, int HB, bool NEIGHBOURS, bool WHOLE, bool BACKWARD>
__global__ __launch_bounds__(64 * kWaves) void hnorm_kernel(HnormP p) {
  constexpr int kGroups = 64 / T, W = 2 * VP;
  __shared__ float turn[kWaves][2][kMostD / 2];
  __shared__ float join[BACKWARD ? kWaves * 64 * W : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, t = lane % T, group = lane / T;
  const int units = p.N * p.slices, step = gridDim.x * kWaves;
  float g[2][NCH][W], sums[BACKWARD ? 2 : 1][NCH][W], cosine[NCH][VP], sine[NCH][VP];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
#pragma unroll
      for (int e = 0; e < VP; ++e) {
        g[w][i][e] = p.set[w].g && e < at.nLo ? p.set[w].g[at.lo + e] : 1.f;
        g[w][i][VP + e] = p.set[w].g && e < at.nHi ? p.set[w].g[at.hi + e] : 1.f;
        if (BACKWARD) sums[w][i][e] = sums[w][i][VP + e] = 0.f;
      }
    }

  // the first heads at or behind a place
  const auto settle = [&](Cursor& c) __attribute__((always_inline)) {
    while (c.unit < units) {
      int slice;
      p.bySlices.divmod(c.unit, &c.n, &slice);
      for (; c.which < 2; ++c.which, c.first = -1) {
        const int before = c.which ? p.set[0].heads : 0;
        c.to = std::min(p.set[c.which].heads, (slice + 1) * p.perSlice - before);
        if (c.first < 0) c.first = std::max(0, slice * p.perSlice - before);
        if (c.first < c.to) return;
      }
      c.unit += step;
      c.which = 0;
      c.first = -1;
    }
  };
  typedef Raw<V, VP> Heads[HB][NCH];
  const auto fetch_heads = [&](Heads& x, Heads& d, const Cursor& c) __attribute__((always_inline)) {
    const HeadsP& set = p.set[c.which];
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int h = c.first + b * kGroups + group;
      const bool mine = h < c.to;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
        const int nLo = mine ? at.nLo : 0, nHi = mine ? at.nHi : 0;
        if (!BACKWARD || p.normalise) {
          const V* from = (const V*)set.x + c.n * set.xPos + h * set.xHead;
          x[b][i].lo = load_some<V, VP, WHOLE>(from + at.lo, nLo);
          x[b][i].hi = load_some<V, VP, WHOLE>(from + at.hi, nHi);
        }
        if (BACKWARD) {
          const V* from = (const V*)set.dy + c.n * set.dyPos + h * set.dyHead;
          d[b][i].lo = load_some<V, VP, WHOLE>(from + at.lo, nLo);
          d[b][i].hi = load_some<V, VP, WHOLE>(from + at.hi, nHi);
        }
      }
    }
  };
  const auto work = [&](const HeadsP& set, const float (&g)[NCH][W], float (&sums)[NCH][W], const Heads& x, const Heads& d, const Cursor& c)
                        __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int h = c.first + b * kGroups + group;
      const bool mine = h < c.to;
      float w[NCH][W];
      float squares = 0.f;
      if (!BACKWARD || p.normalise) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          unpack<V, VP>(w[i], x[b][i]);
#pragma unroll
          for (int e = 0; e < W; ++e) squares += w[i][e] * w[i][e];
        }
      }
      float inv = 1.f;
      if (p.normalise) {
        inv = 1.f / sqrtf(group_sum<T>(squares) / (float)p.D + p.epsilon);
        if (BACKWARD && !mine) inv = 1.f;   // (no head: zero times what is finite, also with an epsilon of 0)
      }
      if (!BACKWARD) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
          if (p.normalise) {
#pragma unroll
            for (int e = 0; e < W; ++e) w[i][e] = w[i][e] * inv * g[i][e];
          }
#pragma unroll
          for (int e = 0; e < VP; ++e) {
            const int F = first_of<VP, NEIGHBOURS>(e), S = second_of<VP, NEIGHBOURS>(e);
            const float lo = w[i][F], hi = w[i][S];
            w[i][F] = at.turned ? lo * cosine[i][e] - hi * sine[i][e] : lo;
            w[i][S] = at.turned ? hi * cosine[i][e] + lo * sine[i][e] : hi;
          }
          if (mine) store<V, VP, WHOLE>((V*)set.out + c.n * set.outPos + h * set.outHead, at.lo, at.hi, at.nLo, at.nHi, w[i]);
        }
      } else {
        float du[NCH][W];
        float product = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
          unpack<V, VP>(du[i], d[b][i]);
#pragma unroll
          for (int e = 0; e < VP; ++e) {
            const int F = first_of<VP, NEIGHBOURS>(e), S = second_of<VP, NEIGHBOURS>(e);
            const float lo = du[i][F], hi = du[i][S];
            du[i][F] = at.turned ? lo * cosine[i][e] + hi * sine[i][e] : lo;
            du[i][S] = at.turned ? hi * cosine[i][e] - lo * sine[i][e] : hi;
          }
          if (p.normalise) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
              w[i][e] *= inv;
              sums[i][e] += du[i][e] * w[i][e];   // (what is no channel, or no head, is zero)
              du[i][e] *= g[i][e];
              product += du[i][e] * w[i][e];
            }
          }
        }
        if (p.normalise) product = group_sum<T>(product) / (float)p.D;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
          if (p.normalise) {
#pragma unroll
            for (int e = 0; e < W; ++e) du[i][e] = (du[i][e] - w[i][e] * product) * inv;
          }
          if (set.out && mine) store<V, VP, WHOLE>((V*)set.out + c.n * set.outPos + h * set.outHead, at.lo, at.hi, at.nLo, at.nHi, du[i]);
        }
      }
    }
  };

  // (asked for ahead of the heads, so that they are waited for alone)
  Turns turns;
#pragma unroll
  for (int a = 0; a < kAxes; ++a) turns.position[a] = turns.frequency[a] = 0.0;
  const auto fetch_position = [&](const Cursor& c) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < kAxes; ++a)
      if (a < p.axes) turns.position[a] = p.positions[(size_t)c.n * p.axes + a];
  };
  const bool keeps = p.pairs && kept(p);
  if (keeps) {
#pragma unroll
    for (int a = 0; a < kAxes; ++a)
      if (a < p.axes && lane < p.pairs) turns.frequency[a] = p.frequencies[(size_t)a * p.pairs + lane];
  }
  Heads xa, da, xb, db;
  Cursor here = {(int)blockIdx.x * kWaves + wave, 0, 0, -1, 0};
  settle(here);
  if (here.unit < units) {
    if (keeps) fetch_position(here);
    fetch_heads(xa, da, here);
  }
  int angled = -1;   // the position whose angles are at hand
  const auto turn_over = [&](Heads& x, Heads& d, Heads& nextX, Heads& nextD) __attribute__((always_inline)) {
    if (angled != here.n && p.pairs) {
      angled = here.n;
      angles(turn[wave], p, turns, here.n, lane);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const Place<VP, NEIGHBOURS, WHOLE> at(i * T + t, p.D, p.pairs);
#pragma unroll
        for (int e = 0; e < VP; ++e) {
          const int j = at.turned && at.pair + e < p.pairs ? at.pair + e : 0;
          cosine[i][e] = turn[wave][0][j];
          sine[i][e] = turn[wave][1][j];
        }
      }
    }
    Cursor next = here;
    next.first += kGroups * HB;
    settle(next);
    if (next.unit < units) {
      if (keeps && next.n != here.n) fetch_position(next);
      fetch_heads(nextX, nextD, next);
    }
    if (here.which == 0) work(p.set[0], g[0], sums[0], x, d, here);
    else work(p.set[1], g[1], sums[BACKWARD ? 1 : 0], x, d, here);
    here = next;
  };
  while (here.unit < units) {
    turn_over(xa, da, xb, db);
    if (here.unit >= units) break;
    turn_over(xb, db, xa, da);
  }
  if (!BACKWARD || !p.partials) return;
  // the workgroup's sums: groups and wavefronts added up in one order
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < W; ++e) join[threadIdx.x * W + e] = sums[which][i][e];
      __syncthreads();
      float* out = p.partials + ((size_t)blockIdx.x * 2 + which) * p.D;
      for (int k = threadIdx.x; k < T * W; k += 64 * kWaves) {
        const Place<VP, NEIGHBOURS, WHOLE> at(i * T + k / W, p.D, p.pairs);
        const int e = k % W;
        float s = 0.f;
#pragma unroll 8
        for (int j = 0; j < kWaves * kGroups; ++j) s += join[j * T * W + k];
        if (e % VP < (e < VP ? at.nLo : at.nHi)) out[(e < VP ? at.lo : at.hi) + e % VP] = s;
      }
    }
}

// dzdg of both sets from the workgroups' sums: 32 of the 2 D sums per workgroup, eight threads each, in double, in one order
__global__ __launch_bounds__(256) void hnorm_join(float* __restrict__ dgq, float* __restrict__ dgk, const float* __restrict__ partials, int D, int parts) {
  __shared__ double slots[8][33];
  const int t = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + t;
  double s = 0.0;
  if (c < 2 * D) {
    int k = r;
    for (; k + 56 < parts; k += 64) {   // eight loads at a time
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = partials[(size_t)(k + 8 * i) * 2 * D + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (double)v[i];
    }
    for (; k < parts; k += 8) s += (double)partials[(size_t)k * 2 * D + c];
  }
  slots[r][t] = s;
  __syncthreads();
  if (r || c >= 2 * D) return;
  for (int k = 1; k < 8; ++k) s += slots[k][t];
  float* out = c < D ? dgq : dgk;
  if (out) out[c < D ? c : c - D] = (float)s;
}

// ---------------------------------------------------------------------------------------------- host

// chunks of a head: of pairs that turn, and of channels of no pair
int chunks_of(const HnormP& p, int VP) { return div_up(p.pairs, VP) + div_up(p.D - 2 * p.pairs, 2 * VP); }

// Workgroups: as many as run at once (forward 4 on a CU, backward 3), each walks over positions
int groups_of(long long units, int perUnit) {
  return (int)std::max<long long>(1, std::min<long long>((long long)perUnit * std::max(1, device_compute_units()), (units + kWaves - 1) / kWaves));
}
int backward_groups(long long units) { return groups_of(units, 3); }

template <class V, int VP, int T, int NCH, bool NEIGHBOURS, bool WHOLE>
void launch_kernel(hipStream_t s, const HnormP& p, bool backward, int groups) {
  constexpr int forwardBatch = NCH == 1 ? 2 : 1, backwardBatch = sizeof(V) == 2 && NCH == 1 ? 2 : 1;
  if (backward)
    hipLaunchKernelGGL((hnorm_kernel<V, VP, T, NCH, backwardBatch, NEIGHBOURS, WHOLE, true>), dim3((unsigned)groups), dim3(64 * kWaves), 0, s, p);
  else
    hipLaunchKernelGGL((hnorm_kernel<V, VP, T, NCH, forwardBatch, NEIGHBOURS, WHOLE, false>), dim3((unsigned)groups_of((long long)p.N * p.slices, 4)),
                       dim3(64 * kWaves), 0, s, p);
}

template <class V, bool NEIGHBOURS>
void choose(hipStream_t s, const HnormP& p, bool wide, bool backward, int groups) {
  constexpr int VP = 4;
  const int chunks = chunks_of(p, VP);
  if (wide) {
    if (chunks <= 4) launch_kernel<V, VP, 4, 1, NEIGHBOURS, true>(s, p, backward, groups);
    else if (chunks <= 8) launch_kernel<V, VP, 8, 1, NEIGHBOURS, true>(s, p, backward, groups);
    else if (chunks <= 16) launch_kernel<V, VP, 16, 1, NEIGHBOURS, true>(s, p, backward, groups);
    else if (chunks <= 32) launch_kernel<V, VP, 32, 1, NEIGHBOURS, true>(s, p, backward, groups);
    else launch_kernel<V, VP, 64, 1, NEIGHBOURS, true>(s, p, backward, groups);
  } else {
    if (chunks <= 8) launch_kernel<V, 4, 8, 1, NEIGHBOURS, false>(s, p, backward, groups);
    else if (chunks <= 16) launch_kernel<V, 4, 16, 1, NEIGHBOURS, false>(s, p, backward, groups);
    else if (chunks <= 64) launch_kernel<V, 4, 64, 1, NEIGHBOURS, false>(s, p, backward, groups);
    else launch_kernel<V, 4, 64, 2, NEIGHBOURS, false>(s, p, backward, groups);
  }
}

bool wide_heads(const mcn_heads* t, int VP) { return aligned16(t->data) && t->position % VP == 0 && t->head % VP == 0; }

int check_geom(const char* who, const mcn_hnorm_geom* g) {
  if (!g) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null geometry", who);
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d", who, g->dataType);
  if (g->D < 0 || g->heads < 0 || g->keyHeads < 0 || g->N < 0 || g->pairs < 0 || g->axes < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative extent", who);
  if (g->D > kMostD) return fail(MCN_UNSUPPORTED, "%s: heads of more than %d channels", who, kMostD);
  if (g->heads > 65536 || g->keyHeads > 65536) return fail(MCN_UNSUPPORTED, "%s: more than 65536 heads", who);
  if (g->N > 1 << 30) return fail(MCN_UNSUPPORTED, "%s: too many positions", who);
  if (2ll * g->pairs > g->D) return fail(MCN_ILLEGAL_ARGUMENT, "%s: %d pairs of %d channels", who, g->pairs, g->D);
  if (g->pairs && g->axes == 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: pairs, but no axes", who);
  if (g->axes > 64) return fail(MCN_UNSUPPORTED, "%s: more than 64 axes", who);
  if (!(g->epsilon >= 0)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: EPSILON is negative", who);
  return MCN_SUCCESS;
}

// A wavefront takes all heads of a position; where that leaves most of the chip idle, a few of them.
void share_out(HnormP* p, int lanes) {
  const int heads = p->set[0].heads + p->set[1].heads, most = std::max(1, heads * lanes / 64);   // (one turn of all groups at least)
  const long long want = 8ll * std::max(1, device_compute_units());
  const int slices = (int)std::max<long long>(1, std::min<long long>(most, want / std::max(1, p->N)));
  p->perSlice = std::max(1, div_up(heads, slices));
  p->slices = std::max(1, div_up(heads, p->perSlice));
  p->bySlices = FastDiv(p->slices);
}

int lanes_of(const HnormP& p, int VP, bool wide) {
  const int chunks = chunks_of(p, wide ? VP : 4);
  if (!wide) return chunks <= 8 ? 8 : chunks <= 16 ? 16 : 64;
  return chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64;
}

struct Call {
  const mcn_heads *xq, *xk, *dyq, *dyk, *outq, *outk;
  const float *gq, *gk;
};

int run(const char* who, hipStream_t s, const mcn_hnorm_geom* g, const Call& c, const double* positions, const double* frequencies, bool backward,
        float* dgq, float* dgk, void* workspace, size_t workspaceBytes) {
  const int size = g->dataType == MCN_BFLOAT16 ? 2 : 4, VP = 4;
  HnormP p = {};
  p.D = g->D; p.N = g->N; p.axes = g->axes;
  p.pairs = positions ? g->pairs : 0;
  p.normalise = g->normalise != 0;
  p.epsilon = (float)g->epsilon;
  p.positions = positions; p.frequencies = frequencies;
  bool wide = p.pairs % VP == 0 && p.D % (2 * VP) == 0;
  const mcn_heads *x[2] = {c.xq, c.xk}, *dy[2] = {c.dyq, c.dyk}, *out[2] = {c.outq, c.outk};
  for (int w = 0; w < 2; ++w) {
    HeadsP& h = p.set[w];
    h.heads = w ? g->keyHeads : g->heads;
    h.g = w ? c.gk : c.gq;
    if (!h.heads) continue;
    const bool reads = !backward || p.normalise;
    int rc = reads ? check_heads(who, w ? "keys" : "queries", x[w], h.heads, g->N, g->D, size, false) : 0;
    if (!rc && backward) rc = check_heads(who, w ? "keys' derivative" : "queries' derivative", dy[w], h.heads, g->N, g->D, size, false);
    if (!rc && (!backward || (out[w] && out[w]->data))) rc = check_heads(who, w ? "keys' output" : "queries' output", out[w], h.heads, g->N, g->D, size, true);
    if (rc) return rc;
    if (reads) {
      h.x = x[w]->data; h.xPos = x[w]->position; h.xHead = x[w]->head;
      wide = wide && wide_heads(x[w], VP);
    }
    if (backward) {
      h.dy = dy[w]->data; h.dyPos = dy[w]->position; h.dyHead = dy[w]->head;
      wide = wide && wide_heads(dy[w], VP);
    }
    if (out[w] && out[w]->data) {
      h.out = out[w]->data; h.outPos = out[w]->position; h.outHead = out[w]->head;
      wide = wide && wide_heads(out[w], VP);
    }
  }
  share_out(&p, lanes_of(p, VP, wide));
  const long long units = (long long)p.N * p.slices;
  const int groups = backward_groups(units);
  const bool sums = backward && p.normalise && (dgq || dgk);
  if (sums) {
    const size_t need = (size_t)groups * 2 * p.D * sizeof(float);
    const int rc = check_workspace(who, workspace, workspaceBytes, need);
    if (rc) return rc;
    p.partials = (float*)workspace;
  }
  {
    KernelTimer timer(backward ? "hnorm_backward" : "hnorm_forward", s);
    if (g->dataType == MCN_BFLOAT16) {
      if (g->neighbours) choose<bf16, true>(s, p, wide, backward, groups);
      else choose<bf16, false>(s, p, wide, backward, groups);
    } else {
      if (g->neighbours) choose<float, true>(s, p, wide, backward, groups);
      else choose<float, false>(s, p, wide, backward, groups);
    }
  }
  int rc = check_launch(who);
  if (rc || !sums) return rc;
  KernelTimer timer("hnorm_join", s);
  hipLaunchKernelGGL(hnorm_join, dim3((unsigned)div_up(2 * p.D, 32)), dim3(256), 0, s, dgq, dgk, p.partials, p.D, groups);
  return check_launch(who);
}

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_hnorm_workspace_bytes(const mcn_hnorm_geom* g) {
  if (!g || g->D <= 0 || g->N <= 0 || !g->normalise) return 0;
  // (as many workgroups as there could be at most)
  return (size_t)backward_groups((long long)g->N * std::max(1, g->heads + g->keyHeads)) * 2 * g->D * sizeof(float);
}

int mcn_hnorm_forward(mcn_stream_t stream, const mcn_hnorm_geom* g, const mcn_heads* yq, const mcn_heads* yk, const mcn_heads* q, const mcn_heads* k,
                      const float* multipliersQ, const float* multipliersK, const double* positions, const double* frequencies) {
  const char* who = "mcn_hnorm_forward";
  int rc = check_geom(who, g);
  if (rc || g->D == 0 || g->N == 0 || g->heads + g->keyHeads == 0) return rc;
  if (g->pairs && (!positions || !frequencies)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null positions or frequencies", who);
  const Call c = {q, k, nullptr, nullptr, yq, yk, multipliersQ, multipliersK};
  return run(who, as_stream(stream), g, c, positions, frequencies, false, nullptr, nullptr, nullptr, 0);
}

int mcn_hnorm_backward(mcn_stream_t stream, const mcn_hnorm_geom* g, const mcn_heads* derQ, const mcn_heads* derK, float* derMultipliersQ,
                       float* derMultipliersK, const mcn_heads* q, const mcn_heads* k, const float* multipliersQ, const float* multipliersK,
                       const double* positions, const double* frequencies, const mcn_heads* derOutputQ, const mcn_heads* derOutputK, void* workspace,
                       size_t workspaceBytes) {
  const char* who = "mcn_hnorm_backward";
  int rc = check_geom(who, g);
  if (rc || g->D == 0) return rc;
  if (!g->normalise && (derMultipliersQ || derMultipliersK)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: derivatives of multipliers without the norm", who);
  if (g->pairs && g->N && (!positions || !frequencies)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null positions or frequencies", who);
  hipStream_t s = as_stream(stream);
  if (g->N == 0 || g->heads + g->keyHeads == 0) {   // no heads: the sums over them are zero
    if (!g->normalise || (!derMultipliersQ && !derMultipliersK)) return MCN_SUCCESS;
    hipLaunchKernelGGL(hnorm_join, dim3((unsigned)div_up(2 * g->D, 32)), dim3(256), 0, s, derMultipliersQ, derMultipliersK, (const float*)nullptr, g->D, 0);
    return check_launch(who);
  }
  const Call c = {q, k, derOutputQ, derOutputK, derQ, derK, multipliersQ, multipliersK};
  return run(who, s, g, c, positions, frequencies, true, derMultipliersQ, derMultipliersK, workspace, workspaceBytes);
}

}  // extern "C"
