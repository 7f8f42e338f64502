// The heads of queries and keys, each divided by the root of its mean square, scaled per channel, and turned pair by pair by angles made of
// its position.
//   sigma = sqrt(mean_d x^2 + epsilon), xh = x/sigma, u = g xh;  angle_j = sum_a position[n][a] frequency[a][j]
//   (y_lo, y_hi) = (u_lo cos - u_hi sin, u_hi cos + u_lo sin) for the two channels of pair j; channels of no pair stay u
//   backward: du = the pairs of dzdy turned back, dzdg = sum over positions and heads of du xh, a = g du,
//             dzdx = (a - xh mean_d(a xh))/sigma
// Bound by memory: a head's channels stay in the registers of T lanes between the sum of squares and the output.  A wavefront takes
// the heads of one position, so that the angles of a position are made once: lane by lane one pair each, the cosines and sines
// then pass through local memory to the lanes that hold the pair in each head.  Angles are products and sums of doubles, brought to a
// revolution in double: position 10^6 times frequency 1 keeps all of a single-precision sine.
//
// A lane holds VP pairs, 2 VP channels: the pairs' first channels and their second ones a run of pairs apart, or neighbours.  Channels of
// no pair are held as pairs that are not turned.
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
  float epsilon;
};

// where VP pairs from the chunk's first one on lie: their first VP channels and the other VP
template <int VP, bool NEIGHBOURS>
struct Place {
  int lo, hi;
  bool turned, live, both;   // both: false where an odd channel is left (VP == 1)
  __device__ __forceinline__ Place(int chunk, int D, int pairs) {
    const int c = chunk * VP;
    turned = c < pairs;
    if (turned) {
      lo = NEIGHBOURS ? 2 * c : c;
      hi = NEIGHBOURS ? 2 * c + VP : c + pairs;
    } else {
      lo = 2 * c;   // = 2 pairs + 2 (c - pairs)
      hi = lo + VP;
    }
    live = lo < D;
    both = hi < D;
  }
};

// Channels of a lane's pairs: w[0..VP) are those at lo, w[VP..2 VP) those at hi.  Pair e: its two channels' indices in w.
template <int VP, bool NEIGHBOURS> __device__ __forceinline__ constexpr int first_of(int e) { return NEIGHBOURS ? 2 * e : e; }
template <int VP, bool NEIGHBOURS> __device__ __forceinline__ constexpr int second_of(int e) { return NEIGHBOURS ? 2 * e + 1 : VP + e; }

template <class V, int VP>
struct Raw {
  Pack<V, VP> lo, hi;
};
template <class V, int VP>
__device__ __forceinline__ Raw<V, VP> fetch(const V* head, int lo, int hi, bool live, bool both) {
  Raw<V, VP> r = {};
  if (live) r.lo = *(const Pack<V, VP>*)(head + lo);
  if (live && both) r.hi = *(const Pack<V, VP>*)(head + hi);
  return r;
}
template <class V, int VP>
__device__ __forceinline__ void unpack(float (&w)[2 * VP], const Raw<V, VP>& r) {
#pragma unroll
  for (int e = 0; e < VP; ++e) {
    w[e] = to_float(r.lo.v[e]);
    w[VP + e] = to_float(r.hi.v[e]);
  }
}
template <class V, int VP>
__device__ __forceinline__ void store(V* head, int lo, int hi, bool both, const float (&w)[2 * VP]) {
  Raw<V, VP> r;
#pragma unroll
  for (int e = 0; e < VP; ++e) {
    r.lo.v[e] = from_float<V>(w[e]);
    r.hi.v[e] = from_float<V>(w[VP + e]);
  }
  *(Pack<V, VP>*)(head + lo) = r.lo;
  if (both) *(Pack<V, VP>*)(head + hi) = r.hi;
}

template <int T>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = T / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// The cosines and sines of position n's pairs, [2][kMostD / 2] in this wavefront's local memory.
// (LDS accesses of a wavefront are in order; the fences keep the compiler to it.)
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ void angles(float (*lds)[kMostD / 2], const HnormP& p, int n, int lane) {
  wave_order();
  for (int j = lane; j < p.pairs; j += 64) {
    double angle = 0.0;
    for (int a = 0; a < p.axes; ++a) angle += p.positions[(size_t)n * p.axes + a] * p.frequencies[(size_t)a * p.pairs + j];
    double r = angle * 0.15915494309189533577;   // revolutions
    r -= rint(r);
    float s, c;
    sincospif((float)(2.0 * r), &s, &c);
    lds[0][j] = c;
    lds[1][j] = s;
  }
  wave_order();
}

// T lanes to a head, NCH chunks of VP pairs a lane, HB heads on their way at a time
template <class V, int VP, int T, int NCH, int HB, bool NEIGHBOURS, bool BACKWARD>
__global__ __launch_bounds__(64 * kWaves) void hnorm_kernel(HnormP p) {
  constexpr int kGroups = 64 / T, W = 2 * VP;
  __shared__ float turn[kWaves][2][kMostD / 2];
  __shared__ float join[BACKWARD ? kWaves * 64 * W : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = lane % T, group = lane / T;
  float sums[2][NCH][W];
  if (BACKWARD) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) sums[w][i][e] = 0.f;
  }
  const long long units = (long long)p.N * p.slices, step = (long long)gridDim.x * kWaves;
  for (long long unit = (long long)blockIdx.x * kWaves + wave; unit < units; unit += step) {
    const int n = __builtin_amdgcn_readfirstlane((int)(unit / p.slices)), slice = __builtin_amdgcn_readfirstlane((int)(unit % p.slices));
    angles(turn[wave], p, n, lane);
    float cosine[NCH][VP], sine[NCH][VP];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
#pragma unroll
      for (int e = 0; e < VP; ++e) {
        const int j = at.turned ? (i * T + t) * VP + e : 0;
        cosine[i][e] = turn[wave][0][j];
        sine[i][e] = turn[wave][1][j];
      }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const HeadsP& set = p.set[which];
      const int before = which ? p.set[0].heads : 0;
      const int from = std::max(0, slice * p.perSlice - before), to = std::min(set.heads, (slice + 1) * p.perSlice - before);
      if (from >= to) continue;
      float g[NCH][W];
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
#pragma unroll
        for (int e = 0; e < VP; ++e) {
          g[i][e] = set.g && at.live ? set.g[at.lo + e] : 1.f;
          g[i][VP + e] = set.g && at.live && at.both ? set.g[at.hi + e] : 1.f;
        }
      }
      for (int first = from; first < to; first += kGroups * HB) {
        Raw<V, VP> x[HB][NCH], d[HB][BACKWARD ? NCH : 1];
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          const int h = first + b * kGroups + group;
          const bool mine = h < to;
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
            x[b][i] = {};
            if (!BACKWARD || p.normalise) x[b][i] = fetch<V, VP>((const V*)set.x + n * set.xPos + h * set.xHead, at.lo, at.hi, mine && at.live, at.both);
            if (BACKWARD) d[b][i] = fetch<V, VP>((const V*)set.dy + n * set.dyPos + h * set.dyHead, at.lo, at.hi, mine && at.live, at.both);
          }
        }
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          const int h = first + b * kGroups + group;
          const bool mine = h < to;
          float w[NCH][W];
          float squares = 0.f;
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            unpack<V, VP>(w[i], x[b][i]);
#pragma unroll
            for (int e = 0; e < W; ++e) squares += w[i][e] * w[i][e];
          }
          float inv = 1.f;
          if (p.normalise) inv = 1.f / sqrtf(group_sum<T>(squares) / (float)p.D + p.epsilon);
          if (!BACKWARD) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
              const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
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
              if (mine && at.live) store<V, VP>((V*)set.out + n * set.outPos + h * set.outHead, at.lo, at.hi, at.both, w[i]);
            }
          } else {
            float du[NCH][W];
            float product = 0.f;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
              const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
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
                  sums[which][i][e] += du[i][e] * w[i][e];   // (what is no channel, or no head, is zero)
                  du[i][e] *= g[i][e];
                  product += du[i][e] * w[i][e];
                }
              }
            }
            if (p.normalise) product = group_sum<T>(product) / (float)p.D;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
              const Place<VP, NEIGHBOURS> at(i * T + t, p.D, p.pairs);
              if (p.normalise) {
#pragma unroll
                for (int e = 0; e < W; ++e) du[i][e] = (du[i][e] - w[i][e] * product) * inv;
              }
              if (set.out && mine && at.live) store<V, VP>((V*)set.out + n * set.outPos + h * set.outHead, at.lo, at.hi, at.both, du[i]);
            }
          }
        }
      }
    }
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
        const Place<VP, NEIGHBOURS> at(i * T + k / W, p.D, p.pairs);
        const int e = k % W;
        float s = 0.f;
#pragma unroll 8
        for (int j = 0; j < kWaves * kGroups; ++j) s += join[j * T * W + k];
        if (at.live && (e < VP || at.both)) out[(e < VP ? at.lo : at.hi) + e % VP] = s;
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

// workgroups of a backward pass: as many as run at once, each sums as it goes
int backward_groups(long long units) { return (int)std::max<long long>(1, std::min<long long>(2ll * std::max(1, device_compute_units()), (units + kWaves - 1) / kWaves)); }

template <class V, int VP, int T, int NCH, bool NEIGHBOURS>
void launch_kernel(hipStream_t s, const HnormP& p, bool backward, int groups) {
  constexpr int forwardBatch = NCH == 1 ? 4 : 2, backwardBatch = NCH == 1 ? 2 : 1;
  const long long units = (long long)p.N * p.slices;
  if (backward)
    hipLaunchKernelGGL((hnorm_kernel<V, VP, T, NCH, backwardBatch, NEIGHBOURS, true>), dim3((unsigned)groups), dim3(64 * kWaves), 0, s, p);
  else
    hipLaunchKernelGGL((hnorm_kernel<V, VP, T, NCH, forwardBatch, NEIGHBOURS, false>), dim3((unsigned)std::min<long long>((units + kWaves - 1) / kWaves, 1 << 20)),
                       dim3(64 * kWaves), 0, s, p);
}

template <class V, bool NEIGHBOURS>
void choose(hipStream_t s, const HnormP& p, bool wide, bool backward, int groups) {
  constexpr int VP = 16 / sizeof(V);
  if (wide) {
    const int chunks = div_up(p.D, 2 * VP);
    if (chunks <= 4) launch_kernel<V, VP, 4, 1, NEIGHBOURS>(s, p, backward, groups);
    else if (chunks <= 8) launch_kernel<V, VP, 8, 1, NEIGHBOURS>(s, p, backward, groups);
    else if (chunks <= 16) launch_kernel<V, VP, 16, 1, NEIGHBOURS>(s, p, backward, groups);
    else if (chunks <= 32) launch_kernel<V, VP, 32, 1, NEIGHBOURS>(s, p, backward, groups);
    else launch_kernel<V, VP, 64, 1, NEIGHBOURS>(s, p, backward, groups);
  } else {
    const int chunks = div_up(p.D, 2);
    if (chunks <= 16) launch_kernel<V, 1, 16, 1, NEIGHBOURS>(s, p, backward, groups);
    else if (chunks <= 64) launch_kernel<V, 1, 64, 1, NEIGHBOURS>(s, p, backward, groups);
    else if (chunks <= 128) launch_kernel<V, 1, 64, 2, NEIGHBOURS>(s, p, backward, groups);
    else launch_kernel<V, 1, 64, 4, NEIGHBOURS>(s, p, backward, groups);
  }
}

int check_heads(const char* who, const char* what, const mcn_heads* t, int heads, int N, int D, int size, bool written) {
  if (!t || !t->data) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null %s", who, what);
  if ((uintptr_t)t->data % size) return fail(MCN_ILLEGAL_ARGUMENT, "%s: %s is not aligned", who, what);
  if (t->position < 0 || t->head < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative stride of %s", who, what);
  if (t->position > (1ll << 31) || t->head > (1ll << 40)) return fail(MCN_UNSUPPORTED, "%s: stride of %s too large", who, what);
  if (!written) return MCN_SUCCESS;
  // the heads of all positions are apart
  const bool inside = (N <= 1 || t->position >= (long long)(heads - 1) * t->head + D) && (heads <= 1 || t->head >= D);
  const bool outside = (heads <= 1 || t->head >= (long long)(N - 1) * t->position + D) && (N <= 1 || t->position >= D);
  if (!inside && !outside) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the heads of %s overlap", who, what);
  return MCN_SUCCESS;
}

bool wide_heads(const mcn_heads* t, int VP) { return aligned16(t->data) && t->position % VP == 0 && t->head % VP == 0; }

int check_geom(const char* who, const mcn_hnorm_geom* g) {
  if (!g) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null geometry", who);
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d", who, g->dataType);
  if (g->D < 0 || g->heads < 0 || g->keyHeads < 0 || g->N < 0 || g->pairs < 0 || g->axes < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative extent", who);
  if (g->D > kMostD) return fail(MCN_UNSUPPORTED, "%s: heads of more than %d channels", who, kMostD);
  if (g->heads > 65536 || g->keyHeads > 65536) return fail(MCN_UNSUPPORTED, "%s: more than 65536 heads", who);
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
}

int lanes_of(const HnormP& p, int VP, bool wide) {
  const int chunks = div_up(p.D, wide ? 2 * VP : 2);
  if (!wide) return chunks <= 16 ? 16 : 64;
  return chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64;
}

struct Call {
  const mcn_heads *xq, *xk, *dyq, *dyk, *outq, *outk;
  const float *gq, *gk;
};

int run(const char* who, hipStream_t s, const mcn_hnorm_geom* g, const Call& c, const double* positions, const double* frequencies, bool backward,
        float* dgq, float* dgk, void* workspace, size_t workspaceBytes) {
  const int size = g->dataType == MCN_BFLOAT16 ? 2 : 4, VP = 16 / size;
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
    if (!workspace || workspaceBytes < need) return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, need);
    if (!aligned16(workspace)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the workspace is not 16-byte aligned", who);
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
