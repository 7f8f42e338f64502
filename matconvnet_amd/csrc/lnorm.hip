// Layer normalisation: the C channels of every pixel (of every image) are brought to mean 0 and deviation 1, then scaled and shifted per
// channel.
//   mu = mean_c x, sigma = sqrt(mean_c (x - mu)^2 + epsilon), xh = (x - mu)/sigma, y = g xh + b
//   a = g dzdy:  dzdx = (a - mean_c a - xh mean_c(a xh))/sigma,  dzdg = sum over pixels of dzdy xh,  dzdb = sum of dzdy
// Bound by memory: x is read once (it stays in registers between the mean, the squares about the mean and the output), x and dzdy
// once in the backward pass.  The derivatives of g and b are sums over all pixels: every workgroup walks over many pixels with its
// share of the sums in registers and leaves one partial sum per channel, which a second launch adds up in a fixed order.
//
// Two layouts.  "Rows": H = W = 1, a pixel's channels are neighbours; T lanes (16 to 1024) share a row.  "Planes": channels are a
// plane apart; lanes are pixels and the wavefronts of a workgroup share the channels.  Pixels with more channels than a workgroup
// holds in registers are walked three times (lnorm_long_*).
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

__device__ __forceinline__ unsigned to_bits(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ unsigned to_bits(bf16 v) { return v; }
template <class V> __device__ __forceinline__ float from_bits(unsigned b) { return __builtin_bit_cast(float, sizeof(V) == 4 ? b : b << 16); }

template <class V, int N> struct alignas(sizeof(V) * N) Pack { V v[N]; };

struct LnP {
  int C, HW;
  size_t items;        // pixels of all images
  float epsilon;
  int given;           // moments are an input
};

// One dimension of a grid holds less than 2^32 threads: more workgroups than kGridRow stand in rows of as many.
constexpr size_t kGridRow = 1 << 20;
__device__ __forceinline__ size_t block_of_grid() { return (size_t)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 grid_of(size_t blocks) { return dim3((unsigned)std::min(blocks, kGridRow), (unsigned)((blocks + kGridRow - 1) / kGridRow)); }

// A barrier for what lies in LDS: __syncthreads() also waits for every load and store that is on its way, the next row's and the last one's
// output among them (8192 rows of 4096 bfloat16 values, backward: 57 us with it, 50 without).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The sums of two values over the T threads of a group; T > 64: over the wavefronts by local memory, with a barrier that the whole
// workgroup reaches (two sets of slots in turn: one barrier per sum).
template <int T>
__device__ __forceinline__ void group_sum(float& a, float& b, float2* slots) {
#pragma unroll
  for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, kWave);
    b += __shfl_xor(b, o, kWave);
  }
  if (T > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) slots[wave] = make_float2(a, b);
    lds_barrier();
    const int first = wave / (T / 64) * (T / 64);
    a = b = 0.f;
#pragma unroll
    for (int k = 0; k < T / 64; ++k) {
      const float2 s = slots[first + k];
      a += s.x;
      b += s.y;
    }
  }
}

// A row's values this thread holds: NCH packs of VEC neighbours, T packs apart, as they lie in memory (a bfloat16 value of its own in a
// register of its own); what is behind the row's end is zero.
constexpr int words_of(int bytes) { return bytes < 4 ? 1 : bytes / 4; }
template <class V, int VEC, int T, int NCH, int N>
__device__ __forceinline__ void fetch_row(unsigned (&out)[NCH][N], const V* __restrict__ row, int C, int t) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * T + t) * VEC;
#pragma unroll
    for (int e = 0; e < N; ++e) out[i][e] = 0u;
    if (c >= C) continue;
    if (VEC == 1) {
      out[i][0] = to_bits(row[c]);
    } else {
      const Pack<unsigned, N> p = *(const Pack<unsigned, N>*)(row + c);
#pragma unroll
      for (int e = 0; e < N; ++e) out[i][e] = p.v[e];
    }
  }
}
// ... and their values.  (The empty assembly keeps what is done with a value behind all loads: moved up beside its load, which is under a
// condition, it makes every load wait for the one before: 8192 rows of 4096 bfloat16 values, backward, 62 us instead of 50.)
template <class V, int VEC, int NCH, int N>
__device__ __forceinline__ void unpack_row(float (&out)[NCH * VEC], unsigned (&in)[NCH][N]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) asm volatile("" : "+v"(in[i][e]));
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (VEC == 1 || sizeof(V) == 4) out[i * VEC + e] = from_bits<V>(in[i][e]);
      else out[i * VEC + e] = __builtin_bit_cast(float, e & 1 ? in[i][e / 2] & 0xffff0000u : in[i][e / 2] << 16);
    }
}
template <class V, int VEC, int T, int NCH>
__device__ __forceinline__ void load_row(float (&out)[NCH * VEC], const V* __restrict__ row, int C, int t) {
  unsigned raw[NCH][words_of(VEC * sizeof(V))];
  fetch_row<V, VEC, T, NCH>(raw, row, C, t);
  unpack_row<V, VEC, NCH>(out, raw);
}
template <class V, int VEC, int T, int NCH>
__device__ __forceinline__ void store_row(V* __restrict__ row, const float (&v)[NCH * VEC], int C, int t) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * T + t) * VEC;
    if (c >= C) continue;
    Pack<V, VEC> p;
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.v[e] = from_float<V>(v[i * VEC + e]);
    *(Pack<V, VEC>*)(row + c) = p;
  }
}

// mean and sigma of a row held by a group; the squares are taken about the mean
template <int VEC, int T, int NCH>
__device__ __forceinline__ void row_moments(const float (&x)[NCH * VEC], int C, float epsilon, int t, float2* slots, float* mu, float* sigma) {
  float s = 0.f, none = 0.f;
#pragma unroll
  for (int i = 0; i < NCH * VEC; ++i) s += x[i];
  group_sum<T>(s, none, slots);
  const float m = s / C;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = (i * T + t) * VEC < C ? x[i * VEC + e] - m : 0.f;
      q += d * d;
    }
  group_sum<T>(q, none, slots + 16);
  *mu = m;
  *sigma = sqrtf(q / C + epsilon);
}

template <class V, int VEC, int T, int NCH>
__global__ __launch_bounds__(T > 256 ? T : 256) void lnorm_rows_forward(V* __restrict__ y, float* __restrict__ moments, const V* __restrict__ x,
                                                                        const float* __restrict__ g, const float* __restrict__ b, LnP p) {
  constexpr int kThreads = T > 256 ? T : 256;
  __shared__ float2 slots[32];
  const size_t row = block_of_grid() * (kThreads / T) + threadIdx.x / T;
  const bool live = row < p.items;   // (whole groups; they stay for the barriers)
  const int t = threadIdx.x % T;
  float v[NCH * VEC];
  load_row<V, VEC, T, NCH>(v, x + (live ? row : 0) * (size_t)p.C, p.C, t);
  float mu, sigma;
  if (p.given) {
    mu = moments[live ? row : 0];
    sigma = moments[p.items + (live ? row : 0)];
  } else {
    row_moments<VEC, T, NCH>(v, p.C, p.epsilon, t, slots, &mu, &sigma);
  }
  if (!live) return;
  if (!p.given && moments && t == 0) {
    moments[row] = mu;
    moments[p.items + row] = sigma;
  }
  const float inv = 1.f / sigma;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * T + t) * VEC;
    Pack<float, VEC> pg = {}, pb = {};
    if (c < p.C) {
      if (g) pg = *(const Pack<float, VEC>*)(g + c);
      if (b) pb = *(const Pack<float, VEC>*)(b + c);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i * VEC + e] = (v[i * VEC + e] - mu) * inv * (g ? pg.v[e] : 1.f) + pb.v[e];
  }
  store_row<V, VEC, T, NCH>(y + row * (size_t)p.C, v, p.C, t);
}

// partials: [workgroups][2][C]
template <class V, int VEC, int T, int NCH>
__global__ __launch_bounds__(1024) void lnorm_rows_backward(V* __restrict__ dx, float* __restrict__ partials, float* __restrict__ moments,
                                                            const V* __restrict__ x, const float* __restrict__ g, const V* __restrict__ dy,
                                                            LnP p) {
  constexpr int kGroups = 1024 / T, W = NCH * VEC;
  __shared__ float2 slots[64];
  __shared__ float join[T * W > 1024 ? T * W : 1024];
  const int t = threadIdx.x % T, group = threadIdx.x / T;
  float scale[W], sumG[W], sumB[W];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * T + t) * VEC;
    Pack<float, VEC> pg = {};
    if (g && c < p.C) pg = *(const Pack<float, VEC>*)(g + c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) scale[i * VEC + e] = g ? pg.v[e] : 1.f;
  }
#pragma unroll
  for (int i = 0; i < W; ++i) sumG[i] = sumB[i] = 0.f;
  const size_t step = (size_t)gridDim.x * kGroups;
  int turn = 0;
  // (the next row is on its way while this one's sums are taken, where that takes barriers and the registers allow it)
  constexpr bool ahead = T > 64 && W <= 8;
  constexpr int N = words_of(VEC * sizeof(V));
  unsigned nextX[NCH][N], nextD[NCH][N];
  float nextMu = 0.f, nextSigma = 1.f;
  const auto fetch = [&](size_t row) __attribute__((always_inline)) {
    const size_t at = (row < p.items ? row : 0) * (size_t)p.C;
    fetch_row<V, VEC, T, NCH>(nextX, x + at, p.C, t);
    fetch_row<V, VEC, T, NCH>(nextD, dy + at, p.C, t);
    if (p.given) {   // (loads come back in order: these, asked for later, would wait for the next row's)
      nextMu = moments[row < p.items ? row : 0];
      nextSigma = moments[p.items + (row < p.items ? row : 0)];
    }
  };
  if (ahead) fetch((size_t)blockIdx.x * kGroups + group);
  for (size_t first = (size_t)blockIdx.x * kGroups; first < p.items; first += step) {
    const size_t row = first + group;
    const bool live = row < p.items;
    const size_t at = (live ? row : 0) * (size_t)p.C;
    if (!ahead) fetch(row);
    float v[W], d[W];
    unpack_row<V, VEC, NCH>(v, nextX);
    unpack_row<V, VEC, NCH>(d, nextD);
    float mu = nextMu, sigma = nextSigma;
    if (ahead) fetch(row + step);
    if (!p.given) {
      row_moments<VEC, T, NCH>(v, p.C, p.epsilon, t, slots, &mu, &sigma);
      if (moments && live && t == 0) {
        moments[row] = mu;
        moments[p.items + row] = sigma;
      }
    }
    const float inv = 1.f / sigma;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[i] = (v[i] - mu) * inv;   // (behind the row's end d is zero)
      const float a = d[i] * scale[i];
      s1 += a;
      s2 += a * v[i];
    }
    group_sum<T>(s1, s2, slots + 32 + 16 * turn);
    turn ^= 1;
    s1 /= p.C;
    s2 /= p.C;
    if (!live) continue;   // (nobody waits for anybody in what is left of this turn)
#pragma unroll
    for (int i = 0; i < W; ++i) {
      sumG[i] += d[i] * v[i];
      sumB[i] += d[i];
      d[i] = (d[i] * scale[i] - s1 - v[i] * s2) * inv;
    }
    if (dx) store_row<V, VEC, T, NCH>(dx + at, d, p.C, t);
  }
  if (!partials) return;
  // the groups' sums, in the order of the groups
  float* out = partials + (size_t)blockIdx.x * 2 * p.C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    for (int k = 0; k < kGroups; ++k) {
      __syncthreads();
      if (group == k) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float mine = which ? sumB[i] : sumG[i];
          join[i * T + t] = k ? join[i * T + t] + mine : mine;
        }
      }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int c = ((i / VEC) * T + t) * VEC + i % VEC;
        if (c < p.C) out[which * p.C + c] = join[i * T + t];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- planes

__device__ __forceinline__ size_t pixel_base(size_t item, const LnP& p) {
  const size_t n = item / p.HW;
  return n * (size_t)p.HW * p.C + (item - n * p.HW);
}

// Sixteen wavefronts; a wavefront's lanes are PIX pixels (64, 32 or 16) times 64 / PIX channels, so that a thread holds K = 16 channels at
// most: channel (k 16 + wave) (64 / PIX) + lane / PIX of pixel lane % PIX.
constexpr int kPlaneWaves = 16;
template <int PIX>
__device__ __forceinline__ int plane_channel(int k, int wave, int lane) { return (k * kPlaneWaves + wave) * (64 / PIX) + lane / PIX; }

// sums over a pixel's lanes of all wavefronts
template <int PIX>
__device__ __forceinline__ void pixel_sum(float& a, float& b, float2* slots, int wave, int lane) {
#pragma unroll
  for (int o = 32; o >= PIX; o >>= 1) {
    a += __shfl_xor(a, o, kWave);
    b += __shfl_xor(b, o, kWave);
  }
  if (lane < PIX) slots[wave * PIX + lane] = make_float2(a, b);
  lds_barrier();
  a = b = 0.f;
#pragma unroll
  for (int w = 0; w < kPlaneWaves; ++w) {
    const float2 s = slots[w * PIX + lane % PIX];
    a += s.x;
    b += s.y;
  }
}

template <int PIX, int K>
__device__ __forceinline__ void pixel_moments(const float (&v)[K], int C, float epsilon, float2* slots, int wave, int lane, float* mu, float* sigma) {
  float s = 0.f, none = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) s += v[k];
  pixel_sum<PIX>(s, none, slots, wave, lane);
  const float m = s / C;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float d = plane_channel<PIX>(k, wave, lane) < C ? v[k] - m : 0.f;
    q += d * d;
  }
  pixel_sum<PIX>(q, none, slots + kPlaneWaves * PIX, wave, lane);
  *mu = m;
  *sigma = sqrtf(q / C + epsilon);
}

template <class V, int PIX, int K>
__global__ __launch_bounds__(64 * kPlaneWaves) void lnorm_planes_forward(V* __restrict__ y, float* __restrict__ moments, const V* __restrict__ x,
                                                                         const float* __restrict__ g, const float* __restrict__ b, LnP p) {
  __shared__ float2 slots[2 * kPlaneWaves * PIX];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const size_t item = block_of_grid() * PIX + lane % PIX;
  const bool live = item < p.items;
  const size_t base = pixel_base(live ? item : 0, p);
  float v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = plane_channel<PIX>(k, wave, lane);
    v[k] = to_float(x[base + (size_t)min(c, p.C - 1) * p.HW]);
    if (c >= p.C) v[k] = 0.f;
  }
  float mu, sigma;
  if (p.given) {
    mu = moments[live ? item : 0];
    sigma = moments[p.items + (live ? item : 0)];
  } else {
    pixel_moments<PIX, K>(v, p.C, p.epsilon, slots, wave, lane, &mu, &sigma);
  }
  if (!live) return;
  if (!p.given && moments && wave == 0 && lane < PIX) {
    moments[item] = mu;
    moments[p.items + item] = sigma;
  }
  const float inv = 1.f / sigma;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = plane_channel<PIX>(k, wave, lane);
    if (c < p.C) y[base + (size_t)c * p.HW] = from_float<V>((v[k] - mu) * inv * (g ? g[c] : 1.f) + (b ? b[c] : 0.f));
  }
}

template <class V, int PIX, int K>
__global__ __launch_bounds__(64 * kPlaneWaves) void lnorm_planes_backward(V* __restrict__ dx, float* __restrict__ partials, float* __restrict__ moments,
                                                                          const V* __restrict__ x, const float* __restrict__ g,
                                                                          const V* __restrict__ dy, LnP p) {
  __shared__ float2 slots[4 * kPlaneWaves * PIX];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  float sumG[K], sumB[K];
#pragma unroll
  for (int k = 0; k < K; ++k) sumG[k] = sumB[k] = 0.f;
  int turn = 0;
  // (the next pixels are on their way while these ones' sums are taken, where the registers allow it)
  constexpr bool ahead = K <= 8;
  // (a register each, also where two would fit one: loads into halves of registers wait for each other)
  unsigned nextX[K], nextD[K];
  float nextMu = 0.f, nextSigma = 1.f;
  const auto fetch = [&](size_t item) __attribute__((always_inline)) {
    const bool live = item < p.items;
    const size_t base = pixel_base(live ? item : 0, p);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = plane_channel<PIX>(k, wave, lane);
      const size_t at = base + (size_t)min(c, p.C - 1) * p.HW;
      nextX[k] = to_bits(x[at]);
      nextD[k] = to_bits(dy[at]);
    }
    if (p.given) {
      nextMu = moments[live ? item : 0];
      nextSigma = moments[p.items + (live ? item : 0)];
    }
  };
  if (ahead) fetch((size_t)blockIdx.x * PIX + lane % PIX);
  for (size_t first = (size_t)blockIdx.x * PIX; first < p.items; first += (size_t)gridDim.x * PIX) {
    const size_t item = first + lane % PIX;
    const bool live = item < p.items;
    const size_t base = pixel_base(live ? item : 0, p);
    if (!ahead) fetch(item);
    float v[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool there = plane_channel<PIX>(k, wave, lane) < p.C;
      v[k] = there ? from_bits<V>(nextX[k]) : 0.f;
      d[k] = there && live ? from_bits<V>(nextD[k]) : 0.f;
    }
    float mu = nextMu, sigma = nextSigma;
    if (ahead) fetch(item + (size_t)gridDim.x * PIX);
    if (!p.given) {
      pixel_moments<PIX, K>(v, p.C, p.epsilon, slots, wave, lane, &mu, &sigma);
      if (moments && live && wave == 0 && lane < PIX) {
        moments[item] = mu;
        moments[p.items + item] = sigma;
      }
    }
    const float inv = 1.f / sigma;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = plane_channel<PIX>(k, wave, lane);
      v[k] = (v[k] - mu) * inv;
      const float a = c < p.C && g ? d[k] * g[c] : d[k];
      s1 += a;
      s2 += c < p.C ? a * v[k] : 0.f;
    }
    pixel_sum<PIX>(s1, s2, slots + (2 + turn) * kPlaneWaves * PIX, wave, lane);
    turn ^= 1;
    s1 /= p.C;
    s2 /= p.C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = plane_channel<PIX>(k, wave, lane);
      if (c >= p.C) continue;
      if (live) sumG[k] += d[k] * v[k];   // (a pixel behind the last may hold anything)
      sumB[k] += d[k];
      if (dx && live) dx[base + (size_t)c * p.HW] = from_float<V>((d[k] * (g ? g[c] : 1.f) - s1 - v[k] * s2) * inv);
    }
  }
  if (!partials) return;
  float* out = partials + (size_t)blockIdx.x * 2 * p.C;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = plane_channel<PIX>(k, wave, lane);
    float a = sumG[k], e = sumB[k];
#pragma unroll
    for (int o = PIX / 2; o > 0; o >>= 1) {
      a += __shfl_xor(a, o, kWave);
      e += __shfl_xor(e, o, kWave);
    }
    if (lane % PIX == 0 && c < p.C) {
      out[c] = a;
      out[p.C + c] = e;
    }
  }
}

// ---------------------------------------------------------------------------------------------- any number of channels

// Rows: a workgroup per pixel, threads along the channels.  Planes: a lane per pixel, four wavefronts share the channels.
template <bool ROWS>
__device__ __forceinline__ void long_sum(float& a, float& b, float2* slots) {
  if (ROWS) {
    group_sum<256>(a, b, slots);
  } else {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    slots[wave * 64 + lane] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 s = slots[w * 64 + lane];
      a += s.x;
      b += s.y;
    }
  }
  __syncthreads();
}

// Sums of two terms over a thread's channels c0, c0 + cs, ...: kLongStep of them at a time (their loads go out together), single precision
// among these, in double one step behind the other, so that the sums are off by no more than those of few channels are (a thread of
// "planes" has a quarter of all channels: added one by one in single precision, 20000 values of 0.1 had a mean off by 4e-5 of itself).
constexpr int kLongStep = 16;
template <class F>
__device__ __forceinline__ void walk_channels(int c0, int cs, int C, float& a, float& b, F term) {
  double sa = 0.0, sb = 0.0;
  for (long long first = c0; first < C; first += (long long)kLongStep * cs) {
    float pa = 0.f, pb = 0.f;
#pragma unroll
    for (int k = 0; k < kLongStep; ++k) {
      const long long c = first + (long long)k * cs;
      const float2 t = term(c < C ? (int)c : c0);
      pa += c < C ? t.x : 0.f;
      pb += c < C ? t.y : 0.f;
    }
    sa += (double)pa;
    sb += (double)pb;
  }
  a = (float)sa;
  b = (float)sb;
}

template <class V, bool ROWS, bool BACKWARD>
__global__ __launch_bounds__(256) void lnorm_long(V* __restrict__ out, float* __restrict__ moments, const V* __restrict__ x,
                                                  const float* __restrict__ g, const float* __restrict__ b, const V* __restrict__ dy, LnP p) {
  __shared__ float2 slots[256];
  const size_t item = ROWS ? block_of_grid() : block_of_grid() * 64 + (threadIdx.x & 63);
  const bool live = item < p.items;
  const size_t base = ROWS ? (live ? item : 0) * p.C : pixel_base(live ? item : 0, p), step = ROWS ? 1 : p.HW;
  const int c0 = ROWS ? threadIdx.x : threadIdx.x >> 6, cs = ROWS ? 256 : 4;
  float mu, sigma, none = 0.f;
  if (p.given) {
    mu = moments[live ? item : 0];
    sigma = moments[p.items + (live ? item : 0)];
  } else {
    float s, q;
    walk_channels(c0, cs, p.C, s, none, [&](int c) { return make_float2(to_float(x[base + c * step]), 0.f); });
    long_sum<ROWS>(s, none, slots);
    mu = s / p.C;
    walk_channels(c0, cs, p.C, q, none, [&](int c) {
      const float d = to_float(x[base + c * step]) - mu;
      return make_float2(d * d, 0.f);
    });
    long_sum<ROWS>(q, none, slots);
    sigma = sqrtf(q / p.C + p.epsilon);
    if (moments && live && c0 == 0) {
      moments[item] = mu;
      moments[p.items + item] = sigma;
    }
  }
  const float inv = 1.f / sigma;
  if (!BACKWARD) {
    if (live)
      for (int c = c0; c < p.C; c += cs)
        out[base + c * step] = from_float<V>((to_float(x[base + c * step]) - mu) * inv * (g ? g[c] : 1.f) + (b ? b[c] : 0.f));
    return;
  }
  if (!out) return;   // (only the moments were wanted)
  float s1, s2;
  walk_channels(c0, cs, p.C, s1, s2, [&](int c) {
    const float a = to_float(dy[base + c * step]) * (g ? g[c] : 1.f);
    return make_float2(a, a * ((to_float(x[base + c * step]) - mu) * inv));
  });
  long_sum<ROWS>(s1, s2, slots);
  s1 /= p.C;
  s2 /= p.C;
  if (live)
    for (int c = c0; c < p.C; c += cs) {
      const float v = (to_float(x[base + c * step]) - mu) * inv;
      out[base + c * step] = from_float<V>((to_float(dy[base + c * step]) * (g ? g[c] : 1.f) - s1 - v * s2) * inv);
    }
}

// Partial sums of dzdg and dzdb from stored moments.  Rows: a thread per channel; planes: a workgroup per channel; blockIdx.z a run of pixels.
template <class V, bool ROWS>
__global__ __launch_bounds__(256) void lnorm_long_sums(float* __restrict__ partials, const float* __restrict__ moments, const V* __restrict__ x,
                                                       const V* __restrict__ dy, LnP p, size_t run) {
  const size_t first = (size_t)blockIdx.z * run, last = std::min(first + run, p.items);
  float a = 0.f, b = 0.f;
  size_t c;
  if (ROWS) {
    c = block_of_grid() * 256 + threadIdx.x;
    if (c >= (size_t)p.C) return;
    for (size_t i = first; i < last; ++i) {
      const float d = to_float(dy[i * p.C + c]);
      a += d * ((to_float(x[i * p.C + c]) - moments[i]) / moments[p.items + i]);
      b += d;
    }
  } else {
    __shared__ float2 slots[16];
    c = block_of_grid();
    if (c >= (size_t)p.C) return;   // (whole workgroups)
    for (size_t i = first + threadIdx.x; i < last; i += 256) {
      const size_t at = pixel_base(i, p) + c * p.HW;
      const float d = to_float(dy[at]);
      a += d * ((to_float(x[at]) - moments[i]) / moments[p.items + i]);
      b += d;
    }
    group_sum<256>(a, b, slots);
    if (threadIdx.x) return;
  }
  float* out = partials + (size_t)blockIdx.z * 2 * p.C;
  out[c] = a;
  out[p.C + c] = b;
}

// dzdg and dzdb from the workgroups' partial sums: 32 of the 2 C sums per workgroup, eight threads each, in double, in a fixed order
__global__ __launch_bounds__(256) void lnorm_join(float* __restrict__ dg, float* __restrict__ db, const float* __restrict__ partials, int C, int parts) {
  __shared__ double slots[8][33];
  const int t = threadIdx.x & 31, r = threadIdx.x >> 5;
  const size_t c = (size_t)blockIdx.x * 32 + t;
  double s = 0.0;
  if (c < 2 * (size_t)C) {
    int k = r;
    for (; k + 56 < parts; k += 64) {   // eight loads at a time
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = partials[(size_t)(k + 8 * i) * 2 * C + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (double)v[i];
    }
    for (; k < parts; k += 8) s += (double)partials[(size_t)k * 2 * C + c];
  }
  slots[r][t] = s;
  __syncthreads();
  if (r || c >= 2 * (size_t)C) return;
  for (int k = 1; k < 8; ++k) s += slots[k][t];
  float* out = c < (size_t)C ? dg : db;
  if (out) out[c < (size_t)C ? c : c - C] = (float)s;
}

// ---------------------------------------------------------------------------------------------- host

constexpr int kMostRow = 16384, kMostPlane = 1024;   // channels that a workgroup of 1024 holds, 16 a thread
constexpr int kRuns = 256;                          // runs of pixels in lnorm_long_sums

bool in_registers(int C, size_t HW) { return HW == 1 ? C <= kMostRow : C <= kMostPlane; }

// threads that share a row in the backward pass
int backward_group(int C) { return C <= 128 ? 16 : C <= 512 ? 64 : C <= 1024 ? 128 : C <= 2048 ? 256 : C <= 4096 ? 512 : 1024; }

// workgroups of a backward pass that sums as it goes: one per compute unit, and no more than there is work for
int backward_groups(int C, size_t HW, size_t items) {
  const size_t cus = std::max(1, device_compute_units());
  const size_t per = HW == 1 ? 1024 / backward_group(C) : C <= 256 ? 64 : C <= 512 ? 32 : 16;
  return (int)std::max<size_t>(1, std::min(cus, (items + per - 1) / per));
}

struct LnArgs {
  void* out;
  float *partials, *moments;
  const void* x;
  const float *g, *b;
  const void* dy;
  LnP p;
  int groups;
};

template <class V, int VEC, int T, int NCH>
void launch_rows(hipStream_t s, const LnArgs& a, bool backward) {
  if (backward)
    hipLaunchKernelGGL((lnorm_rows_backward<V, VEC, T, NCH>), dim3((unsigned)a.groups), dim3(1024), 0, s, (V*)a.out, a.partials, a.moments,
                       (const V*)a.x, a.g, (const V*)a.dy, a.p);
  else
    hipLaunchKernelGGL((lnorm_rows_forward<V, VEC, T, NCH>), grid_of((a.p.items * T + (T > 256 ? T : 256) - 1) / (T > 256 ? T : 256)),
                       dim3(T > 256 ? T : 256), 0, s, (V*)a.out, a.moments, (const V*)a.x, a.g, a.b, a.p);
}

// Forward, the narrowest group that holds a row with 16 values a thread; backward, with 8 (16 and the sums beside them take more registers
// than 1024 threads have: 8192 rows of 4096 single-precision values 90 us with 16, 81 with 8); and the fewest packs.
template <class V, int VEC, int T>
void choose_packs(hipStream_t s, const LnArgs& a, bool backward) {
  const int packs = div_up(a.p.C, T * VEC);
  if (packs <= 1) launch_rows<V, VEC, T, 1>(s, a, backward);
  else if (16 / VEC > 1 && packs <= 2) launch_rows<V, VEC, T, 16 / VEC >= 2 ? 2 : 1>(s, a, backward);
  else if (16 / VEC > 2 && packs <= 4) launch_rows<V, VEC, T, 16 / VEC >= 4 ? 4 : 1>(s, a, backward);
  else if (16 / VEC > 4 && packs <= 8) launch_rows<V, VEC, T, 16 / VEC >= 8 ? 8 : 1>(s, a, backward);
  else launch_rows<V, VEC, T, 16 / VEC>(s, a, backward);
}
template <class V, int VEC>
void choose_group(hipStream_t s, const LnArgs& a, bool backward) {
  const int C = a.p.C;
  if (backward) {
    switch (backward_group(C)) {
      case 16: return choose_packs<V, VEC, 16>(s, a, true);
      case 64: return choose_packs<V, VEC, 64>(s, a, true);
      case 128: return choose_packs<V, VEC, 128>(s, a, true);
      case 256: return choose_packs<V, VEC, 256>(s, a, true);
      case 512: return choose_packs<V, VEC, 512>(s, a, true);
      default: return choose_packs<V, VEC, 1024>(s, a, true);
    }
  }
  if (C <= 64) choose_packs<V, VEC, 16>(s, a, false);
  else if (C <= 1024) choose_packs<V, VEC, 64>(s, a, false);
  else if (C <= 4096) choose_packs<V, VEC, 256>(s, a, false);
  else choose_packs<V, VEC, 1024>(s, a, false);
}

template <class V, int PIX, int K>
void launch_planes(hipStream_t s, const LnArgs& a, bool backward) {
  const dim3 block(64 * kPlaneWaves);
  if (backward)
    hipLaunchKernelGGL((lnorm_planes_backward<V, PIX, K>), dim3((unsigned)a.groups), block, 0, s, (V*)a.out, a.partials, a.moments, (const V*)a.x, a.g,
                       (const V*)a.dy, a.p);
  else
    hipLaunchKernelGGL((lnorm_planes_forward<V, PIX, K>), grid_of((a.p.items + PIX - 1) / PIX), block, 0, s, (V*)a.out, a.moments, (const V*)a.x,
                       a.g, a.b, a.p);
}

template <class V>
int launch(hipStream_t s, const char* who, LnArgs& a, bool backward, float* dg, float* db) {
  constexpr int VEC = 16 / sizeof(V);
  const bool rows = a.p.HW == 1;
  if (in_registers(a.p.C, a.p.HW)) {
    KernelTimer timer(backward ? "lnorm_backward" : "lnorm_forward", s);
    if (rows) {
      const bool wide = a.p.C % VEC == 0 && aligned16(a.x) && aligned16(a.out) && aligned16(a.dy) && aligned16(a.g) && aligned16(a.b);
      if (wide) choose_group<V, VEC>(s, a, backward);
      else choose_group<V, 1>(s, a, backward);
    } else {
      if (a.p.C <= 64) launch_planes<V, 64, 4>(s, a, backward);
      else if (a.p.C <= 128) launch_planes<V, 64, 8>(s, a, backward);
      else if (a.p.C <= 256) launch_planes<V, 64, 16>(s, a, backward);
      else if (a.p.C <= 512) launch_planes<V, 32, 16>(s, a, backward);
      else launch_planes<V, 16, 16>(s, a, backward);
    }
  } else {
    KernelTimer timer(backward ? "lnorm_backward" : "lnorm_forward", s);
    const dim3 grid = grid_of(rows ? a.p.items : (a.p.items + 63) / 64), block(256);
    if (!backward) {
      if (rows) hipLaunchKernelGGL((lnorm_long<V, true, false>), grid, block, 0, s, (V*)a.out, a.moments, (const V*)a.x, a.g, a.b, (const V*)a.dy, a.p);
      else hipLaunchKernelGGL((lnorm_long<V, false, false>), grid, block, 0, s, (V*)a.out, a.moments, (const V*)a.x, a.g, a.b, (const V*)a.dy, a.p);
    } else {
      if (rows) hipLaunchKernelGGL((lnorm_long<V, true, true>), grid, block, 0, s, (V*)a.out, a.moments, (const V*)a.x, a.g, a.b, (const V*)a.dy, a.p);
      else hipLaunchKernelGGL((lnorm_long<V, false, true>), grid, block, 0, s, (V*)a.out, a.moments, (const V*)a.x, a.g, a.b, (const V*)a.dy, a.p);
      if (a.partials) {
        const size_t run = (a.p.items + a.groups - 1) / a.groups;
        dim3 sums = grid_of(rows ? div_up(a.p.C, 256) : a.p.C);
        sums.z = (unsigned)a.groups;
        if (rows) hipLaunchKernelGGL((lnorm_long_sums<V, true>), sums, block, 0, s, a.partials, a.moments, (const V*)a.x, (const V*)a.dy, a.p, run);
        else hipLaunchKernelGGL((lnorm_long_sums<V, false>), sums, block, 0, s, a.partials, a.moments, (const V*)a.x, (const V*)a.dy, a.p, run);
      }
    }
  }
  int rc = check_launch(who);
  if (rc || !backward || !a.partials) return rc;
  KernelTimer timer("lnorm_join", s);
  hipLaunchKernelGGL(lnorm_join, dim3((unsigned)div_up(2ll * a.p.C, 32)), dim3(256), 0, s, dg, db, a.partials, a.p.C, a.groups);
  return check_launch(who);
}

int setup(const char* who, int dataType, int H, int W, int C, int N, double epsilon, int given, LnP* p) {
  if (dataType != MCN_FLOAT && dataType != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d", who, dataType);
  if (H < 0 || W < 0 || C < 0 || N < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative tensor extent", who);
  if (!(epsilon >= 0)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: EPSILON is negative", who);
  if ((long long)H * W >= (1ll << 31)) return fail(MCN_UNSUPPORTED, "%s: plane too large", who);
  if (C > (1 << 24) || (size_t)H * W * N >= (1ull << 31)) return fail(MCN_UNSUPPORTED, "%s: tensor too large", who);
  p->C = C;
  p->HW = H * W;
  p->items = (size_t)H * W * N;
  p->epsilon = (float)epsilon;
  p->given = given != 0;
  return MCN_SUCCESS;
}

int long_groups(size_t items) { return (int)std::max<size_t>(1, std::min<size_t>(kRuns, items)); }

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_lnorm_workspace_bytes(int H, int W, int C, int N) {
  if (H <= 0 || W <= 0 || C <= 0 || N <= 0) return 0;
  const size_t items = (size_t)H * W * N;
  const bool regs = in_registers(C, (size_t)H * W);
  const size_t groups = regs ? backward_groups(C, (size_t)H * W, items) : long_groups(items);
  return groups * 2 * C * sizeof(float) + (regs ? 0 : 2 * items * sizeof(float));
}

int mcn_lnorm_forward(mcn_stream_t stream, int dataType, void* y, float* moments, const void* x, const float* multipliers, const float* biases, int H,
                      int W, int C, int N, double epsilon, int givenMoments) {
  const char* who = "mcn_lnorm_forward";
  LnArgs a = {};
  int rc = setup(who, dataType, H, W, C, N, epsilon, givenMoments, &a.p);
  if (rc || a.p.items == 0 || C == 0) return rc;
  if (!y || !x) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  if (givenMoments && !moments) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null moments", who);
  a.out = y; a.moments = moments; a.x = x; a.g = multipliers; a.b = biases;
  hipStream_t s = as_stream(stream);
  return dataType == MCN_BFLOAT16 ? launch<bf16>(s, who, a, false, nullptr, nullptr) : launch<float>(s, who, a, false, nullptr, nullptr);
}

int mcn_lnorm_backward(mcn_stream_t stream, int dataType, void* derInput, float* derMultipliers, float* derBiases, float* moments, const void* x,
                       const float* multipliers, const void* derOutput, int H, int W, int C, int N, double epsilon, int givenMoments, void* workspace,
                       size_t workspaceBytes) {
  const char* who = "mcn_lnorm_backward";
  LnArgs a = {};
  int rc = setup(who, dataType, H, W, C, N, epsilon, givenMoments, &a.p);
  if (rc || C == 0 || (!derInput && !derMultipliers && !derBiases && !moments)) return rc;
  hipStream_t s = as_stream(stream);
  const bool sums = derMultipliers || derBiases;
  if (a.p.items == 0) {   // no pixels: the sums over them are zero
    if (!sums) return MCN_SUCCESS;
    hipLaunchKernelGGL(lnorm_join, dim3((unsigned)div_up(2ll * C, 32)), dim3(256), 0, s, derMultipliers, derBiases, (const float*)nullptr, C, 0);
    return check_launch(who);
  }
  if (!x || !derOutput) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  if (givenMoments && !moments) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null moments", who);
  const size_t need = mcn_lnorm_workspace_bytes(H, W, C, N);
  if (!workspace || workspaceBytes < need)
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, need);
  if ((uintptr_t)workspace & 3) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the workspace is not 4-byte aligned", who);
  a.out = derInput; a.moments = moments; a.x = x; a.g = multipliers; a.dy = derOutput;
  a.partials = sums ? (float*)workspace : nullptr;
  const bool regs = in_registers(C, a.p.HW);
  a.groups = regs ? backward_groups(C, a.p.HW, a.p.items) : long_groups(a.p.items);
  if (!regs && !moments) a.moments = (float*)workspace + (size_t)a.groups * 2 * C;   // (the sums read them back)
  return dataType == MCN_BFLOAT16 ? launch<bf16>(s, who, a, true, derMultipliers, derBiases) : launch<float>(s, who, a, true, derMultipliers, derBiases);
}

}  // extern "C"
