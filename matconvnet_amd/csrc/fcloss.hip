// A fully connected layer and the softmax cross entropy behind it as one operator: the scores of N instances for K classes are made in
// pieces of the classes and never kept.
//
//   z = x f + b, y = sum_n w_n (log sum_k exp z_nk - z_n,c(n)) [/ N],  P = softmax(z) - (1 at c(n)),
//   dzdx = sum_k w P f, dzdf = sum_n w P x, dzdb = sum_n w P   (times the scalar derivative of y [/ N])
//
// Forward: every tile of scores leaves, per instance, its largest score and the sum of exponentials against it; a pass over those
// (N x K / 256 pairs) gives the logarithms of the sums.  Backward: a piece of the classes at a time, the scores are made
// again, P is written as 16-bit operands, and two products over it give the piece's dzdf and its share of dzdx.  The largest
// buffer is the piece's P.  8 N D K operations in all, a quarter of them the scores made again: keeping N x K scores is
// what this operator is there to avoid.
#include "product.hpp"

#include <algorithm>

namespace mcn {
namespace {

struct FcP {
  int D, K, N, type;           // type: kPairs (single precision) or kBf16
  int nWeights;
  float factor;                // of all derivatives: derOutput / N or derOutput
};

__device__ __forceinline__ float instance_weight(const float* labels, const float* weights, int nWeights, int n) {
  return labels[n] != 0.f ? (weights ? weights[n % nWeights] : 1.f) : 0.f;
}
__device__ __forceinline__ int class_of(float label, int K) { return label >= 1.f ? min((int)fminf(label, 2147483520.f) - 1, K - 1) : 0; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}

// ---------------------------------------------------------------------------------------------- operands

// The largest magnitude of n values, as the bits of a float (whole numbers: the order of the atomics does not matter; a NaN or an
// infinity wins, and pair_scale leaves such a tensor as it is)
__device__ __forceinline__ unsigned magnitude4(uintx4p v) {
  return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
}
__device__ __forceinline__ unsigned wave_most(unsigned m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, kWave));
  return m;
}
constexpr int kMagnitudeStep = 256 * 4 * 8;   // values of a workgroup
__global__ __launch_bounds__(256) void fc_magnitude(unsigned* __restrict__ bits, const float* __restrict__ x, size_t n, int vec) {
  __shared__ unsigned lds[4];
  unsigned m = 0;
  const size_t first = (size_t)blockIdx.x * kMagnitudeStep;
  if (vec && first + kMagnitudeStep <= n) {
    const uintx4p* x4 = (const uintx4p*)(x + first) + threadIdx.x;
    uintx4p v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x4[256 * i];
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude4(v[i]));
  } else {
    for (size_t i = first + threadIdx.x; i < std::min(first + kMagnitudeStep, n); i += 256) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  }
  m = wave_most(m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) atomicMax(bits, max(max(lds[0], lds[1]), max(lds[2], lds[3])));
}

// the magnitudes, and the products' counters behind them
__global__ __launch_bounds__(256) void fc_clear(unsigned* p, int n) {
  for (int i = threadIdx.x; i < n; i += 256) p[i] = 0;
}

// (K D / 1024 workgroups: at most 2^34)
__global__ __launch_bounds__(256) void fc_zero(void* __restrict__ p, size_t n, int is16) {
  const size_t first = (size_t)blockIdx.x * 1024 + threadIdx.x;
  for (size_t i = first; i < std::min(first + 1024, n); i += 256) {
    if (is16) ((unsigned short*)p)[i] = 0;
    else ((float*)p)[i] = 0.f;
  }
}

// Rows of single-precision values as pairs, each by its own largest magnitude: 1 / scale in unscale[row]; the largest magnitude of all
// rows times their instances' weights in `all` (not null).  A wavefront per row.
__global__ __launch_bounds__(256) void fc_pack_rows(unsigned short* __restrict__ out, float* __restrict__ unscale, unsigned* __restrict__ all,
                                                    const float* __restrict__ x, int D, int rows, long long pitch, const float* __restrict__ labels,
                                                    const float* __restrict__ weights, int nWeights, int wide) {
  const int row = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const float* from = x + (size_t)row * D;
  unsigned m = 0;
  float v[8];
  for (int c = 8 * lane; c < D; c += 512) {
    load8(v, from, c, D, wide);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  }
  m = wave_most(m);
  const float scale = pair_scale(m);
  if (lane == 0) {
    unscale[row] = pair_unscale(m);
    const float w = all ? instance_weight(labels, weights, nWeights, row) : 0.f;
    if (w != 0.f) atomicMax(all, __float_as_uint(fabsf(__uint_as_float(m) * w)));
  }
  for (int c = 8 * lane; c < pitch / 2; c += 512) {
    load8(v, from, c, D, wide);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= scale;
    store8_pairs(out + (size_t)row * pitch, c, v);
  }
}

// Rows as the operand of a product: single precision as pairs by the tensor's magnitude, bfloat16 at a pitch of whole stages.  With
// labels, times the instance's weight, and zeros for instances that do not count, whatever they hold.  A thread per eight
// values.
template <int TYPE>
__global__ __launch_bounds__(256) void fc_pack(unsigned short* __restrict__ out, const unsigned* __restrict__ magnitude, const void* __restrict__ x,
                                               int D, int rows, long long pitch, const float* __restrict__ labels, const float* __restrict__ weights,
                                               int nWeights, int wide) {
  const int per = (int)(pitch / (TYPE == kPairs ? 16 : 8));
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)rows * per) return;
  const int row = (int)(i / per), c = (int)(i - (size_t)row * per) * 8;
  const float w = labels ? instance_weight(labels, weights, nWeights, row) : 1.f;
  float v[8] = {};
  if (TYPE == kPairs) {
    const float scale = pair_scale(*magnitude);
    if (w != 0.f) load8(v, (const float*)x + (size_t)row * D, c, D, wide);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = w != 0.f ? v[k] * w * scale : 0.f;
    store8_pairs(out + (size_t)row * pitch, c, v);
  } else {
    if (w != 0.f) load8(v, (const unsigned short*)x + (size_t)row * D, c, D, wide);
    uintx4p h;
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = (unsigned)to_bf16(v[2 * k] * w) | (unsigned)to_bf16(v[2 * k + 1] * w) << 16;
    if (w == 0.f) h = (uintx4p){0, 0, 0, 0};
    *(uintx4p*)(out + (size_t)row * pitch + c) = h;
  }
}

// ---------------------------------------------------------------------------------------------- products

// What the scores need: z = acc * unscale[m] * 1/scale(filters) + bias[n], -infinity behind the piece's last class
struct Scores {
  const float *unscale, *bias;     // unscale: null for bfloat16
  const unsigned* magnitude;       // of the filters
  int N, K, first;                 // instances, classes in this piece, the piece's first class
  template <class S>
  __device__ __forceinline__ void make(floatx16p (&acc)[S::TM][S::TN], int m0, int n0, int tileEnd) const {
    if (unscale) {
      const float f = pair_unscale(*magnitude);
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        // (both are powers of two: one product, kept from infinity, where the sums are nothing but zeros or past the range)
        const float u = fminf(unscale[min(m0 + 32 * i, N - 1)] * f, 3.0e38f);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] *= u;
      }
    }
    if (bias) {
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = n0 + 32 * j + 8 * (r / 4) + r % 4;
          const float b = n < K ? bias[first + n] : 0.f;
#pragma unroll
          for (int i = 0; i < S::TM; ++i) acc[i][j][r] += b;
        }
    }
    if (tileEnd > K) {             // (the last column of tiles alone)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (n0 + 32 * j + 8 * (r / 4) + r % 4 >= K) {
#pragma unroll
            for (int i = 0; i < S::TM; ++i) acc[i][j][r] = -__builtin_inff();
          }
    }
  }
};
// whether column c (against a lane's first one) is among the lane's: of a block of 32, eight times four from 4 (lane / 32) on
template <class S>
__device__ __forceinline__ bool has_column(int c) { return c >= 0 && c < 32 * S::TN && (c & 4) == 0; }

// Forward: (largest score, sum of exponentials against it) per instance and tile, the score of the instance's class
struct StatsEnd {
  Scores z;
  float2* parts;                   // [N][tiles]
  float* own;                      // [N]
  const float* labels;
  int tiles, firstTile, classes;   // of all pieces
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
    z.make<S>(acc, m0, n0, (tn + 1) * S::BN);
    float2* rows = (float2*)lds;   // [WN][BM]
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m = m0 + 32 * i;
      const int c = m < z.N ? class_of(labels[m], classes) - z.first - n0 : -1;
      if (__any(has_column<S>(c) && n0 + c < z.K)) {   // (few tiles have the class of one of their instances)
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (c == 32 * j + 8 * (r / 4) + r % 4 && n0 + c < z.K) own[m] = acc[i][j][r];
      }
      float most = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, acc[i][j][r]);
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      const float from = most == -__builtin_inff() ? 0.f : most;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __expf(acc[i][j][r] - from);
      sum += __shfl_xor(sum, 32, kWave);
      if (lane < 32) rows[wn * S::BM + 32 * (wm * S::TM + i) + lane] = make_float2(most, sum);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < S::BM; t += S::threads) {
      const int m = tm * S::BM + t;
      if (m >= z.N) continue;
      float most = rows[t].x;
#pragma unroll
      for (int w = 1; w < S::WN; ++w) most = fmaxf(most, rows[w * S::BM + t].x);
      const float from = most == -__builtin_inff() ? 0.f : most;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < S::WN; ++w) sum += rows[w * S::BM + t].y * __expf(rows[w * S::BM + t].x - from);
      parts[(size_t)m * tiles + firstTile + tn] = make_float2(most, sum);
    }
  }
};

constexpr float kProbability = 16384.f;   // P as pairs: in [-1, 1], by 2^14

// Sums over the 32 lanes of a half-wavefront of N values a lane (N a power of two, at most 32): lane l of the half ends up with the sum of
// value l % N.  Every exchange halves what is left to add: 31 exchanges for 32 values, where adding each across takes 160.
template <int N>
__device__ __forceinline__ float lanes_fold(float (&v)[N], int lane) {
#pragma unroll
  for (int h = N / 2; h >= 1; h >>= 1) {
#pragma unroll
    for (int k = 0; k < h; ++k) {
      const bool upper = (lane & h) != 0;
      const float give = upper ? v[k] : v[k + h], keep = upper ? v[k + h] : v[k];
      v[k] = keep + __shfl_xor(give, h, kWave);
    }
  }
  float s = v[0];
#pragma unroll
  for (int o = N; o < 32; o <<= 1) s += __shfl_xor(s, o, kWave);
  return s;
}

// Backward: P as the operand of two products (the instances' weights go into the other operand, or the result), and the columns' sums of
// w P before it is rounded, one per tile.
struct ProbabilitiesEnd {
  Scores z;
  unsigned short* out;
  long long pitch;
  const float *labels, *weights, *logSums;
  int nWeights, classes;
  float* sums;                     // [tile rows][classes]; may be null
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
    z.make<S>(acc, m0, n0, (tn + 1) * S::BN);
    float* columns = (float*)lds;  // [WM][BN]
    float weight[S::TM];
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m = m0 + 32 * i;
      const bool live = m < z.N;
      const float w = live ? instance_weight(labels, weights, nWeights, m) : 0.f;
      const float lse = live ? logSums[m] : 0.f;
      const int c = live ? class_of(labels[m], classes) - z.first - n0 : -1;
      weight[i] = w;
      // (classes behind the piece's last one have a score of -infinity: 0)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = __expf(acc[i][j][r] - lse);
      if (__any(has_column<S>(c) && n0 + c < z.K)) {
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (c == 32 * j + 8 * (r / 4) + r % 4 && n0 + c < z.K) acc[i][j][r] -= 1.f;
      }
      if (__any(w == 0.f)) {       // (such an instance's scores may be anything)
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = w == 0.f ? 0.f : acc[i][j][r];
      }
    }
    if (sums) {
      // value v of a block's 16: column 8 (v / 4) + v % 4 (+ 4 in the upper half-wavefront)
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          v[r] = 0.f;
#pragma unroll
          for (int i = 0; i < S::TM; ++i) v[r] += weight[i] * acc[i][j][r];
        }
        const float s = lanes_fold<16>(v, lane);
        const int r = lane & 15;
        if ((lane & 16) == 0) columns[wm * S::BN + 32 * (wn * S::TN + j) + 8 * (r / 4) + 4 * (lane >> 5) + r % 4] = s;
      }
      __syncthreads();
      for (int t = threadIdx.x; t < S::BN; t += S::threads) {
        const int n = tn * S::BN + t;
        if (n >= z.K) continue;
        float s = columns[t];
#pragma unroll
        for (int w = 1; w < S::WM; ++w) s += columns[w * S::BN + t];
        sums[(size_t)tm * classes + z.first + n] = s;
      }
    }
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m = m0 + 32 * i;
      if (m >= z.N) continue;
      unsigned short* row = out + (size_t)m * pitch;
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + 32 * j + 8 * q;
          const floatx16p& a = acc[i][j];
          if ((S::type == kPairs ? 2 * (n / 32 * 32) : n) >= pitch) continue;
          unsigned h[4];
          if (S::type == kPairs) {
#pragma unroll
            for (int r = 0; r < 4; ++r) h[r] = split_pair(a[4 * q + r] * kProbability);
            uintx2p* at = (uintx2p*)(row + (n / 32) * 64 + n % 32);
            at[0] = (uintx2p){(h[0] & 0xffffu) | h[1] << 16, (h[2] & 0xffffu) | h[3] << 16};
            at[8] = (uintx2p){h[0] >> 16 | (h[1] & 0xffff0000u), h[2] >> 16 | (h[3] & 0xffff0000u)};
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) h[r] = to_bf16(a[4 * q + r]);
            *(uintx2p*)(row + n) = (uintx2p){h[0] | h[1] << 16, h[2] | h[3] << 16};
          }
        }
    }
  }
};

// out[m][n] = sum[m][n] + acc * factor * 1/scale of an operand * the instance's weight
struct StoreEnd {
  void* out;
  int bf16Out;
  const float* sum;                   // what other pieces gave, may be null (and may be `out`)
  int M, Ncols;
  float factor;
  const unsigned* magnitude;          // may be null
  const float *labels, *weights;      // may be null: rows are instances
  int nWeights;
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char*) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
    const float u = magnitude ? pair_unscale(*magnitude) : 1.f;
    const bool wide = (Ncols & 3) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)sum & 15) == 0;
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m = m0 + 32 * i;
      if (m >= M) continue;
      const float w = labels ? instance_weight(labels, weights, nWeights, m) * factor : factor;
      const size_t row = (size_t)m * Ncols;
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        const int n1 = n0 + 32 * j;
        if (wide) {
          float4 s[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            s[q] = sum && n1 + 8 * q < Ncols ? *(const float4*)(sum + row + n1 + 8 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (n1 + 8 * q >= Ncols) continue;
            const float4 v = make_float4(s[q].x + acc[i][j][4 * q] * u * w, s[q].y + acc[i][j][4 * q + 1] * u * w,
                                         s[q].z + acc[i][j][4 * q + 2] * u * w, s[q].w + acc[i][j][4 * q + 3] * u * w);
            if (bf16Out)
              *(uintx2p*)((unsigned short*)out + row + n1 + 8 * q) =
                  (uintx2p){(unsigned)to_bf16(v.x) | (unsigned)to_bf16(v.y) << 16, (unsigned)to_bf16(v.z) | (unsigned)to_bf16(v.w) << 16};
            else
              *(float4*)((float*)out + row + n1 + 8 * q) = v;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = n1 + 8 * (r / 4) + r % 4;
            if (n >= Ncols) continue;
            const float v = (sum ? sum[row + n] : 0.f) + acc[i][j][r] * u * w;
            if (bf16Out) ((unsigned short*)out)[row + n] = to_bf16(v);
            else ((float*)out)[row + n] = v;
          }
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------- what follows a product

// log sums of an instance from its tiles, and its term of the value; a wavefront per instance
__global__ __launch_bounds__(256) void fc_log_sums(float* __restrict__ logSums, float* __restrict__ terms, const float2* __restrict__ parts,
                                                   const float* __restrict__ own, const float* __restrict__ labels,
                                                   const float* __restrict__ weights, int nWeights, int N, int tiles) {
  const int n = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= N) return;
  const float2* p = parts + (size_t)n * tiles;
  float most = -__builtin_inff();
  for (int t = lane; t < tiles; t += 64) most = fmaxf(most, p[t].x);
  most = wave_max(most);
  const float from = most == -__builtin_inff() ? 0.f : most;
  float sum = 0.f;
  for (int t = lane; t < tiles; t += 64) sum += p[t].y * expf(p[t].x - from);
  sum = wave_sum(sum);
  if (lane) return;
  const float lse = from + logf(sum);
  logSums[n] = lse;
  const float w = instance_weight(labels, weights, nWeights, n);
  terms[n] = w != 0.f ? w * (lse - own[n]) : 0.f;
}

__global__ __launch_bounds__(256) void fc_total(float* __restrict__ y, const float* __restrict__ terms, int n, int divide) {
  __shared__ double lds[4];
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += (double)terms[i];
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double s = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    y[0] = (float)(divide ? s / divide : s);
  }
}

// dzdb: the tiles' column sums added up
__global__ __launch_bounds__(256) void fc_join_columns(float* __restrict__ db, const float* __restrict__ sums, int K, int tileRows, float factor) {
  const int c = (int)blockIdx.x * 256 + threadIdx.x;
  if (c >= K) return;
  double s = 0.0;
  for (int t = 0; t < tileRows; ++t) s += (double)sums[(size_t)t * K + c];
  db[c] = (float)s * factor;
}

// ---------------------------------------------------------------------------------------------- host

// What a call keeps in the caller's workspace
struct Plan {
  int type;
  bool xInPlace, fInPlace;         // bfloat16 rows of whole stages are read where they are
  long long xPitch, fPitch, pPitch;
  int piece, pieces, tiles;        // classes per piece; tiles of scores over all classes
  ProductPlan scores, dx, df;      // of a whole piece; the last one, if smaller, is cut as they are
  size_t x, xUnscale, xw, f, magnitudes, counters, parts, own, terms, logSums, p, sum, columns, products, total;
  int nCounters;
  // whether rows of D values can be read 16 bytes at a time; workgroups that pack rows
  int wide(const void* t, const mcn_fcloss_geom* g) const { return g->D % (type == kPairs ? 4 : 8) == 0 && aligned16(t); }
  unsigned pack_blocks(int rows, long long pitch) const { return (unsigned)(((size_t)rows * (pitch / (type == kPairs ? 16 : 8)) + 255) / 256); }
};

size_t kPieceBytes_() { return (size_t)std::max(1, tunable("fcloss_piece", 128)) << 20; }

Plan make_plan(const mcn_fcloss_geom* g, const void* x, const void* f, bool backward) {
  Plan p;
  p.type = g->dataType == MCN_BFLOAT16 ? kBf16 : kPairs;
  const bool whole = p.type == kBf16 && g->D % 64 == 0;
  p.fInPlace = whole && aligned16(f);
  p.xInPlace = whole && aligned16(x);
  p.xPitch = row_halves(p.type, g->D);
  p.fPitch = p.fInPlace ? g->D : row_halves(p.type, g->D);
  // a piece: P (backward) and the packed filters stay within kPieceBytes, whole tiles
  const long long most = (g->K + 255ll) / 256 * 256;
  const long long perClass = std::max<long long>(backward ? g->N * 2ll * (p.type == kPairs ? 2 : 1) : 0, p.fInPlace ? 0 : p.fPitch * 2);
  long long piece = perClass ? std::max(256ll, (long long)kPieceBytes_() / perClass / 256 * 256) : most;
  if (piece < most) {              // equal pieces
    const long long n = (most + piece - 1) / piece;
    piece = ((most + n - 1) / n + 255) / 256 * 256;
  }
  p.piece = (int)std::min(piece, most);
  p.pieces = (int)((g->K + (long long)p.piece - 1) / p.piece);
  const int classes = std::min(p.piece, g->K);
  p.scores = plan_product(p.type, g->N, classes, g->D);
  p.dx = plan_product(p.type, g->N, g->D, classes);
  p.df = plan_product(p.type, classes, g->D, g->N);
  p.tiles = div_up(g->K, kTileSize[p.scores.tile]);
  p.pPitch = row_halves(p.type, std::min<long long>(p.piece, (g->K + 63) / 64 * 64));
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.nCounters = (int)(backward ? std::max({p.scores.counters(), p.dx.counters(), p.df.counters()}) : p.scores.counters());
  p.magnitudes = take(8 + 4 * p.nCounters);
  p.counters = p.magnitudes + 8;
  p.products = take(backward ? std::max({p.scores.partBytes(), p.dx.partBytes(), p.df.partBytes()}) : p.scores.partBytes());
  p.x = take(p.xInPlace ? 0 : (size_t)g->N * p.xPitch * 2);
  p.xUnscale = take(p.type == kPairs ? (size_t)g->N * 4 : 0);
  p.f = take(p.fInPlace ? 0 : (size_t)std::min(p.piece, g->K) * p.fPitch * 2);
  p.parts = take((size_t)g->N * p.tiles * 8);
  p.own = take((size_t)g->N * 4);
  p.terms = take((size_t)g->N * 4);
  p.logSums = take((size_t)g->N * 4);
  p.xw = p.p = p.sum = p.columns = 0;
  if (backward) {
    p.xw = take((size_t)g->N * p.xPitch * 2);
    p.columns = take((size_t)div_up(g->N, kTileSize[p.scores.tile]) * g->K * 4);
    p.p = take((size_t)g->N * p.pPitch * 2);
    p.sum = take(p.type == kBf16 && p.pieces > 1 ? (size_t)g->N * g->D * 4 : 0);
  }
  p.total = at;
  return p;
}

int check(const char* who, const mcn_fcloss_geom* g, size_t nLabels, const float* weights, size_t nWeights) {
  if (!g) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null geometry", who);
  if (g->D < 0 || g->K < 0 || g->N < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative tensor extent", who);
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d", who, g->dataType);
  if (g->D > (1 << 20) || g->K > (1 << 24)) return fail(MCN_UNSUPPORTED, "%s: more than 2^20 features or 2^24 classes", who);
  if (g->N > 0 && (g->D == 0 || g->K == 0)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: instances without features or classes", who);
  if (nLabels != (size_t)g->N) return fail(MCN_ILLEGAL_ARGUMENT, "%s: C does not have one label per image", who);
  if (weights && g->N > 0 && (nWeights == 0 || (size_t)g->N % nWeights != 0))
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: the instance weights cannot be broadcast to the labels", who);
  return MCN_SUCCESS;
}

// x as the operand of the scores, and the magnitudes of the filters and of the weighted features
int pack_x(hipStream_t s, const char* who, const Plan& p, const mcn_fcloss_geom* g, char* ws, const void* x, const void* f, const float* labels,
           const float* weights, int nWeights, bool weighted, Matrix* op) {
  *op = {p.xInPlace ? x : ws + p.x, p.xPitch, 0, g->N};
  unsigned* m = (unsigned*)(ws + p.magnitudes);
  if (p.type == kPairs || p.nCounters) {
    KernelTimer timer("fc_clear", s);
    hipLaunchKernelGGL(fc_clear, dim3(1), dim3(256), 0, s, m, 2 + p.nCounters);
  }
  if (p.type == kPairs) {
    const size_t n = (size_t)g->K * g->D;
    KernelTimer timer("fc_magnitude", s);
    hipLaunchKernelGGL(fc_magnitude, dim3((unsigned)((n + kMagnitudeStep - 1) / kMagnitudeStep)), dim3(256), 0, s, m, (const float*)f, n, (int)aligned16(f));
  }
  if (p.xInPlace) return MCN_SUCCESS;
  KernelTimer timer("fc_pack", s);
  if (p.type == kPairs)
    hipLaunchKernelGGL(fc_pack_rows, dim3((unsigned)div_up(g->N, 4)), dim3(256), 0, s, (unsigned short*)(ws + p.x), (float*)(ws + p.xUnscale),
                       weighted ? m + 1 : nullptr, (const float*)x, g->D, g->N, p.xPitch, labels, weights, nWeights, p.wide(x, g));
  else
    hipLaunchKernelGGL(fc_pack<kBf16>, dim3(p.pack_blocks(g->N, p.xPitch)), dim3(256), 0, s, (unsigned short*)(ws + p.x), (const unsigned*)nullptr, x, g->D,
                       g->N, p.xPitch, (const float*)nullptr, (const float*)nullptr, 1, p.wide(x, g));
  return check_launch(who);
}

// rows of x or the filters as an operand of all products (by the tensor's magnitude), or times the instances' weights
template <int TYPE>
void pack(hipStream_t s, const Plan& p, const mcn_fcloss_geom* g, char* out, const unsigned* magnitude, const void* x, int rows, long long pitch,
          const float* labels, const float* weights, int nWeights) {
  KernelTimer timer("fc_pack", s);
  hipLaunchKernelGGL(fc_pack<TYPE>, dim3(p.pack_blocks(rows, pitch)), dim3(256), 0, s, (unsigned short*)out, magnitude, x, g->D, rows, pitch, labels, weights,
                     nWeights, p.wide(x, g));
}

// the filters of a piece
template <int TYPE>
Matrix pack_f(hipStream_t s, const Plan& p, const mcn_fcloss_geom* g, char* ws, const void* f, int first, int count) {
  const char* from = (const char*)f + (size_t)first * g->D * (TYPE == kPairs ? 4 : 2);
  if (!p.fInPlace) pack<TYPE>(s, p, g, ws + p.f, (const unsigned*)(ws + p.magnitudes), from, count, p.fPitch, nullptr, nullptr, 1);
  return {p.fInPlace ? from : ws + p.f, p.fPitch, 0, count};
}

template <int TYPE>
int forward(hipStream_t s, const char* who, const Plan& p, const mcn_fcloss_geom* g, float* logSums, const void* f, const float* biases,
            const float* labels, const float* weights, int nWeights, char* ws, const Matrix& X) {
  const Scratch scratch = {(float*)(ws + p.products), (unsigned*)(ws + p.counters)};
  for (int k = 0; k < p.pieces; ++k) {
    const int first = k * p.piece, count = std::min(p.piece, g->K - first);
    const Matrix F = pack_f<TYPE>(s, p, g, ws, f, first, count);
    StatsEnd e;
    e.z = {TYPE == kPairs ? (const float*)(ws + p.xUnscale) : nullptr, biases, (const unsigned*)(ws + p.magnitudes), g->N, count, first};
    e.parts = (float2*)(ws + p.parts);
    e.own = (float*)(ws + p.own);
    e.labels = labels;
    e.tiles = p.tiles; e.firstTile = first / kTileSize[p.scores.tile]; e.classes = g->K;
    const int rc = product<TYPE, false, false>(s, who, "fc_scores", X, F, g->N, count, p.scores.of(g->N, count), scratch, e);
    if (rc) return rc;
  }
  KernelTimer timer("fc_log_sums", s);
  hipLaunchKernelGGL(fc_log_sums, dim3((unsigned)div_up(g->N, 4)), dim3(256), 0, s, logSums, (float*)(ws + p.terms), (const float2*)(ws + p.parts),
                     (const float*)(ws + p.own), labels, weights, nWeights, g->N, p.tiles);
  return check_launch(who);
}

template <int TYPE>
int backward(hipStream_t s, const char* who, const Plan& p, const mcn_fcloss_geom* g, void* derInput, void* derFilters, float* derBiases,
             const float* logSums, const void* f, const float* biases, const float* labels, const float* weights, int nWeights, float factor,
             char* ws, const Matrix& X, const void* x) {
  const unsigned* mag = (const unsigned*)(ws + p.magnitudes);
  const Matrix Xw = {ws + p.xw, p.xPitch, 0, g->N};
  const Scratch scratch = {(float*)(ws + p.products), (unsigned*)(ws + p.counters)};
  if (derFilters) pack<TYPE>(s, p, g, ws + p.xw, mag + 1, x, g->N, p.xPitch, labels, weights, nWeights);
  const float times = TYPE == kPairs ? factor / kProbability : factor;
  for (int k = 0; k < p.pieces; ++k) {
    const int first = k * p.piece, count = std::min(p.piece, g->K - first);
    const Matrix F = pack_f<TYPE>(s, p, g, ws, f, first, count);
    ProbabilitiesEnd e;
    e.z = {TYPE == kPairs ? (const float*)(ws + p.xUnscale) : nullptr, biases, mag, g->N, count, first};
    e.out = (unsigned short*)(ws + p.p);
    e.pitch = p.pPitch;
    e.labels = labels; e.weights = weights; e.logSums = logSums;
    e.nWeights = nWeights; e.classes = g->K;
    e.sums = derBiases ? (float*)(ws + p.columns) : nullptr;
    int rc = product<TYPE, false, false>(s, who, "fc_probabilities", X, F, g->N, (count + 63) / 64 * 64, p.scores.of(g->N, (count + 63) / 64 * 64), scratch, e);
    if (rc) return rc;
    const Matrix P = {ws + p.p, p.pPitch, 0, g->N};
    if (derInput) {
      // (the pieces add up in single precision: in derInput itself, or beside it)
      float* sum = TYPE == kPairs ? (float*)derInput : (float*)(ws + p.sum);
      const bool last = k == p.pieces - 1;
      const StoreEnd d = {TYPE == kPairs || last ? derInput : sum, TYPE == kBf16 && last, k > 0 ? sum : nullptr, g->N, g->D, times,
                          TYPE == kPairs ? mag : nullptr, labels, weights, nWeights};
      ProductPlan q = p.dx;
      q.stages = div_up(count, stage_depth(TYPE));
      rc = product<TYPE, false, true>(s, who, "fc_derivative_x", P, F, g->N, g->D, q, scratch, d);
      if (rc) return rc;
    }
    if (derFilters) {
      const StoreEnd d = {(char*)derFilters + (size_t)first * g->D * (TYPE == kPairs ? 4 : 2), TYPE == kBf16, nullptr, count, g->D, times,
                          TYPE == kPairs ? mag + 1 : nullptr, nullptr, nullptr, 1};
      rc = product<TYPE, true, true>(s, who, "fc_derivative_f", P, Xw, count, g->D, p.df.of(count, g->D), scratch, d);
      if (rc) return rc;
    }
  }
  if (derBiases) {
    KernelTimer timer("fc_join", s);
    hipLaunchKernelGGL(fc_join_columns, dim3((unsigned)div_up(g->K, 256)), dim3(256), 0, s, derBiases, (const float*)(ws + p.columns), g->K,
                       div_up(g->N, kTileSize[p.scores.tile]), factor);
  }
  return check_launch(who);
}

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_fcloss_workspace_bytes(const mcn_fcloss_geom* g, int backward) {
  if (!g || g->D <= 0 || g->K <= 0 || g->N <= 0 || g->D > (1 << 20) || g->K > (1 << 24)) return 0;
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return 0;
  // (the larger of the two ways tensors can be aligned)
  const void* odd = (const void*)2;
  return std::max(make_plan(g, nullptr, nullptr, backward != 0).total, make_plan(g, odd, odd, backward != 0).total);
}

int mcn_fcloss_forward(mcn_stream_t stream, const mcn_fcloss_geom* g, float* y, float* logSums, const void* x, const void* filters,
                       const float* biases, const float* labels, size_t nLabels, const float* instanceWeights, size_t nWeights, void* workspace,
                       size_t workspaceBytes) {
  const char* who = "mcn_fcloss_forward";
  int rc = check(who, g, nLabels, instanceWeights, nWeights);
  if (rc) return rc;
  if (!y) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null output", who);
  hipStream_t s = as_stream(stream);
  char* ws = (char*)workspace;
  Plan p;
  if (g->N > 0) {
    if (!x || !filters || !labels) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
    p = make_plan(g, x, filters, false);
    if (!workspace || workspaceBytes < p.total)
      return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, p.total);
    Matrix X;
    rc = pack_x(s, who, p, g, ws, x, filters, labels, instanceWeights, (int)nWeights, false, &X);
    if (rc) return rc;
    float* sums = logSums ? logSums : (float*)(ws + p.logSums);
    rc = p.type == kPairs ? forward<kPairs>(s, who, p, g, sums, filters, biases, labels, instanceWeights, (int)nWeights, ws, X)
                          : forward<kBf16>(s, who, p, g, sums, filters, biases, labels, instanceWeights, (int)nWeights, ws, X);
    if (rc) return rc;
  }
  KernelTimer timer("fc_total", s);
  hipLaunchKernelGGL(fc_total, dim3(1), dim3(256), 0, s, y, g->N > 0 ? (const float*)(ws + p.terms) : nullptr, g->N, g->normalise ? g->N : 0);
  return check_launch(who);
}

int mcn_fcloss_backward(mcn_stream_t stream, const mcn_fcloss_geom* g, void* derInput, void* derFilters, float* derBiases, const float* logSums,
                        const void* x, const void* filters, const float* biases, const float* labels, size_t nLabels, const float* instanceWeights,
                        size_t nWeights, double derOutput, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_fcloss_backward";
  int rc = check(who, g, nLabels, instanceWeights, nWeights);
  if (rc) return rc;
  if (!derInput && !derFilters && !derBiases) return MCN_SUCCESS;
  if (g->N == 0) {   // sums over no images
    if (derFilters && (size_t)g->K * g->D) {
      hipLaunchKernelGGL(fc_zero, dim3((unsigned)(((size_t)g->K * g->D + 1023) / 1024)), dim3(256), 0, as_stream(stream), derFilters,
                         (size_t)g->K * g->D, g->dataType == MCN_BFLOAT16);
    }
    if (derBiases && g->K)
      hipLaunchKernelGGL(fc_zero, dim3((unsigned)((g->K + 1023) / 1024)), dim3(256), 0, as_stream(stream), derBiases, (size_t)g->K, 0);
    return check_launch(who);
  }
  if (!x || !filters || !labels) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  const Plan p = make_plan(g, x, filters, true);
  if (!workspace || workspaceBytes < p.total)
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, p.total);
  hipStream_t s = as_stream(stream);
  char* ws = (char*)workspace;
  Matrix X;
  rc = pack_x(s, who, p, g, ws, x, filters, labels, instanceWeights, (int)nWeights, true, &X);
  if (rc) return rc;
  const float factor = (float)(g->normalise ? derOutput / g->N : derOutput);
  if (!logSums) {
    float* sums = (float*)(ws + p.logSums);
    rc = p.type == kPairs ? forward<kPairs>(s, who, p, g, sums, filters, biases, labels, instanceWeights, (int)nWeights, ws, X)
                          : forward<kBf16>(s, who, p, g, sums, filters, biases, labels, instanceWeights, (int)nWeights, ws, X);
    if (rc) return rc;
    logSums = sums;
  }
  return p.type == kPairs ? backward<kPairs>(s, who, p, g, derInput, derFilters, derBiases, logSums, filters, biases, labels, instanceWeights,
                                             (int)nWeights, factor, ws, X, x)
                          : backward<kBf16>(s, who, p, g, derInput, derFilters, derBiases, logSums, filters, biases, labels, instanceWeights,
                                            (int)nWeights, factor, ws, X, x);
}

}  // extern "C"
