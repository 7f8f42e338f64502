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

// What a call's first launches leave: per workgroup of fc_magnitudes the largest magnitude of its filters, or of its instances' weighted
// features, as the bits of floats (a NaN or an infinity wins, and pair_scale leaves such a tensor as it is); every instance's own;
// and, from fc_pack, the two tensors'.
constexpr int kFilterParts = 1024, kFeatureParts = 512;
struct Magnitudes {
  unsigned filters, features;                                     // (what the products' ends read)
  unsigned filterParts[kFilterParts], featureParts[kFeatureParts];
};
constexpr int kMagnitudeStep = 256 * 4 * 8;   // values a workgroup takes at a time

__device__ __forceinline__ unsigned magnitude4(uintx4p v) {
  return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
}
__device__ __forceinline__ unsigned wave_most(unsigned m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, kWave));
  return m;
}
__device__ __forceinline__ unsigned group_most(unsigned m, unsigned* lds) {   // of 256 threads
  m = wave_most(m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

// Workgroups [0, filterGroups): the filters; the rest: a wavefront per instance.
__global__ __launch_bounds__(256) void fc_magnitudes(Magnitudes* __restrict__ out, unsigned* __restrict__ rows, const float* __restrict__ f, size_t n,
                                                     int filterGroups, int vec, const float* __restrict__ x, int D, int N,
                                                     const float* __restrict__ labels, const float* __restrict__ weights, int nWeights) {
  __shared__ unsigned lds[4];
  unsigned most = 0;
  if ((int)blockIdx.x < filterGroups) {
    for (size_t first = (size_t)blockIdx.x * kMagnitudeStep; first < n; first += (size_t)filterGroups * kMagnitudeStep) {
      if (vec && first + kMagnitudeStep <= n) {
        const uintx4p* f4 = (const uintx4p*)(f + first) + threadIdx.x;
        uintx4p v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f4[256 * i];
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, magnitude4(v[i]));
      } else {
        for (size_t i = first + threadIdx.x; i < std::min(first + kMagnitudeStep, n); i += 256) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);
      }
    }
    most = group_most(most, lds);
    if (threadIdx.x == 0) out->filterParts[blockIdx.x] = most;
    return;
  }
  const int group = blockIdx.x - filterGroups, groups = gridDim.x - filterGroups, lane = threadIdx.x & 63;
  for (int row = group * 4 + (int)(threadIdx.x >> 6); row < N; row += groups * 4) {
    unsigned m = 0;
    for (int c = 8 * lane; c < D; c += 512) {
      float v[8];
      load8(v, x + (size_t)row * D, c, D);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    m = wave_most(m);
    if (lane == 0) rows[row] = m;
    const float w = instance_weight(labels, weights, nWeights, row);
    if (w != 0.f) most = max(most, __float_as_uint(fabsf(__uint_as_float(m) * w)));
  }
  most = group_most(most, lds);
  if (threadIdx.x == 0) out->featureParts[group] = most;
}

// Rows brought into the form the products read: pairs by a magnitude, or bfloat16 at a pitch of whole stages.
enum { kFilters, kFeatures, kWeighted };   // by the tensor's magnitude; each row by its own; times the instance's weight (zeros for instances
                                           // that do not count, whatever they hold), by the tensor's
// (In bfloat16 the weighted features are rounded, for dzdf alone.  Weights in P would round what both derivatives are made of by as much:
// without them the label's -1, most of P, is exact.)
struct PackPart {
  const void* x;
  unsigned short* out;
  long long pitch;
  int rows, form;
  unsigned firstGroup;
};
struct PackJob {
  PackPart parts[3];
  int nParts, D;
  Magnitudes* magnitudes;                  // pairs
  int filterGroups, featureGroups;         // 0: `filters` and `features` are there already
  const unsigned* rowMagnitudes;
  float* unscale;                          // of the rows by their own magnitudes
  const float *labels, *weights;
  int nWeights;
  unsigned* counters;                      // cleared on the way
  int nCounters;
};
constexpr int kPackSteps = 4;              // times eight values a thread

template <int TYPE>
__global__ __launch_bounds__(256) void fc_pack(PackJob j) {
  __shared__ unsigned lds[4];
  const int which = j.nParts > 2 && blockIdx.x >= j.parts[2].firstGroup ? 2 : j.nParts > 1 && blockIdx.x >= j.parts[1].firstGroup ? 1 : 0;
  const PackPart p = j.parts[which];
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < j.nCounters; i += 256) j.counters[i] = 0;
  // (all of a thread's loads first, not each behind the store before it: 32000 x 1024 single-precision values 56 -> 52 us, 21841 x 1001 bfloat16
  // ones 22 -> 20)
  const int per = (int)(p.pitch / (TYPE == kPairs ? 16 : 8));
  const size_t all = (size_t)p.rows * per;
  int row[kPackSteps], c[kPackSteps];
  float w[kPackSteps], v[kPackSteps][8];
  unsigned own[kPackSteps];
#pragma unroll
  for (int step = 0; step < kPackSteps; ++step) {
    const size_t i = ((size_t)(blockIdx.x - p.firstGroup) * kPackSteps + step) * 256 + threadIdx.x;
    const bool live = i < all;
    row[step] = live ? (int)(i / per) : -1;
    c[step] = live ? (int)(i - (size_t)row[step] * per) * 8 : 0;
    w[step] = !live ? 0.f : p.form == kWeighted ? instance_weight(j.labels, j.weights, j.nWeights, row[step]) : 1.f;
    own[step] = TYPE == kPairs && p.form == kFeatures && live ? j.rowMagnitudes[row[step]] : 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[step][k] = 0.f;
    if (w[step] != 0.f) {
      if (TYPE == kPairs) load8(v[step], (const float*)p.x + (size_t)row[step] * j.D, c[step], j.D);
      else load8(v[step], (const unsigned short*)p.x + (size_t)row[step] * j.D, c[step], j.D);
    }
  }
  float scale = 1.f;
  if (TYPE == kPairs && p.form != kFeatures) {
    unsigned m = 0;
    const int parts = p.form == kFilters ? j.filterGroups : j.featureGroups;
    const unsigned* from = p.form == kFilters ? j.magnitudes->filterParts : j.magnitudes->featureParts;
    if (parts) {
      for (int i = threadIdx.x; i < parts; i += 256) m = max(m, from[i]);
      m = group_most(m, lds);
      if (blockIdx.x == p.firstGroup && threadIdx.x == 0) (p.form == kFilters ? j.magnitudes->filters : j.magnitudes->features) = m;
    } else {
      m = j.magnitudes->filters;
    }
    scale = pair_scale(m);
  }
#pragma unroll
  for (int step = 0; step < kPackSteps; ++step) {
    if (row[step] < 0) return;
    unsigned short* const to = p.out + (size_t)row[step] * p.pitch;
    if (TYPE == kPairs) {
      if (p.form == kFeatures) {
        scale = pair_scale(own[step]);
        if (c[step] == 0) j.unscale[row[step]] = pair_unscale(own[step]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[step][k] = v[step][k] * w[step] * scale;
      store8_pairs(to, c[step], v[step]);
    } else {
      uintx4p h;
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = (unsigned)to_bf16(v[step][2 * k] * w[step]) | (unsigned)to_bf16(v[step][2 * k + 1] * w[step]) << 16;
      *(uintx4p*)(to + c[step]) = h;
    }
  }
}

__global__ __launch_bounds__(256) void fc_zero(void* __restrict__ p, size_t n, int is16) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    if (is16) ((unsigned short*)p)[i] = 0;
    else ((float*)p)[i] = 0.f;
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
  float* sums;                     // [tile rows][classes], times `factor`; may be null
  float factor;
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
    z.make<S>(acc, m0, n0, (tn + 1) * S::BN);
    float* columns = (float*)(lds + S::ldsBytes - S::WM * S::BN * 4);  // [WM][BN]
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
        sums[(size_t)tm * classes + z.first + n] = s * factor;
      }
    }
    constexpr int size = S::type == kPairs ? 4 : 2, J = turned_blocks<S, size>();
    const RowTurn<J * 32 * size> turn(lds, wn * S::WM + wm);
    static_assert(S::WM * S::WN * RowTurn<J * 32 * size>::size + S::WM * S::BN * 4 <= S::ldsBytes, "beside the columns");
    const int half = lane >> 5, l32 = lane & 31, first = tn * S::BN + 32 * wn * S::TN;
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j0 = 0; j0 < S::TN; j0 += J) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx16p& a = acc[i][j0 + j];
            const int column = 8 * q + 4 * half;
            unsigned h[4];
            if (S::type == kPairs) {
#pragma unroll
              for (int r = 0; r < 4; ++r) h[r] = split_pair(a[4 * q + r] * kProbability);
              *(uintx2p*)turn.at(l32, 128 * j + 2 * column) = (uintx2p){(h[0] & 0xffffu) | h[1] << 16, (h[2] & 0xffffu) | h[3] << 16};
              *(uintx2p*)turn.at(l32, 128 * j + 64 + 2 * column) = (uintx2p){h[0] >> 16 | (h[1] & 0xffff0000u), h[2] >> 16 | (h[3] & 0xffff0000u)};
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) h[r] = to_bf16(a[4 * q + r]);
              *(uintx2p*)turn.at(l32, 64 * j + 2 * column) = (uintx2p){h[0] | h[1] << 16, h[2] | h[3] << 16};
            }
          }
        const int m1 = tm * S::BM + 32 * (wm * S::TM + i), start = (first + 32 * j0) * size;   // bytes from the row's first class
        turn.each(lane, [&](int row, int offset, uintx4p v) {
          if (m1 + row < z.N && start + offset < 2 * pitch) *(uintx4p*)((char*)(out + (size_t)(m1 + row) * pitch) + start + offset) = v;
        });
      }
  }
};

// out[m][n] = sum[m][n] + acc / the operands' scales * factor * the instance's weight
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
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    // (P as pairs is 2^14 too large; taken off together with the other operand's scale, before the factor, so that nothing leaves the range on
    // the way.  Both are powers of two.)
    const float u = magnitude ? pair_unscale(*magnitude) * (1.f / kProbability) : 1.f;
    const bool wide = (Ncols & 3) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)sum & 15) == 0;
    constexpr int J = turned_blocks<S, 4>();
    const RowTurn<J * 128> turn(lds, wn * S::WM + wm);
    const int half = lane >> 5, l32 = lane & 31;
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m1 = tm * S::BM + 32 * (wm * S::TM + i);
      const float w = labels && m1 + l32 < M ? instance_weight(labels, weights, nWeights, m1 + l32) * factor : factor;
#pragma unroll
      for (int j0 = 0; j0 < S::TN; j0 += J) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx16p& a = acc[i][j0 + j];
            *(float4*)turn.at(l32, 128 * j + 32 * q + 16 * half) =
                make_float4(a[4 * q] * u * w, a[4 * q + 1] * u * w, a[4 * q + 2] * u * w, a[4 * q + 3] * u * w);
          }
        const int n1 = tn * S::BN + 32 * (wn * S::TN + j0);
        if (wide) {
          turn.each(lane, [&](int row, int offset, uintx4p bits) {
            const int n = n1 + offset / 4;
            if (m1 + row >= M || n >= Ncols) return;
            const size_t at = (size_t)(m1 + row) * Ncols + n;
            float4 v = __builtin_bit_cast(float4, bits);
            if (sum) {
              const float4 s = *(const float4*)(sum + at);
              v = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
            }
            if (bf16Out)
              *(uintx2p*)((unsigned short*)out + at) =
                  (uintx2p){(unsigned)to_bf16(v.x) | (unsigned)to_bf16(v.y) << 16, (unsigned)to_bf16(v.z) | (unsigned)to_bf16(v.w) << 16};
            else
              *(float4*)((float*)out + at) = v;
          });
        } else {
          // (rows that start anywhere: a value a lane, J * 32 lanes along a row)
          turn.single(lane, [&](int row, int column, float v) {
            const int n = n1 + column;
            if (m1 + row >= M || n >= Ncols) return;
            const size_t at = (size_t)(m1 + row) * Ncols + n;
            if (sum) v += sum[at];
            if (bf16Out) ((unsigned short*)out)[at] = to_bf16(v);
            else ((float*)out)[at] = v;
          });
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------- what follows a product

// (largest, sum of exponentials against it) of two sets of scores together
__device__ __forceinline__ float2 both(float2 a, float2 b) {
  const float most = fmaxf(a.x, b.x), from = most == -__builtin_inff() ? 0.f : most;
  return make_float2(most, a.y * expf(a.x - from) + b.y * expf(b.x - from));
}
// log sums of an instance from its tiles, WAVES wavefronts per instance, and its term of the value; the workgroup that comes last adds
// the terms up, in double and in order (they go past the XCDs' L2s, as the parts of a product do)
template <int WAVES>
__global__ __launch_bounds__(256) void fc_log_sums(float* __restrict__ y, float* __restrict__ logSums, float* __restrict__ terms, unsigned* __restrict__ counter,
                                                   const float2* __restrict__ parts, const float* __restrict__ own, const float* __restrict__ labels,
                                                   const float* __restrict__ weights, int nWeights, int N, int tiles, int divide) {
  __shared__ double lds[4];
  __shared__ float2 joint[4];
  __shared__ unsigned last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = threadIdx.x % (64 * WAVES);
  constexpr int kPer = 4 / WAVES;
  for (int first = (int)blockIdx.x * kPer; first < N; first += (int)gridDim.x * kPer) {
    const int n = first + wave / WAVES;
    // four at a time, and the four among each other: a chain of as few exponentials as there are steps
    float2 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = make_float2(-__builtin_inff(), 0.f);
    if (n < N) {
      const float2* p = parts + (size_t)n * tiles;
      for (int i = t; i < tiles; i += 64 * WAVES * 4)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + 64 * WAVES * k < tiles) v[k] = both(v[k], p[i + 64 * WAVES * k]);
    }
    float2 s = both(both(v[0], v[1]), both(v[2], v[3]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = both(s, make_float2(__shfl_xor(s.x, o, kWave), __shfl_xor(s.y, o, kWave)));
    if (WAVES > 1) {
      __syncthreads();
      if (lane == 0) joint[wave] = s;
      __syncthreads();
      s = both(both(joint[0], joint[1]), both(joint[2], joint[3]));
    }
    if (t == 0 && n < N) {
      const float lse = (s.x == -__builtin_inff() ? 0.f : s.x) + logf(s.y);
      logSums[n] = lse;
      const float w = instance_weight(labels, weights, nWeights, n);
      __hip_atomic_store(terms + n, w != 0.f ? w * (lse - own[n]) : 0.f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (!y) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  double acc = 0.0;
  for (int i = threadIdx.x; i < N; i += 256) acc += (double)__hip_atomic_load(terms + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  acc = wave_sum(acc);
  if (lane == 0) lds[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double s = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    y[0] = (float)(divide ? s / divide : s);
  }
}

// the value from the terms of many instances
__global__ __launch_bounds__(1024) void fc_total(float* __restrict__ y, const float* __restrict__ terms, int n, int divide) {
  __shared__ double lds[16];
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) acc += (double)terms[i];
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x) return;
  double s = 0.0;
  for (int w = 0; w < 16; ++w) s += lds[w];
  y[0] = (float)(divide ? s / divide : s);
}

// dzdb: the tiles' column sums added up
__global__ __launch_bounds__(256) void fc_join_columns(float* __restrict__ db, const float* __restrict__ sums, int K, int tileRows) {
  const int c = (int)blockIdx.x * 256 + threadIdx.x;
  if (c >= K) return;
  double s = 0.0;
  for (int t = 0; t < tileRows; ++t) s += (double)sums[(size_t)t * K + c];
  db[c] = (float)s;
}

// ---------------------------------------------------------------------------------------------- host

// What a call keeps in the caller's workspace
struct Plan {
  int type;
  bool xInPlace, fInPlace;         // bfloat16 rows of whole stages are read where they are
  long long xPitch, fPitch, pPitch;
  int piece, pieces, tiles;        // classes per piece; tiles of scores over all classes
  ProductPlan scores, dx, df;      // of a whole piece; the last one, if smaller, is cut as they are
  size_t x, xUnscale, xw, f, magnitudes, rowMagnitudes, counters, parts, own, terms, logSums, p, sum, columns, products, total;
  int nCounters, tileRows;         // (counters: the last is fc_log_sums')
  // workgroups that pack rows
  unsigned pack_groups(int rows, long long pitch) const {
    return (unsigned)(((size_t)rows * (pitch / (type == kPairs ? 16 : 8)) + 256 * kPackSteps - 1) / (256 * kPackSteps));
  }
};

// A piece's P, or packed filters: larger ones save passes over the sums of dzdx (128, 256, 512 MiB: 29.5, 29.5, 29.2 ms for 128000 classes in
// bfloat16, 1.76, 1.72, 1.72 ms for 32000 in single precision)
size_t piece_bytes() {
  const int kib = tunable("fcloss_piece_kib", 0);
  return kib > 0 ? (size_t)kib << 10 : (size_t)256 << 20;
}

Plan make_plan(const mcn_fcloss_geom* g, const void* x, const void* f, bool backward) {
  Plan p;
  p.type = g->dataType == MCN_BFLOAT16 ? kBf16 : kPairs;
  const bool whole = p.type == kBf16 && g->D % 64 == 0;
  p.fInPlace = whole && aligned16(f);
  p.xInPlace = whole && aligned16(x);
  p.xPitch = row_halves(p.type, g->D);
  p.fPitch = p.fInPlace ? g->D : row_halves(p.type, g->D);
  // a piece: P (backward) and the packed filters stay within piece_bytes(), whole tiles
  const long long most = (g->K + 255ll) / 256 * 256;
  const long long perClass = std::max<long long>(backward ? g->N * 2ll * (p.type == kPairs ? 2 : 1) : 0, p.fInPlace ? 0 : p.fPitch * 2);
  long long piece = perClass ? std::max(256ll, (long long)piece_bytes() / perClass / 256 * 256) : most;
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
  p.tileRows = div_up(g->N, kTileSize[p.scores.tile]);
  p.nCounters = 1 + (int)(backward ? std::max({p.scores.counters(), p.dx.counters(), p.df.counters()}) : p.scores.counters());
  p.magnitudes = take(p.type == kPairs ? sizeof(Magnitudes) : 0);
  p.rowMagnitudes = take(p.type == kPairs ? (size_t)g->N * 4 : 0);
  p.counters = take(4 * (size_t)p.nCounters);
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
    p.columns = take(p.tileRows > 1 ? (size_t)p.tileRows * g->K * 4 : 0);
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
  if (g->D > (1 << 20) || g->K > (1 << 24) || g->N > (1 << 30))
    return fail(MCN_UNSUPPORTED, "%s: more than 2^20 features, 2^24 classes or 2^30 images", who);
  if (g->N > 0 && (g->D == 0 || g->K == 0)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: instances without features or classes", who);
  if (nLabels != (size_t)g->N) return fail(MCN_ILLEGAL_ARGUMENT, "%s: C does not have one label per image", who);
  if (weights && g->N > 0 && (nWeights == 0 || (size_t)g->N % nWeights != 0))
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: the instance weights cannot be broadcast to the labels", who);
  return MCN_SUCCESS;
}

struct Call {
  hipStream_t s;
  const char* who;
  const mcn_fcloss_geom* g;
  const void *x, *filters;
  const float *biases, *labels, *weights;
  int nWeights;
  char* ws;
  Plan p;
  Magnitudes* magnitudes() const { return (Magnitudes*)(ws + p.magnitudes); }
  Scratch scratch() const { return {(float*)(ws + p.products), (unsigned*)(ws + p.counters)}; }
  Matrix X() const { return {p.xInPlace ? x : ws + p.x, p.xPitch, 0, g->N}; }
  const char* piece_of(const void* t, int first) const { return (const char*)t + (size_t)first * g->D * (p.type == kPairs ? 4 : 2); }
  int classes(int piece) const { return std::min(p.piece, g->K - piece * p.piece); }
  Matrix F(int piece) const { return {p.fInPlace ? piece_of(filters, piece * p.piece) : ws + p.f, p.fPitch, 0, classes(piece)}; }
};

void launch_pack(const Call& c, PackJob& j) {
  unsigned groups = 0;
  for (int k = 0; k < j.nParts; ++k) {
    j.parts[k].firstGroup = groups;
    groups += c.p.pack_groups(j.parts[k].rows, j.parts[k].pitch);
  }
  if (groups == 0) {               // (the counters alone)
    j.parts[0] = {};
    groups = 1;
  }
  KernelTimer timer("fc_pack", c.s);
  if (c.p.type == kPairs) hipLaunchKernelGGL(fc_pack<kPairs>, dim3(groups), dim3(256), 0, c.s, j);
  else hipLaunchKernelGGL(fc_pack<kBf16>, dim3(groups), dim3(256), 0, c.s, j);
}

// What comes before the products: magnitudes, the features (and, for dzdf, the weighted ones), the first piece of the filters, counters
int prepare(const Call& c, bool weighted) {
  const Plan& p = c.p;
  PackJob j = {};
  j.D = c.g->D;
  j.labels = c.labels; j.weights = c.weights; j.nWeights = c.nWeights;
  j.counters = (unsigned*)(c.ws + p.counters); j.nCounters = p.nCounters;
  if (p.type == kPairs) {
    const size_t n = (size_t)c.g->K * c.g->D;
    j.magnitudes = c.magnitudes();
    j.rowMagnitudes = (unsigned*)(c.ws + p.rowMagnitudes);
    j.unscale = (float*)(c.ws + p.xUnscale);
    j.filterGroups = (int)std::min<size_t>(kFilterParts, (n + kMagnitudeStep - 1) / kMagnitudeStep);
    j.featureGroups = std::min(kFeatureParts, div_up(c.g->N, 4));
    KernelTimer timer("fc_magnitudes", c.s);
    hipLaunchKernelGGL(fc_magnitudes, dim3((unsigned)(j.filterGroups + j.featureGroups)), dim3(256), 0, c.s, j.magnitudes, (unsigned*)(c.ws + p.rowMagnitudes),
                       (const float*)c.filters, n, j.filterGroups, (int)aligned16(c.filters), (const float*)c.x, c.g->D, c.g->N, c.labels, c.weights,
                       c.nWeights);
  }
  if (!p.fInPlace) j.parts[j.nParts++] = {c.filters, (unsigned short*)(c.ws + p.f), p.fPitch, c.classes(0), kFilters, 0};
  if (!p.xInPlace) j.parts[j.nParts++] = {c.x, (unsigned short*)(c.ws + p.x), p.xPitch, c.g->N, kFeatures, 0};
  if (weighted) j.parts[j.nParts++] = {c.x, (unsigned short*)(c.ws + p.xw), p.xPitch, c.g->N, kWeighted, 0};
  launch_pack(c, j);
  return check_launch(c.who);
}

// the filters of a piece, where its products read them (`there`: prepare() has done it)
void pack_piece(const Call& c, int piece, bool there) {
  if (c.p.fInPlace || there) return;
  PackJob j = {};
  j.D = c.g->D;
  j.magnitudes = c.magnitudes();
  j.parts[j.nParts++] = {c.piece_of(c.filters, piece * c.p.piece), (unsigned short*)(c.ws + c.p.f), c.p.fPitch, c.classes(piece), kFilters, 0};
  launch_pack(c, j);
}

template <int TYPE>
Scores scores_of(const Call& c, int piece) {
  return {TYPE == kPairs ? (const float*)(c.ws + c.p.xUnscale) : nullptr, c.biases, TYPE == kPairs ? &c.magnitudes()->filters : nullptr, c.g->N,
          c.classes(piece), piece * c.p.piece};
}

// y may be null (the log sums alone)
template <int TYPE>
int forward(const Call& c, float* y, float* logSums) {
  const Plan& p = c.p;
  const int N = c.g->N;
  for (int k = 0; k < p.pieces; ++k) {
    pack_piece(c, k, k == 0);
    StatsEnd e;
    e.z = scores_of<TYPE>(c, k);
    e.parts = (float2*)(c.ws + p.parts);
    e.own = (float*)(c.ws + p.own);
    e.labels = c.labels;
    e.tiles = p.tiles; e.firstTile = k * p.piece / kTileSize[p.scores.tile]; e.classes = c.g->K;
    const int rc = product<TYPE, false, false>(c.s, c.who, "fc_scores", c.X(), c.F(k), N, c.classes(k), p.scores.of(N, c.classes(k)), c.scratch(), e);
    if (rc) return rc;
  }
  // Few instances: four wavefronts each.  Up to 1024 of them, the value is added up on the way (256 workgroups that count themselves in take
  // less than a launch, 2048 of them, for 8192 instances, 30 us more than one).
  const bool few = N <= 256, joined = N <= 1024;
  const int divide = c.g->normalise ? N : 0;
  float* const terms = (float*)(c.ws + p.terms);
  {
    KernelTimer timer("fc_log_sums", c.s);
    hipLaunchKernelGGL(few ? fc_log_sums<4> : fc_log_sums<1>, dim3((unsigned)std::min(1 << 20, div_up(N, few ? 1 : 4))), dim3(256), 0, c.s, joined ? y : nullptr, logSums, terms,
                       (unsigned*)(c.ws + p.counters) + p.nCounters - 1, (const float2*)(c.ws + p.parts), (const float*)(c.ws + p.own), c.labels, c.weights,
                       c.nWeights, N, p.tiles, divide);
  }
  if (y && !joined) {
    KernelTimer timer("fc_total", c.s);
    hipLaunchKernelGGL(fc_total, dim3(1), dim3(1024), 0, c.s, y, terms, N, divide);
  }
  return check_launch(c.who);
}

template <int TYPE>
int backward(const Call& c, void* derInput, void* derFilters, float* derBiases, const float* logSums, float factor, bool firstThere) {
  const Plan& p = c.p;
  const int N = c.g->N, D = c.g->D;
  const Matrix Xw = {c.ws + p.xw, p.xPitch, 0, N};
  for (int k = 0; k < p.pieces; ++k) {
    const int first = k * p.piece, count = c.classes(k), columns = (count + 63) / 64 * 64;
    pack_piece(c, k, k == 0 && firstThere);
    ProbabilitiesEnd e;
    e.z = scores_of<TYPE>(c, k);
    e.out = (unsigned short*)(c.ws + p.p);
    e.pitch = p.pPitch;
    e.labels = c.labels; e.weights = c.weights; e.logSums = logSums;
    e.nWeights = c.nWeights; e.classes = c.g->K;
    e.sums = !derBiases ? nullptr : p.tileRows > 1 ? (float*)(c.ws + p.columns) : derBiases;
    e.factor = factor;
    int rc = product<TYPE, false, false>(c.s, c.who, "fc_probabilities", c.X(), c.F(k), N, columns, p.scores.of(N, columns), c.scratch(), e);
    if (rc) return rc;
    const Matrix P = {c.ws + p.p, p.pPitch, 0, N};
    if (derInput) {
      // (the pieces add up in single precision: in derInput itself, or beside it)
      float* sum = TYPE == kPairs ? (float*)derInput : (float*)(c.ws + p.sum);
      const bool last = k == p.pieces - 1;
      const StoreEnd d = {TYPE == kPairs || last ? derInput : sum, TYPE == kBf16 && last, k > 0 ? sum : nullptr, N, D, factor,
                          TYPE == kPairs ? &c.magnitudes()->filters : nullptr, c.labels, c.weights, c.nWeights};
      ProductPlan q = p.dx;
      q.stages = div_up(count, stage_depth(TYPE));
      rc = product<TYPE, false, true>(c.s, c.who, "fc_derivative_x", P, c.F(k), N, D, q, c.scratch(), d);
      if (rc) return rc;
    }
    if (derFilters) {
      const StoreEnd d = {(void*)c.piece_of(derFilters, first), TYPE == kBf16, nullptr, count, D, factor,
                          TYPE == kPairs ? &c.magnitudes()->features : nullptr, nullptr, nullptr, 1};
      rc = product<TYPE, true, true>(c.s, c.who, "fc_derivative_f", P, Xw, count, D, p.df.of(count, D), c.scratch(), d);
      if (rc) return rc;
    }
  }
  if (derBiases && p.tileRows > 1) {
    KernelTimer timer("fc_join", c.s);
    hipLaunchKernelGGL(fc_join_columns, dim3((unsigned)div_up(c.g->K, 256)), dim3(256), 0, c.s, derBiases, (const float*)(c.ws + p.columns), c.g->K, p.tileRows);
  }
  return check_launch(c.who);
}

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_fcloss_workspace_bytes(const mcn_fcloss_geom* g, int backward) {
  if (!g || g->D <= 0 || g->K <= 0 || g->N <= 0 || g->D > (1 << 20) || g->K > (1 << 24) || g->N > (1 << 30)) return 0;
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return 0;
  // (the largest of the ways the tensors can be aligned)
  const void* odd = (const void*)2;
  size_t most = 0;
  for (int k = 0; k < 4; ++k) most = std::max(most, make_plan(g, k & 1 ? odd : nullptr, k & 2 ? odd : nullptr, backward != 0).total);
  return most;
}

int mcn_fcloss_forward(mcn_stream_t stream, const mcn_fcloss_geom* g, float* y, float* logSums, const void* x, const void* filters,
                       const float* biases, const float* labels, size_t nLabels, const float* instanceWeights, size_t nWeights, void* workspace,
                       size_t workspaceBytes) {
  const char* who = "mcn_fcloss_forward";
  int rc = check(who, g, nLabels, instanceWeights, nWeights);
  if (rc) return rc;
  if (!y) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null output", who);
  if (g->N == 0) {
    hipLaunchKernelGGL(fc_zero, dim3(1), dim3(256), 0, as_stream(stream), y, (size_t)1, 0);
    return check_launch(who);
  }
  if (!x || !filters || !labels) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  const Call c = {as_stream(stream), who, g, x, filters, biases, labels, instanceWeights, (int)nWeights, (char*)workspace, make_plan(g, x, filters, false)};
  if (!workspace || workspaceBytes < c.p.total)
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, c.p.total);
  if (!aligned16(workspace)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the workspace is not 16-byte aligned", who);
  rc = prepare(c, false);
  if (rc) return rc;
  float* sums = logSums ? logSums : (float*)(c.ws + c.p.logSums);
  return c.p.type == kPairs ? forward<kPairs>(c, y, sums) : forward<kBf16>(c, y, sums);
}

int mcn_fcloss_backward(mcn_stream_t stream, const mcn_fcloss_geom* g, void* derInput, void* derFilters, float* derBiases, const float* logSums,
                        const void* x, const void* filters, const float* biases, const float* labels, size_t nLabels, const float* instanceWeights,
                        size_t nWeights, double derOutput, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_fcloss_backward";
  int rc = check(who, g, nLabels, instanceWeights, nWeights);
  if (rc) return rc;
  if (!derInput && !derFilters && !derBiases) return MCN_SUCCESS;
  if (g->N == 0) {   // sums over no images
    const size_t n = (size_t)g->K * g->D;
    if (derFilters && n)
      hipLaunchKernelGGL(fc_zero, dim3((unsigned)std::min<size_t>(4096, (n + 1023) / 1024)), dim3(256), 0, as_stream(stream), derFilters, n, g->dataType == MCN_BFLOAT16);
    if (derBiases && g->K)
      hipLaunchKernelGGL(fc_zero, dim3((unsigned)((g->K + 1023) / 1024)), dim3(256), 0, as_stream(stream), derBiases, (size_t)g->K, 0);
    return check_launch(who);
  }
  if (!x || !filters || !labels) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  const Call c = {as_stream(stream), who, g, x, filters, biases, labels, instanceWeights, (int)nWeights, (char*)workspace, make_plan(g, x, filters, true)};
  if (!workspace || workspaceBytes < c.p.total)
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, c.p.total);
  if (!aligned16(workspace)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the workspace is not 16-byte aligned", who);
  rc = prepare(c, derFilters != nullptr);
  if (rc) return rc;
  const float factor = (float)(g->normalise ? derOutput / g->N : derOutput);
  const bool recompute = logSums == nullptr;
  if (recompute) {
    float* sums = (float*)(c.ws + c.p.logSums);
    rc = c.p.type == kPairs ? forward<kPairs>(c, nullptr, sums) : forward<kBf16>(c, nullptr, sums);
    if (rc) return rc;
    logSums = sums;
  }
  // (with more than one piece the log sums' pass leaves the last one's filters behind)
  const bool there = !recompute || c.p.pieces == 1;
  return c.p.type == kPairs ? backward<kPairs>(c, derInput, derFilters, derBiases, logSums, factor, there)
                            : backward<kBf16>(c, derInput, derFilters, derBiases, logSums, factor, there);
}

}  // extern "C"
