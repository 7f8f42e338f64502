// A fully connected layer and the softmax cross entropy behind it as one operator: the scores of N instances for K classes are made in
// pieces of the classes and never kept.
//
//   z = x f + b, y = sum_n w_n (log sum_k exp z_nk - z_n,c(n)) [/ N],  P = softmax(z) - (1 at c(n)),
//   dzdx = sum_k w P f, dzdf = sum_n w P x, dzdb = sum_n w P   (times the scalar derivative of y [/ N])
//
// Forward: every tile of scores leaves, per instance, its largest score and the sum of exponentials against it; a pass over those
// (8 bytes for 64 to 256 scores) gives the logarithms of the sums.  Backward: a piece of the classes at a time, the scores are made
// again, P is written as operands, and two products over it give the piece's dzdf and its share of dzdx.  The largest buffers are the
// piece's P and, where instances times classes are very many, the tiles' leavings over all classes.  8 N D K operations in all, a
// quarter of them the scores made again: keeping N x K scores is what this operator is there to avoid.
//
// Single precision (pairs, product.hpp).  What shares a power of two as its scale decides what is lost, so each product has its own:
//   scores  an instance's features, a class's filter: e_n and e_k, the exponents of their largest magnitudes;
//   dzdf    (sum over n) a class's w P 2^e_n, a feature's x 2^-e_n over the instances: C_k and S_d, the exponents of the largest;
//   dzdx    (sum over k) an instance's w P 2^e_k: R_n; the filters as in the scores.
// So a class that is hardly ever likely, a feature that is small for all instances, a small filter or instance costs nobody anything.  P is
// made in single precision first, with the magnitudes for R and C on the way (maxima by atomics: the order does not matter), and split by
// them in a pass of its own (fc_split).
#include "product.hpp"

#include <algorithm>

namespace mcn {
namespace {

__device__ __forceinline__ float instance_weight(const float* labels, const float* weights, int nWeights, int n) {
  return labels[n] != 0.f ? (weights ? weights[n % nWeights] : 1.f) : 0.f;
}
__device__ __forceinline__ int class_of(float label, int K) { return label >= 1.f ? min((int)fminf(label, 2147483520.f) - 1, K - 1) : 0; }

// ---------------------------------------------------------------------------------------------- operands

__device__ __forceinline__ unsigned wave_most(unsigned m, int lanes) {   // over groups of `lanes` neighbours
  for (int o = lanes / 2; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, kWave));
  return m;
}

// Largest magnitudes, as the bits of floats
__device__ __forceinline__ void raise(unsigned* at, unsigned bits) {
  if (bits) __hip_atomic_fetch_max(at, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void clear_words(unsigned* words, size_t n) {   // by all workgroups of 256
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) words[i] = 0;
}

// Single precision: rows as pairs, each by its own magnitude.  `lanes` neighbours share a row (one pack of eight values each where that is
// enough); rows of up to kHeld packs a lane are read once.
struct RowsPart {
  const float* x;
  unsigned short* out;
  int* exponents;
  int rows;
  unsigned firstGroup, groups;
};
struct RowsJob {
  RowsPart parts[2];
  int nParts, D, lanes;
  long long pitch;
  unsigned* clear;             // counters and magnitudes, cleared on the way
  size_t nClear;
};
constexpr int kHeld = 8;
__global__ __launch_bounds__(256) void fc_pack_rows(RowsJob j) {
  clear_words(j.clear, j.nClear);
  if (j.nParts == 0) return;
  const RowsPart p = j.parts[j.nParts > 1 && blockIdx.x >= j.parts[1].firstGroup ? 1 : 0];
  const int t = (int)threadIdx.x % j.lanes, per = (int)(j.pitch / 16), rows = 256 / j.lanes;
  for (long long first = (long long)(blockIdx.x - p.firstGroup) * rows; first < p.rows; first += (long long)p.groups * rows) {
    const long long row = first + (int)threadIdx.x / j.lanes;
    const bool live = row < p.rows;
    const float* from = p.x + (size_t)(live ? row : 0) * j.D;
    float v[kHeld][8];
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int c = 8 * (t + j.lanes * i);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = 0.f;
      if (8 * j.lanes * i < j.D && live && c < j.D) load8(v[i], from, c, j.D);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(v[i][k]) & 0x7fffffffu);
    for (int i = kHeld; j.lanes * i < per; ++i) {
      const int c = 8 * (t + j.lanes * i);
      float u[8];
      if (live && c < j.D) {
        load8(u, from, c, j.D);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(u[k]) & 0x7fffffffu);
      }
    }
    most = wave_most(most, j.lanes);
    if (!live) continue;
    const int e = exponent_of(most);
    if (t == 0) p.exponents[row] = e;
    unsigned short* const to = p.out + (size_t)row * j.pitch;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int pack = t + j.lanes * i;
      if (j.lanes * i >= per || pack >= per) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = ldexpf(v[i][k], kPairExponent - e);
      store8_pairs(to, 8 * pack, v[i]);
    }
    for (int i = kHeld; j.lanes * i < per; ++i) {
      const int pack = t + j.lanes * i;
      if (pack >= per) continue;
      float u[8] = {};
      if (8 * pack < j.D) load8(u, from, 8 * pack, j.D);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = ldexpf(u[k], kPairExponent - e);
      store8_pairs(to, 8 * pack, u);
    }
  }
}

// S_d: the largest magnitudes of x 2^-e_n over the instances that count.  A wavefront's lanes lie along 512 features, its rows one behind the
// other.
__global__ __launch_bounds__(1024) void fc_feature_magnitudes(unsigned* __restrict__ out, const float* __restrict__ x, const int* __restrict__ exponents,
                                                             const float* __restrict__ labels, const float* __restrict__ weights, int nWeights, int D,
                                                             int N, int rows) {
  __shared__ unsigned joint[16][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)blockIdx.x * 512 + 8 * lane;
  unsigned most[8] = {};
  for (long long k = 0; k < rows; ++k) {
    const long long n = ((long long)blockIdx.y * rows + k) * 16 + wave;
    if (n >= N || instance_weight(labels, weights, nWeights, (int)n) == 0.f) continue;
    const int e = exponents[n];
    if (c >= D) continue;
    float v[8];
    load8(v, x + (size_t)n * D, c, D);
#pragma unroll
    for (int i = 0; i < 8; ++i) most[i] = max(most[i], __float_as_uint(ldexpf(fabsf(v[i]), -e)));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) joint[wave][8 * lane + i] = most[i];
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= 512 || (int)blockIdx.x * 512 + t >= D) return;
  unsigned m = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) m = max(m, joint[w][t]);
  raise(out + (size_t)blockIdx.x * 512 + t, m);
}

// bfloat16: rows at a pitch of whole stages: all of them; those of instances that count (zeros for the others, whatever they hold); or these
// times the instances' weights, which as one bfloat16 value would round dzdf a third time, behind P and before the result, so as two, of each 64
// rows (up to the next multiple: zeros) first the values, then what they miss.  (Weights in P would be rounded with it: without them the
// label's -1, most of P, is exact.)
enum { kAll, kCounting, kWeighted };
struct PackPart {
  const unsigned short* x;
  unsigned short* out;
  long long pitch;
  int rows, form;
  unsigned firstGroup;
};
struct PackJob {
  PackPart parts[3];
  int nParts, D, N;
  const float *labels, *weights;
  int nWeights;
  unsigned* clear;                         // counters, cleared on the way
  size_t nClear;
};
constexpr int kPackSteps = 4;              // times eight values a thread

__global__ __launch_bounds__(256) void fc_pack(PackJob j) {
  clear_words(j.clear, j.nClear);
  const int which = j.nParts > 2 && blockIdx.x >= j.parts[2].firstGroup ? 2 : j.nParts > 1 && blockIdx.x >= j.parts[1].firstGroup ? 1 : 0;
  const PackPart p = j.parts[which];
  // (all of a thread's loads first, not each behind the store before it: 21841 x 1001 values 22 -> 20 us)
  const int per = (int)(p.pitch / 8);
  const size_t all = (size_t)p.rows * per;
  int row[kPackSteps], c[kPackSteps];
  float w[kPackSteps], v[kPackSteps][8];
#pragma unroll
  for (int step = 0; step < kPackSteps; ++step) {
    const size_t i = ((size_t)(blockIdx.x - p.firstGroup) * kPackSteps + step) * 256 + threadIdx.x;
    const bool live = i < all;
    row[step] = live ? (int)(i / per) : -1;
    c[step] = live ? (int)(i - (size_t)row[step] * per) * 8 : 0;
    w[step] = !live ? 0.f : p.form == kAll ? 1.f : row[step] < j.N ? instance_weight(j.labels, j.weights, j.nWeights, row[step]) : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[step][k] = 0.f;
    if (w[step] != 0.f) load8(v[step], p.x + (size_t)row[step] * j.D, c[step], j.D);
  }
#pragma unroll
  for (int step = 0; step < kPackSteps; ++step) {
    if (row[step] < 0) return;
    const float by = p.form == kWeighted ? w[step] : 1.f;
    const size_t out = p.form == kWeighted ? (size_t)(row[step] / 64) * 128 + row[step] % 64 : (size_t)row[step];
    uintx4p h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float u[2] = {v[step][2 * k] * by, v[step][2 * k + 1] * by};
      const unsigned short a = to_bf16(u[0]), b = to_bf16(u[1]);
      h[k] = (unsigned)a | (unsigned)b << 16;
      l[k] = (unsigned)to_bf16(u[0] - from_bf16(a)) | (unsigned)to_bf16(u[1] - from_bf16(b)) << 16;
    }
    *(uintx4p*)(p.out + out * p.pitch + c[step]) = h;
    if (p.form == kWeighted) *(uintx4p*)(p.out + (out + 64) * p.pitch + c[step]) = l;
  }
}

// Single precision: w P, as the scores' product left it, into the two derivatives' operands, and (the first piece) the features over their
// instances' magnitudes and their own.  One of P's operands takes P's place: the 128 bytes of 32 values are 32 h and 32 l, and the four
// threads that hold these values are neighbours of one wavefront, whose loads are all done before its first store.
struct SplitGrid { int lanes, across, down; };   // threads to a row in a workgroup; workgroups to a row, and rows of these
struct SplitJob {
  SplitGrid grid, featureGrid;             // of P, of the features
  float* p;
  unsigned short *forFilters, *forInput;   // may be null; one of them is `p`
  long long pitch;                         // of all three, in 16-bit values
  int N, columns;                          // columns: whole blocks of 32
  const int *instances, *classes;          // e_n, e_k
  const unsigned *classMost, *instanceMost;   // whose exponents are C_k, R_n
  unsigned featureGroup;                   // the first workgroup of the features
  const float* x;
  unsigned short* features;
  long long xPitch;
  int D;
  const unsigned* featureMost;             // ... S_d
  const float *labels, *weights;
  int nWeights;
};
// A thread keeps its eight columns (`lanes` neighbours share a row) and goes over the rows STEPS at a time: their exponents are worked out
// once, and STEPS rows are on their way together.
template <int STEPS>
__global__ __launch_bounds__(256) void fc_split(SplitJob j) {
  const bool features = blockIdx.x >= j.featureGroup;
  const SplitGrid g = features ? j.featureGrid : j.grid;
  const int per = features ? (int)(j.xPitch / 16) : j.columns / 8, group = (int)(blockIdx.x - (features ? j.featureGroup : 0u));
  const int c = 8 * (group % g.across * g.lanes + (int)threadIdx.x % g.lanes), rows = 256 / g.lanes;
  if (c >= 8 * per) return;
  int ck[8], ek[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    ck[k] = features ? (c + k < j.D ? kPairExponent - exponent_of(j.featureMost[c + k]) : 0) : j.forFilters ? kPairExponent - exponent_of(j.classMost[c + k]) : 0;
    ek[k] = !features && j.forInput ? kPairExponent + j.classes[c + k] : 0;
  }
  for (long long first = (long long)(group / g.across) * rows * STEPS + (int)threadIdx.x / g.lanes; first < j.N; first += (long long)g.down * rows * STEPS) {
    float v[STEPS][8];
    int en[STEPS];
    unsigned rn[STEPS];
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      const long long n = first + step * rows;
      const bool live = n < j.N;
      en[step] = live ? j.instances[n] : 0;
      rn[step] = live && j.forInput && !features ? j.instanceMost[n] : 0u;
      if (features) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[step][k] = 0.f;
        if (live && c < j.D && instance_weight(j.labels, j.weights, j.nWeights, (int)n) != 0.f) load8(v[step], j.x + (size_t)n * j.D, c, j.D);
      } else {
        const uintx4p* from = (const uintx4p*)((const char*)j.p + ((size_t)(live ? n : first) * j.pitch + 2 * c) * 2);
        const uintx4p a = from[0], b = from[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[step][k] = __uint_as_float(a[k]);
          v[step][4 + k] = __uint_as_float(b[k]);
        }
      }
    }
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      const long long n = first + step * rows;
      if (n >= j.N) break;
      float u[8];
      if (features) {
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = ldexpf(v[step][k], ck[k] - en[step]);
        store8_pairs(j.features + (size_t)n * j.xPitch, c, u);
        continue;
      }
      if (j.forFilters) {
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = ldexpf(v[step][k], ck[k] + en[step]);
        store8_pairs(j.forFilters + (size_t)n * j.pitch, c, u);
      }
      if (j.forInput) {
        const int e = exponent_of(rn[step]);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = ldexpf(v[step][k], ek[k] - e);
        store8_pairs(j.forInput + (size_t)n * j.pitch, c, u);
      }
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

// What the scores need: z = acc * 2^(e_n + e_k - 28) + bias[k], -infinity behind the piece's last class
struct Scores {
  const int *instances, *classes;  // e_n and the piece's e_k (that of the filters' places up to whole tiles); bfloat16: null
  const float* bias;
  int N, K, first;                 // instances, classes in this piece, the piece's first class
  template <class S>
  __device__ __forceinline__ void make(floatx16p (&acc)[S::TM][S::TN], int m0, int n0, int tileEnd) const {
    if (S::type == kPairs) {
      // (one exact step: the two scales one after the other could leave the range and come back)
      int e[S::TM];
#pragma unroll
      for (int i = 0; i < S::TM; ++i) e[i] = instances[min(m0 + 32 * i, N - 1)] - 2 * kPairExponent;
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int4 k = *(const int4*)(classes + n0 + 32 * j + 8 * q);
          const int ek[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int i = 0; i < S::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][4 * q + r] = ldexpf(acc[i][j][4 * q + r], e[i] + ek[r]);
          __builtin_amdgcn_sched_barrier(0);   // (not all blocks' exponents at once: there are no registers for them)
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

// Forward: (largest score, sum of exponentials against it) per instance and tile, the score of the instance's class.  (__expf, here and
// for P, is off by 2^-24 of its argument's size, relative to its value; the roundings of the score and the log sum, whose difference
// the argument is, make as much of it.)
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

// One of two registers goes to the lane h away, the other stays.  (The empty assembly keeps the two apart: from a choice between two entries of
// an array the compiler makes an index, and of that a comparison with every entry: P's kernel took 588 us for 32000 classes, 500 so, and 92 for
// 21841 in bfloat16, 72 so.)
__device__ __forceinline__ void choose(bool upper, float& give, float& keep) {
  float a = give, b = keep;
  asm("" : "+v"(a), "+v"(b));
  give = upper ? a : b;
  keep = upper ? b : a;
}

// Sums over the 32 lanes of a half-wavefront of N values a lane (N a power of two, at most 32): lane l of the half ends up with the sum of
// value l % N.  Every exchange halves what is left to add: 31 exchanges for 32 values, where adding each across takes 160.
template <int N>
__device__ __forceinline__ float lanes_fold(float (&v)[N], int lane) {
#pragma unroll
  for (int h = N / 2; h >= 1; h >>= 1) {
#pragma unroll
    for (int k = 0; k < h; ++k) {
      float give = v[k], keep = v[k + h];
      choose((lane & h) != 0, give, keep);
      v[k] = keep + __shfl_xor(give, h, kWave);
    }
  }
  float s = v[0];
#pragma unroll
  for (int o = N; o < 32; o <<= 1) s += __shfl_xor(s, o, kWave);
  return s;
}

// The same for the largest
template <int N>
__device__ __forceinline__ float lanes_most(float (&v)[N], int lane) {
#pragma unroll
  for (int h = N / 2; h >= 1; h >>= 1) {
#pragma unroll
    for (int k = 0; k < h; ++k) {
      float give = v[k], keep = v[k + h];
      choose((lane & h) != 0, give, keep);
      v[k] = fmaxf(keep, __shfl_xor(give, h, kWave));
    }
  }
  float m = v[0];
#pragma unroll
  for (int o = N; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
  return m;
}

// Backward: P, and the columns' sums of w P, one per tile.  bfloat16: P as the operand of two products (the instances' weights go into the
// other operand, or the result).  Single precision: w P itself, and the exponents that it is split by.
struct ProbabilitiesEnd {
  Scores z;
  void* out;
  long long pitch;                 // in 16-bit values
  const float *labels, *weights, *logSums;
  int nWeights, classes;
  float* sums;                     // [tile rows][classes], times `factor`; may be null
  float factor;
  unsigned *classMost, *instanceMost;   // the largest |w P| 2^e_n of a class, |w P| 2^e_k of an instance; null where nobody asks for them
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
    z.make<S>(acc, m0, n0, (tn + 1) * S::BN);
    constexpr bool pairs = S::type == kPairs;
    unsigned* magnitudes = (unsigned*)(lds + S::ldsBytes - 2 * S::WM * S::BN * 4);  // [WM][BN]
    float* columns = (float*)(lds + S::ldsBytes - S::WM * S::BN * 4);         // [WM][BN]
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
      if (pairs && weights) {
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] *= w;
      }
      if (__any(w == 0.f)) {       // (such an instance's scores may be anything)
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = w == 0.f ? 0.f : acc[i][j][r];
      }
    }
    if (pairs && (classMost || instanceMost)) {
      // (magnitudes that leave the range here do so in the derivatives)
      int en[S::TM];
      float most[S::TM];
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        en[i] = z.instances[min(m0 + 32 * i, z.N - 1)];
        most[i] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        float v[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int4 k = *(const int4*)(z.classes + n0 + 32 * j + 8 * q);
          const int ek[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < S::TM; ++i) {
              const float p = acc[i][j][4 * q + r];
              m = fmaxf(m, fabsf(ldexpf(p, en[i])));
              most[i] = fmaxf(most[i], fabsf(ldexpf(p, ek[r])));
            }
            v[4 * q + r] = m;
          }
        }
        const unsigned m = __float_as_uint(lanes_most<16>(v, lane));
        const int r = lane & 15;
        if ((lane & 16) == 0) magnitudes[wm * S::BN + 32 * (wn * S::TN + j) + 8 * (r / 4) + 4 * (lane >> 5) + r % 4] = m;
        __builtin_amdgcn_sched_barrier(0);   // (nor all blocks' exchanges: 1200 registers went to memory, 2.2 ms for 32000 classes instead of 1.7)
      }
      if (instanceMost) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i) {
          const float m = fmaxf(most[i], __shfl_xor(most[i], 32, kWave));
          if (lane < 32 && m0 + 32 * i < z.N) raise(instanceMost + m0 + 32 * i, __float_as_uint(m));
        }
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
          for (int i = 0; i < S::TM; ++i) v[r] += pairs ? acc[i][j][r] : weight[i] * acc[i][j][r];
        }
        const float s = lanes_fold<16>(v, lane);
        const int r = lane & 15;
        if ((lane & 16) == 0) columns[wm * S::BN + 32 * (wn * S::TN + j) + 8 * (r / 4) + 4 * (lane >> 5) + r % 4] = s;
      }
    }
    const bool raising = pairs && classMost;
    if (sums || raising) {
      __syncthreads();
      for (int t = threadIdx.x; t < S::BN; t += S::threads) {
        const int n = tn * S::BN + t;
        if (n >= z.K) continue;
        if (sums) {
          float s = columns[t];
#pragma unroll
          for (int w = 1; w < S::WM; ++w) s += columns[w * S::BN + t];
          sums[(size_t)tm * classes + z.first + n] = s * factor;
        }
        if (raising) {
          unsigned m = magnitudes[t];
#pragma unroll
          for (int w = 1; w < S::WM; ++w) m = max(m, magnitudes[w * S::BN + t]);
          raise(classMost + n, m);
        }
      }
    }
    constexpr int size = pairs ? 4 : 2, J = turned_blocks<S, size>();
    const RowTurn<J * 32 * size> turn(lds, wn * S::WM + wm);
    static_assert(S::WM * S::WN * RowTurn<J * 32 * size>::size + 2 * S::WM * S::BN * 4 <= S::ldsBytes, "beside the columns and the magnitudes");
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
            if (pairs) {
              *(float4*)turn.at(l32, 128 * j + 4 * column) = make_float4(a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]);
            } else {
              unsigned h[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) h[r] = to_bf16(a[4 * q + r]);
              *(uintx2p*)turn.at(l32, 64 * j + 2 * column) = (uintx2p){h[0] | h[1] << 16, h[2] | h[3] << 16};
            }
          }
        const int m1 = tm * S::BM + 32 * (wm * S::TM + i), start = (first + 32 * j0) * size;   // bytes from the row's first class
        turn.each(lane, [&](int row, int offset, uintx4p v) {
          if (m1 + row < z.N && start + offset < 2 * pitch) *(uintx4p*)((char*)out + (size_t)(m1 + row) * pitch * 2 + start + offset) = v;
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
  const unsigned *rowMost, *columnMost;   // pairs: the magnitudes whose exponents the rows and (may be null) the columns were scaled by
  const float *labels, *weights;      // bfloat16, rows that are instances; or null
  int nWeights;
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int, int lane, int wm, int wn, char* lds) const {
    const bool wide = (Ncols & 3) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)sum & 15) == 0;
    constexpr int J = turned_blocks<S, 4>();
    const RowTurn<J * 128> turn(lds, wn * S::WM + wm);
    const int half = lane >> 5, l32 = lane & 31;
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m1 = tm * S::BM + 32 * (wm * S::TM + i);
      const float w = labels && m1 + l32 < M ? instance_weight(labels, weights, nWeights, m1 + l32) * factor : factor;
      const int e = S::type == kPairs ? (m1 + l32 < M ? exponent_of(rowMost[m1 + l32]) : 0) - 2 * kPairExponent : 0;
#pragma unroll
      for (int j0 = 0; j0 < S::TN; j0 += J) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx16p& a = acc[i][j0 + j];
            float4 v = make_float4(a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]);
            if (S::type == kPairs) {   // (one exact step, and before the factor: nothing leaves the range on the way)
              int4 k = {};
              if (columnMost) {
                const uint4 c = *(const uint4*)(columnMost + tn * S::BN + 32 * (wn * S::TN + j0 + j) + 8 * q + 4 * half);
                k = make_int4(exponent_of(c.x), exponent_of(c.y), exponent_of(c.z), exponent_of(c.w));
              }
              v = make_float4(ldexpf(v.x, e + k.x), ldexpf(v.y, e + k.y), ldexpf(v.z, e + k.z), ldexpf(v.w, e + k.w));
            }
            *(float4*)turn.at(l32, 128 * j + 32 * q + 16 * half) = make_float4(v.x * w, v.y * w, v.z * w, v.w * w);
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
  ProductPlan dfWeighted;          // bfloat16: over weighted features in two parts
  long long weightedRows;
  size_t x, xExponents, xw, f, fExponents, cleared, parts, own, terms, logSums, p, p2, sum, columns, products, total;
  int nCounters, tileRows;         // (counters: the last is fc_log_sums')
  // words that are cleared before they are used: counters; S_d; and, by piece, R_n and C_k
  size_t featureMost, instanceMost, classMost, words;
  // workgroups that pack eight values a thread, a few times
  unsigned pack_groups(long long rows, long long packs) const { return (unsigned)((rows * packs + 256 * kPackSteps - 1) / (256 * kPackSteps)); }
};

// A piece's P (single precision: each of its two), or packed filters: larger ones save passes over the sums of dzdx (128, 256, 512 MiB: 29.5,
// 29.5, 29.2 ms for 128000 classes in bfloat16; in single precision, before P was split in a pass of its own, 1.76, 1.72, 1.72 ms for 32000)
size_t piece_bytes() {
  const int kib = tunable("fcloss_piece_kib", 0);
  return kib > 0 ? (size_t)kib << 10 : (size_t)256 << 20;
}

Plan make_plan(const mcn_fcloss_geom* g, const void* x, const void* f, bool backward) {
  Plan p;
  p.type = g->dataType == MCN_BFLOAT16 ? kBf16 : kPairs;
  const bool whole = p.type == kBf16 && g->D % 64 == 0, pairs = p.type == kPairs;
  p.fInPlace = whole && aligned16(f);
  p.xInPlace = whole && aligned16(x);
  p.xPitch = row_halves(p.type, g->D);
  p.fPitch = p.fInPlace ? g->D : row_halves(p.type, g->D);
  // a piece: P (backward) and the packed filters stay within piece_bytes(), whole tiles
  const long long most = (g->K + 255ll) / 256 * 256;
  const long long perClass = std::max<long long>(backward ? g->N * 2ll * (pairs ? 2 : 1) : 0, p.fInPlace ? 0 : p.fPitch * 2);
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
  p.weightedRows = pairs ? 0 : (g->N + 63ll) / 64 * 128;
  p.dfWeighted = pairs ? p.df : plan_product(p.type, classes, g->D, p.weightedRows);
  p.tiles = div_up(g->K, kTileSize[p.scores.tile]);
  p.pPitch = row_halves(p.type, std::min<long long>(p.piece, (g->K + 63) / 64 * 64));
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const auto whole_tiles = [](size_t n) { return (n + 255) / 256 * 256; };
  p.tileRows = div_up(g->N, kTileSize[p.scores.tile]);
  p.nCounters = 1 + (int)(backward ? std::max({p.scores.counters(), p.dx.counters(), p.df.counters(), p.dfWeighted.counters()}) : p.scores.counters());
  p.featureMost = whole_tiles((size_t)p.nCounters);
  p.instanceMost = p.featureMost + (pairs && backward ? whole_tiles((size_t)g->D) : 0);
  p.classMost = p.instanceMost + (pairs && backward ? whole_tiles((size_t)g->N) : 0);
  p.words = p.classMost + (pairs && backward ? (size_t)p.piece : 0);
  p.cleared = take(4 * p.words);
  p.xExponents = take(pairs ? (size_t)g->N * 4 : 0);
  p.fExponents = take(pairs ? whole_tiles((size_t)g->K) * 4 : 0);
  p.products = take(backward ? std::max({p.scores.partBytes(), p.dx.partBytes(), p.df.partBytes(), p.dfWeighted.partBytes()}) : p.scores.partBytes());
  p.x = take(p.xInPlace ? 0 : (size_t)g->N * p.xPitch * 2);
  p.f = take(p.fInPlace ? 0 : (size_t)std::min(p.piece, g->K) * p.fPitch * 2);
  p.parts = take((size_t)g->N * p.tiles * 8);
  p.own = take((size_t)g->N * 4);
  p.terms = take((size_t)g->N * 4);
  p.logSums = take((size_t)g->N * 4);
  p.xw = p.p = p.p2 = p.sum = p.columns = 0;
  if (backward) {
    p.xw = take((size_t)(pairs ? g->N : p.weightedRows) * p.xPitch * 2);
    p.columns = take(p.tileRows > 1 ? (size_t)p.tileRows * g->K * 4 : 0);
    p.p = take((size_t)g->N * p.pPitch * 2);
    p.p2 = take(pairs ? (size_t)g->N * p.pPitch * 2 : 0);
    p.sum = take(!pairs && p.pieces > 1 ? (size_t)g->N * g->D * 4 : 0);
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
  unsigned* words(size_t at) const { return (unsigned*)(ws + p.cleared) + at; }
  Scratch scratch() const { return {(float*)(ws + p.products), words(0)}; }
  int* instances() const { return (int*)(ws + p.xExponents); }
  int* classExponents(int piece) const { return (int*)(ws + p.fExponents) + (size_t)piece * p.piece; }
  Matrix X() const { return {p.xInPlace ? x : ws + p.x, p.xPitch, 0, g->N}; }
  const char* piece_of(const void* t, int first) const { return (const char*)t + (size_t)first * g->D * (p.type == kPairs ? 4 : 2); }
  int classes(int piece) const { return std::min(p.piece, g->K - piece * p.piece); }
  Matrix F(int piece) const { return {p.fInPlace ? piece_of(filters, piece * p.piece) : ws + p.f, p.fPitch, 0, classes(piece)}; }
};

// The filters of a piece and, before the first (`all`), the features, where the products read them; the words that the piece's products count and
// take maxima in are cleared, all of them before the first.  `derived`: bfloat16 features for dzdf too; without weights, where they are
// copied anyway, one copy serves both (behind the forward call it does not matter what the scores of instances that do not count are
// made of).
void pack(const Call& c, int piece, bool all, bool derived) {
  const Plan& p = c.p;
  const int D = c.g->D, N = c.g->N;
  unsigned groups = 0;
  const auto at = [&](unsigned n) {
    const unsigned first = groups;
    groups += n;
    return first;
  };
  const size_t from = all ? 0 : p.instanceMost;
  unsigned* const clear = c.words(from);
  const size_t nClear = p.words - from;
  if (p.type == kPairs) {
    RowsJob j = {};
    j.D = D;
    j.pitch = p.xPitch;
    j.lanes = 1;
    while (j.lanes < 64 && j.lanes < j.pitch / 16) j.lanes *= 2;
    j.clear = clear; j.nClear = nClear;
    const auto rows = [&](const void* x, size_t out, int* exponents, int n) {
      const unsigned blocks = (unsigned)std::min<long long>(1 << 22, div_up(n, 256 / j.lanes));
      j.parts[j.nParts++] = {(const float*)x, (unsigned short*)(c.ws + out), exponents, n, at(blocks), blocks};
    };
    rows(c.piece_of(c.filters, piece * p.piece), p.f, c.classExponents(piece), c.classes(piece));
    if (all) rows(c.x, p.x, c.instances(), N);
    KernelTimer timer("fc_pack", c.s);
    hipLaunchKernelGGL(fc_pack_rows, dim3(groups), dim3(256), 0, c.s, j);
    return;
  }
  PackJob j = {};
  j.D = D; j.N = N;
  j.labels = c.labels; j.weights = c.weights; j.nWeights = c.nWeights;
  j.clear = clear; j.nClear = nClear;
  const auto rows = [&](const void* x, size_t out, long long pitch, int n, int form) {
    j.parts[j.nParts++] = {(const unsigned short*)x, (unsigned short*)(c.ws + out), pitch, n, form, at(p.pack_groups(n, pitch / 8))};
  };
  if (!p.fInPlace) rows(c.piece_of(c.filters, piece * p.piece), p.f, p.fPitch, c.classes(piece), kAll);
  if (all && !p.xInPlace) rows(c.x, p.x, p.xPitch, N, derived && !c.weights ? kCounting : kAll);
  if (all && derived && c.weights) rows(c.x, p.xw, p.xPitch, (int)(p.weightedRows / 2), kWeighted);
  else if (all && derived && p.xInPlace) rows(c.x, p.xw, p.xPitch, N, kCounting);
  if (groups == 0) {
    if (nClear == 0) return;       // (filters in place)
    groups = 1;                    // (the counters alone)
  }
  KernelTimer timer("fc_pack", c.s);
  hipLaunchKernelGGL(fc_pack, dim3(groups), dim3(256), 0, c.s, j);
}

template <int TYPE>
Scores scores_of(const Call& c, int piece) {
  return {TYPE == kPairs ? c.instances() : nullptr, TYPE == kPairs ? c.classExponents(piece) : nullptr, c.biases, c.g->N, c.classes(piece), piece * c.p.piece};
}

// Single precision: w P of a piece into the operands of the derivatives that are wanted, and before the first piece's the features into dzdf's
void split(const Call& c, int piece, bool forInput, bool forFilters) {
  const Plan& p = c.p;
  SplitJob j = {};
  j.p = (float*)(c.ws + p.p);
  j.forInput = forInput ? (unsigned short*)(c.ws + p.p) : nullptr;
  j.forFilters = !forFilters ? nullptr : (unsigned short*)(c.ws + (forInput ? p.p2 : p.p));
  j.pitch = p.pPitch;
  j.N = c.g->N; j.columns = (c.classes(piece) + 31) / 32 * 32;
  j.instances = c.instances(); j.classes = c.classExponents(piece);
  j.classMost = c.words(p.classMost); j.instanceMost = c.words(p.instanceMost);
  j.x = (const float*)c.x; j.features = (unsigned short*)(c.ws + p.xw); j.xPitch = p.xPitch; j.D = c.g->D;
  j.featureMost = c.words(p.featureMost);
  j.labels = c.labels; j.weights = c.weights; j.nWeights = c.nWeights;
  // (2048 x 32000 values: two rows at a time 247 us, four 190, eight 165, and by eight workgroups to a unit that go on down the rows 153, 5.1
  // TB/s; few values: one, so that there are workgroups for all units)
  const int steps = (long long)j.N * (j.columns + p.xPitch / 2) >= 4ll << 20 ? 8 : 1;
  unsigned groups = 0;
  const auto plan = [&](long long packs) {
    SplitGrid g = {4, 0, 0};
    while (g.lanes < 256 && g.lanes < packs) g.lanes *= 2;
    g.across = div_up(packs, g.lanes);
    g.down = (int)std::min<long long>(div_up(j.N, 256 / g.lanes * steps), std::max(1, 2048 / g.across));
    groups += (unsigned)g.across * (unsigned)g.down;
    return g;
  };
  j.grid = plan(j.columns / 8);
  j.featureGroup = groups;
  if (forFilters && piece == 0) j.featureGrid = plan(p.xPitch / 16);
  KernelTimer timer("fc_split", c.s);
  if (steps == 1) hipLaunchKernelGGL(fc_split<1>, dim3(groups), dim3(256), 0, c.s, j);
  else hipLaunchKernelGGL(fc_split<8>, dim3(groups), dim3(256), 0, c.s, j);
}

// y may be null (the log sums alone)
template <int TYPE>
int forward(const Call& c, float* y, float* logSums) {
  const Plan& p = c.p;
  const int N = c.g->N;
  for (int k = 0; k < p.pieces; ++k) {
    if (k > 0) pack(c, k, false, false);
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
                       c.words((size_t)p.nCounters - 1), (const float2*)(c.ws + p.parts), (const float*)(c.ws + p.own), c.labels, c.weights,
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
  const bool pairs = TYPE == kPairs;
  const bool weighted = !pairs && c.weights;
  const Matrix Xf = weighted ? Matrix{c.ws + p.xw, p.xPitch, 0, p.weightedRows} : Matrix{c.ws + (pairs || p.xInPlace ? p.xw : p.x), p.xPitch, 0, N};
  if (pairs && derFilters) {
    const int columns = div_up(D, 512), rows = std::max(1, div_up((long long)N * columns, 16 * 512));   // (some 512 workgroups)
    KernelTimer timer("fc_feature_magnitudes", c.s);
    hipLaunchKernelGGL(fc_feature_magnitudes, dim3((unsigned)columns, (unsigned)div_up(N, 16ll * rows)), dim3(1024), 0, c.s, c.words(p.featureMost),
                       (const float*)c.x, c.instances(), c.labels, c.weights, c.nWeights, D, N, rows);
  }
  for (int k = 0; k < p.pieces; ++k) {
    const int first = k * p.piece, count = c.classes(k), columns = (count + 63) / 64 * 64;
    if (k > 0 || !firstThere) pack(c, k, false, false);
    ProbabilitiesEnd e;
    e.z = scores_of<TYPE>(c, k);
    e.out = c.ws + p.p;
    e.pitch = p.pPitch;
    e.labels = c.labels; e.weights = c.weights; e.logSums = logSums;
    e.nWeights = c.nWeights; e.classes = c.g->K;
    e.sums = !derBiases ? nullptr : p.tileRows > 1 ? (float*)(c.ws + p.columns) : derBiases;
    e.factor = factor;
    e.classMost = pairs && derFilters ? c.words(p.classMost) : nullptr;
    e.instanceMost = pairs && derInput ? c.words(p.instanceMost) : nullptr;
    int rc = product<TYPE, false, false>(c.s, c.who, "fc_probabilities", c.X(), c.F(k), N, columns, p.scores.of(N, columns), c.scratch(), e);
    if (rc) return rc;
    if (pairs && (derInput || derFilters)) split(c, k, derInput != nullptr, derFilters != nullptr);
    const Matrix P = {c.ws + p.p, p.pPitch, 0, N};
    if (derInput) {
      // (the pieces add up in single precision: in derInput itself, or beside it)
      float* sum = pairs ? (float*)derInput : (float*)(c.ws + p.sum);
      const bool last = k == p.pieces - 1;
      const StoreEnd d = {pairs || last ? derInput : sum, !pairs && last, k > 0 ? sum : nullptr, N, D, factor, c.words(p.instanceMost), nullptr,
                          pairs ? nullptr : c.labels, c.weights, c.nWeights};
      ProductPlan q = p.dx;
      q.stages = div_up(count, stage_depth(TYPE));
      rc = product<TYPE, false, true>(c.s, c.who, "fc_derivative_x", P, c.F(k), N, D, q, c.scratch(), d);
      if (rc) return rc;
    }
    if (derFilters) {
      const StoreEnd d = {(void*)c.piece_of(derFilters, first), !pairs, nullptr, count, D, factor, c.words(p.classMost), c.words(p.featureMost), nullptr, nullptr, 1};
      const Matrix Pf = {c.ws + (pairs && derInput ? p.p2 : p.p), p.pPitch, 0, N};
      if constexpr (TYPE == kBf16)
        rc = weighted ? product<TYPE, true, true, 2>(c.s, c.who, "fc_derivative_f", Pf, Xf, count, D, p.dfWeighted.of(count, D), c.scratch(), d)
                      : product<TYPE, true, true>(c.s, c.who, "fc_derivative_f", Pf, Xf, count, D, p.df.of(count, D), c.scratch(), d);
      else
        rc = product<TYPE, true, true>(c.s, c.who, "fc_derivative_f", Pf, Xf, count, D, p.df.of(count, D), c.scratch(), d);
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
  pack(c, 0, true, false);
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
  pack(c, 0, true, derFilters != nullptr);
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
