// Orthogonalised updates: a matrix G of K filters x D values is replaced by (nearly) the closest one with orthonormal rows or columns, U V'
// of its singular value decomposition U S V', by matrix products alone:
//   X = G/|G|,  five times (or as asked)  X <- a X + (b A + c A^2) X,  A = X X'      (A = X'X and products from the right if K > D)
// Every singular value s goes through p(s) = a s + b s^3 + c s^5; with a = 3.4445, b = -4.7750, c = 2.0315 (K. Jordan et al., "Muon: an
// optimizer for hidden layers in neural networks", 2024) values from 0.005 on end within [0.68, 1.21] after five steps, and none ever
// passes 1.22.  So X, A and B (its eigenvalues lie in [0.6, 3.4445]) stay below 3.5 in magnitude,
// and the operands of the products are pairs of half-precision values (product.hpp) at a scale that is always the same, 2^14
// (3.4445 * 2^14 < 65504): an entry of X is held to 2^-23 of itself or, below 2^-16, to 2^-39.
// A step is three products, in three launches or two (ClosingEnd), for small matrices all steps in one (ortho_narrow): A and A^2 are symmetric, of them only the tiles on and below the diagonal are made and written twice;
// 3 m^2 n + m^3 operations for an m x n matrix, m <= n.  All of a call's matrices (of one size) go through one launch per product.
#include "product.hpp"

#include <climits>

namespace mcn {
namespace {

constexpr float kScale = 16384.f, kUnscale = 1.f / kScale;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kNormParts = 256;   // workgroups per matrix that sum squares, at most

// ---------------------------------------------------------------------------------------------- G to pairs

// sums of squares, in double (single-precision squares of small gradients vanish)
__global__ __launch_bounds__(256) void ortho_squares(double* __restrict__ parts, const float* __restrict__ x, size_t size, unsigned* __restrict__ counters,
                                                     int nCounters) {
  __shared__ double lds[4];
  // (the products' counters are cleared on the way, by the first matrix's workgroups: over all of them, up to 65535 matrices, the threads do
  // not fit an int)
  static_assert(kNormParts * 256ll <= INT_MAX / 2, "a thread's number among those of one matrix, and one stride behind it");
  if (blockIdx.y == 0)
    for (int i = (int)(blockIdx.x * 256 + threadIdx.x); i < nCounters; i += (int)(gridDim.x * 256)) counters[i] = 0;
  const float* v = x + (size_t)blockIdx.y * size;
  double s[4] = {};
  const size_t step = (size_t)gridDim.x * 256;
  size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  for (; i + 7 * step < size; i += 8 * step) {
    float u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = v[i + k * step];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k & 3] += (double)u[k] * (double)u[k];
  }
  for (; i < size; i += step) s[0] += (double)v[i] * (double)v[i];
  const double sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) parts[(size_t)blockIdx.y * kNormParts + blockIdx.x] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}
__device__ __forceinline__ double norm_square(const double* parts, int matrix, int used) {
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kNormParts / 64; ++k) {
    const int i = 64 * k + (threadIdx.x & 63);
    s += i < used ? parts[(size_t)matrix * kNormParts + i] : 0.0;
  }
  return wave_sum(s);
}
__device__ __forceinline__ double norm_factor(double square, double scale) { return square > 0.0 ? scale / sqrt(square) : square; }

// X = G/|G| as pairs, a thread per eight values; the zero matrix stays zero
__global__ __launch_bounds__(256) void ortho_pack(unsigned short* __restrict__ out, const float* __restrict__ x, const double* __restrict__ parts,
                                                  int used, int rows, int cols, long long pitch) {
  const int matrix = blockIdx.y, per = (int)(pitch / 16);
  const double factor = norm_factor(norm_square(parts, matrix, used), (double)kScale);
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)rows * per) return;
  const int row = (int)(i / per), c = (int)(i - (size_t)row * per) * 8;
  const float* from = x + ((size_t)matrix * rows + row) * cols;
  float v[8];
  load8(v, from, c, cols);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (float)((double)v[k] * factor);
  store8_pairs(out + ((size_t)matrix * rows + row) * pitch, c, v);
}

// ---------------------------------------------------------------------------------------------- products

// D = add * C + times * A B + identity, as pairs or as single-precision values
struct OrthoEnd {
  unsigned short* out;      // pairs, at outPitch / outSize
  float* result;            // not null: single precision, rows of `cols` values
  const unsigned short* c;  // pairs of the output's shape; null: nothing is added
  long long pitch, size;
  int rows, cols;
  float add, times;         // (times: with the scales of the two operands)
  float identity;           // on the diagonal, at the output's scale
  int symmetric;            // tiles below the diagonal are written a second time, turned
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int tm, int tn, int which, int lane, int wm, int wn, char*) const {
    const int m0 = tm * S::BM + 32 * wm * S::TM + (lane & 31), n0 = tn * S::BN + 32 * wn * S::TN + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int m = m0 + 32 * i;
      // (the columns behind the last one, up to whole blocks of 32, are zeros: of the part that is written turned, these are rows here)
      const bool live = m < rows;
      if (!live && !(symmetric && tm != tn && 2 * (m / 32 * 32) < pitch)) continue;
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + 32 * j + 8 * q;
          const long long at = which * size + m * pitch + (n / 32) * 64 + n % 32;
          if (n / 32 * 64 >= pitch) continue;
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = acc[i][j][4 * q + r] * times;
          if (c && live) {
            const uintx2p h = *(const uintx2p*)(c + at), l = *(const uintx2p*)(c + at + 32);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const unsigned sh = 16 * (r & 1);
              v[r] += add * (half_bits((unsigned short)(h[r / 2] >> sh)) + half_bits((unsigned short)(l[r / 2] >> sh)));
            }
          }
          if (identity != 0.f) {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += m == n + r ? identity : 0.f;
          }
          if (result) {
            float* o = result + ((long long)which * rows + m) * cols + n;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r < cols) o[r] = v[r] * kUnscale;
            continue;
          }
          unsigned p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = live && n + r < cols ? split_pair(v[r]) : 0u;
          if (live) {
            *(uintx2p*)(out + at) = (uintx2p){(p[0] & 0xffffu) | p[1] << 16, (p[2] & 0xffffu) | p[3] << 16};
            *(uintx2p*)(out + at + 32) = (uintx2p){p[0] >> 16 | (p[1] & 0xffff0000u), p[2] >> 16 | (p[3] & 0xffff0000u)};
          }
          if (symmetric && tm != tn) {
            // (32 lanes hold 32 neighbouring m: the turned rows are written 64 bytes at a time)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (n + r >= rows) continue;
              unsigned short* o = out + which * size + (n + r) * pitch + (m / 32) * 64 + m % 32;
              o[0] = (unsigned short)p[r];
              o[32] = (unsigned short)(p[r] >> 16);
            }
          }
        }
    }
  }
};

// ---------------------------------------------------------------------------------------------- narrow matrices

// Matrices whose shorter side is at most 64 and whose longer one at most 576 (what fits the local memory as pairs): a workgroup each
// goes through all steps in one launch.  (3 banks of 64 filters of 576 values: 106 us through the launches above, 54 here.)  X lies
// in LDS as 64 rows; the reads of one product run along its rows, of the other across them: of every four 64-byte granules
// (32 values' h or l) of a row the order is turned by r % 4, of their 16-byte chunks by r / 4 % 4, which spreads sixteen rows' equal
// chunks, and four rows' equal granules, over all banks.  A, then B lie behind it, rows of 256 bytes, chunks turned by r % 16.
constexpr int kNarrowRows = 64, kNarrowColumns = 576, kNarrowThreads = 512;
constexpr int kSquareBytes = 64 * 256;

__device__ __forceinline__ int narrow_at(int rowBytes, int r, int c, int part) {
  return r * rowBytes + (((2 * (c >> 5) + part) ^ (r & 3)) << 6) + ((((c & 31) >> 3) ^ ((r >> 2) & 3)) << 4) + (c & 7) * 2;
}
__device__ __forceinline__ int square_at(int r, int c, int part) { return r * 256 + (((((c >> 5) << 3) + (part << 2) + ((c & 31) >> 3)) ^ (r & 15)) << 4) + (c & 7) * 2; }

// four neighbours (from a multiple of four on) of a row, as pairs at two addresses
__device__ __forceinline__ void put4(char* h, char* l, const float (&v)[4]) {
  unsigned p[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) p[r] = split_pair(v[r]);
  *(uintx2p*)h = (uintx2p){(p[0] & 0xffffu) | p[1] << 16, (p[2] & 0xffffu) | p[3] << 16};
  *(uintx2p*)l = (uintx2p){p[0] >> 16 | (p[1] & 0xffff0000u), p[2] >> 16 | (p[3] & 0xffff0000u)};
}
__device__ __forceinline__ void get4(const char* h, const char* l, float (&v)[4]) {
  const uintx2p a = *(const uintx2p*)h, b = *(const uintx2p*)l;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    v[r] = half_bits((unsigned short)(a[r / 2] >> (16 * (r & 1)))) + half_bits((unsigned short)(b[r / 2] >> (16 * (r & 1))));
}
// hh + hl + lh of one step of 16 indices, the small ones first
__device__ __forceinline__ floatx16p multiply_pairs(const uintx4p (&a)[2], const uintx4p (&b)[2], floatx16p c) {
  c = multiply<kPairs>(b[0], a[1], c);
  c = multiply<kPairs>(b[1], a[0], c);
  return multiply<kPairs>(b[0], a[0], c);
}

// ---------------------------------------------------------------------------------------------- A and B at once

// Where one tile holds all of A = X X' (m <= 128) the workgroup that finishes it goes on to B = a I + b A + c A^2: A as pairs in LDS, rows of
// 4 BM bytes with their 16-byte chunks turned by r % 16, read along its rows for both operands (it is symmetric).  One launch of three
// less per step, which is what small matrices wait for: 64 x 2000 111 -> 86 us, 120 x 120 93 -> 86.  (Not where the tile of 128's long
// reduction takes longer than three tiles of 64 and a launch: 128 x 4000 185 us by it, 142 without.)
struct ClosingEnd {
  unsigned short* out;      // B as pairs
  long long pitch, size;
  int m;
  template <class S>
  __device__ __forceinline__ void finish(floatx16p (&acc)[S::TM][S::TN], int, int, int which, int lane, int wm, int wn, char* lds) const {
    static_assert(S::BM == S::BN && S::BM * S::BM * 4 <= S::ldsBytes, "A lies in LDS");
    const int half = lane >> 5, l32 = lane & 31, m0 = 32 * wm * S::TM + l32, n0 = 32 * wn * S::TN + 4 * half;
    const auto at = [&](int r, int c, int part) { return lds + r * (S::BM * 4) + (((((c >> 5) << 3) + (part << 2) + ((c & 31) >> 3)) ^ (r & 15)) << 4) + (c & 7) * 2; };
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = m0 + 32 * i, c = n0 + 32 * j + 8 * q;
          float v[4];   // (what stands behind the last row or column of X may belong to other rows)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = r < m && c + e < m ? acc[i][j][4 * q + e] * kUnscale : 0.f;
          put4(at(r, c, 0), at(r, c, 1), v);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = 0.f;
        }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S::BM / 16; ++s) {
      uintx4p a[S::TM][2], b[S::TN][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i) a[i][q] = *(const uintx4p*)at(m0 + 32 * i, 16 * s + 8 * half, q);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) b[j][q] = *(const uintx4p*)at(32 * (wn * S::TN + j) + l32, 16 * s + 8 * half, q);
      }
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] = multiply_pairs(a[i], b[j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = m0 + 32 * i, c = n0 + 32 * j + 8 * q;
          if (r >= m || c / 32 * 64 >= pitch) continue;
          float v[4];
          get4(at(r, c, 0), at(r, c, 1), v);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e] * (kC * kUnscale) + kB * v[e] + (r == c + e ? kA * kScale : 0.f);
          unsigned short* o = out + which * size + r * pitch + (c / 32) * 64 + c % 32;
          put4((char*)o, (char*)(o + 32), v);
        }
  }
};

// m rows (the shorter side), n columns.  FORM: how the matrix lies in memory, 0: rows of n values that can be read 16 bytes at a time,
// 1: rows of n values, 2 (tall): columns of m values.
template <int FORM>
__global__ __launch_bounds__(kNarrowThreads) void ortho_narrow(float* __restrict__ y, const float* __restrict__ x, int m, int n, int steps) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  constexpr bool tall = FORM == 2;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int blocks = (n + 63) / 64 * 2, rowBytes = blocks * 128;   // (blocks of 32 columns, an even number)
  char* const X = lds;
  char* const Q = lds + kNarrowRows * rowBytes;
  x += (size_t)blockIdx.x * m * n;
  y += (size_t)blockIdx.x * m * n;

  // The matrix into registers, four columns a piece: a wavefront takes every eighth row and lanes lie along the columns, or (tall) lanes lie
  // along the rows and a wavefront takes every eighth four columns.
  constexpr int kWaves = kNarrowThreads / 64, kPieces = tall ? kNarrowColumns / 4 / kWaves : kNarrowRows / kWaves * 3;
  static_assert(kNarrowColumns <= 3 * 256 && kNarrowColumns % (4 * kWaves) == 0, "pieces");
  const auto row_of = [&](int k) { return tall ? lane : wave + kWaves * (k / 3); };
  const auto column_of = [&](int k) { return tall ? 4 * (wave + kWaves * k) : 4 * lane + 256 * (k % 3); };
  float v[kPieces][4];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int r = row_of(k), c = column_of(k);
    if (FORM == 0) {
      const float4 t = r < m && c < n ? *(const float4*)(x + r * n + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[k][0] = t.x; v[k][1] = t.y; v[k][2] = t.z; v[k][3] = t.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = r < m && c + e < n ? (tall ? x[(c + e) * m + r] : x[r * n + c + e]) : 0.f;
    }
  }
  // |G|: of the matrix brought near 1 by a power of two (squares stay in range), four squares at a time in single precision, those in
  // double; then everything times 2^14/|G|, that factor as a single-precision value and what it misses
  unsigned most = 0;
#pragma unroll
  for (int k = 0; k < kPieces; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(v[k][e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, o, kWave));
  unsigned* const maxima = (unsigned*)Q;
  double* const sums = (double*)(Q + 4 * kWaves);
  if (lane == 0) maxima[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) most = max(most, maxima[w]);
  const int shift = most == 0 || most >= 0x7f800000u ? 0 : 127 - max(1, (int)(most >> 23));
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    float four = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[k][e] = ldexpf(v[k][e], shift);
      four += v[k][e] * v[k][e];
    }
    sum += (double)four;
  }
  sum = wave_sum(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += sums[w];
  const double factor = norm_factor(sum, (double)kScale);
  const float high = (float)factor, low = (float)(factor - (double)high);
  // X as pairs, zeros around it
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int r = row_of(k), c = column_of(k);
    if (c >= blocks * 32) continue;
    // (zeros stay zeros where the factor is not finite: they lie outside of the matrix)
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = r < m && c + e < n ? fmaf(v[k][e], high, v[k][e] * low) : 0.f;
    put4(X + narrow_at(rowBytes, r, c, 0), X + narrow_at(rowBytes, r, c, 1), u);
  }
  __syncthreads();

  constexpr int kShares = kWaves / 4;
  const int bi = wave & 1, bj = wave >> 1 & 1, share = wave >> 2;   // of A: a block of 32 x 32, and which share of the reduction
  for (int step = 0; step < steps; ++step) {
    // A = X X': the wavefronts kShares to a block, two steps of 16 columns at a time
    floatx16p acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    for (int s = share; s < blocks; s += kShares) {
      uintx4p a[2][2], b[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          a[h][q] = *(const uintx4p*)(X + narrow_at(rowBytes, 32 * bi + l32, 32 * s + 16 * h + 8 * half, q));
          b[h][q] = *(const uintx4p*)(X + narrow_at(rowBytes, 32 * bj + l32, 32 * s + 16 * h + 8 * half, q));
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) acc = multiply_pairs(a[h], b[h], acc);
    }
    const int m0 = 32 * bi + l32, n0 = 32 * bj + 4 * half;   // acc[4 q + r]: (m0, n0 + 8 q + r)
    float* const whole = (float*)Q;                          // [64][64], before A takes its place
    const bool closes = share == kShares - 1;                // (the four wavefronts that hold A in the end)
#pragma unroll
    for (int turn = 0; turn < kShares; ++turn) {
      if (share == turn) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float4* const at = (float4*)(whole + m0 * 64 + n0 + 8 * q);
          const float4 o = turn ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
          acc[4 * q] += o.x; acc[4 * q + 1] += o.y; acc[4 * q + 2] += o.z; acc[4 * q + 3] += o.w;
          if (turn < kShares - 1) *at = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        }
      }
      __syncthreads();
    }
    if (closes) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {acc[4 * q] * kUnscale, acc[4 * q + 1] * kUnscale, acc[4 * q + 2] * kUnscale, acc[4 * q + 3] * kUnscale};
        put4(Q + square_at(m0, n0 + 8 * q, 0), Q + square_at(m0, n0 + 8 * q, 1), v);
      }
    }
    __syncthreads();
    // B = a I + b A + c A^2 (by the same four wavefronts)
    if (closes) {
      floatx16p sq;
#pragma unroll
      for (int r = 0; r < 16; ++r) sq[r] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uintx4p a[2], b[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          a[q] = *(const uintx4p*)(Q + square_at(32 * bi + l32, 16 * s + 8 * half, q));
          b[q] = *(const uintx4p*)(Q + square_at(32 * bj + l32, 16 * s + 8 * half, q));
        }
        sq = multiply_pairs(a, b, sq);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
        get4(Q + square_at(m0, n0 + 8 * q, 0), Q + square_at(m0, n0 + 8 * q, 1), v);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[4 * q + r] = sq[4 * q + r] * (kC * kUnscale) + kB * v[r] + (m0 == n0 + 8 * q + r ? kA * kScale : 0.f);
      }
    }
    __syncthreads();
    if (closes) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        put4(Q + square_at(m0, n0 + 8 * q, 0), Q + square_at(m0, n0 + 8 * q, 1), v);
      }
    }
    __syncthreads();
    // X <- B X: a wavefront takes 32 columns at a time, nobody else reads or writes them
    uintx4p B[2][4][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int q = 0; q < 2; ++q) B[i][k][q] = *(const uintx4p*)(Q + square_at(32 * i + l32, 16 * k + 8 * half, q));
    for (int cb = wave; cb < blocks; cb += kWaves) {
      floatx16p d[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) d[i][r] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uintx4p b[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          typedef __attribute__((address_space(3))) shortx4* lds_shorts;
          const int r = 16 * k + 8 * half + ((lane >> 2) & 3), within = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
          uintx2p part[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = (r + 4 * e) * rowBytes + (((2 * cb + q) ^ (r & 3)) << 6) + (((within >> 4) ^ (((r + 4 * e) >> 2) & 3)) << 4) + (within & 15);
            part[e] = __builtin_bit_cast(uintx2p, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shorts)(X + at)));
          }
          b[q] = (uintx4p){part[0].x, part[0].y, part[1].x, part[1].y};
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) d[i] = multiply_pairs(B[i][k], b, d[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = 32 * i + l32, c = 32 * cb + 4 * half + 8 * q;
          char* const h = X + narrow_at(rowBytes, r, c, 0);
          char* const l = X + narrow_at(rowBytes, r, c, 1);
          float u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = d[i][4 * q + e] * kUnscale;
          if (step < steps - 1) {
            put4(h, l, u);
          } else if (r < m) {
            if (FORM == 0) {
              if (c < n) *(float4*)(y + r * n + c) = make_float4(u[0] * kUnscale, u[1] * kUnscale, u[2] * kUnscale, u[3] * kUnscale);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c + e < n) y[tall ? (c + e) * m + r : r * n + c + e] = u[e] * kUnscale;
            }
          }
        }
    }
    __syncthreads();
  }
}

struct OrthoPlan {
  int m;                          // the shorter side
  int normParts;
  long long pitch, mPitch;
  ProductPlan gram, square, update;   // A = X X', B = a I + b A + c A A, X <- B X
  bool closes;                    // the first two in one launch
  size_t x[2], a, b, parts, sums, counters, total;
};

OrthoPlan ortho_plan(int K, int D, int count) {
  OrthoPlan p;
  p.m = std::min(K, D);
  p.gram = plan_product(kPairs, p.m, p.m, std::max(K, D), count, true);
  p.closes = false;
  if (p.m <= 128 && !tunable("ortho_no_narrow", 0)) {
    // (a tile of all of A against smaller ones and a launch more, which costs some 5 us)
    const ProductPlan whole = plan_product(kPairs, p.m, p.m, std::max(K, D), count, true, p.m <= 64 ? 64 : 128);
    p.closes = p.m <= kTileSize[whole.tile] && whole.tile != kTile256 && whole.cost < p.gram.cost + 5.0;
    if (p.closes) p.gram = whole;
  }
  p.square = plan_product(kPairs, p.m, p.m, p.m, count, true);
  p.update = plan_product(kPairs, K, D, p.m, count);
  p.normParts = (int)std::max<size_t>(1, std::min<size_t>(kNormParts, (size_t)K * D / 2048));
  p.pitch = row_halves(kPairs, D);
  p.mPitch = row_halves(kPairs, p.m);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.x[0] = take((size_t)count * K * p.pitch * 2);
  p.x[1] = take((size_t)count * K * p.pitch * 2);
  p.a = take((size_t)count * p.m * p.mPitch * 2);
  p.b = take((size_t)count * p.m * p.mPitch * 2);
  p.parts = take((size_t)count * kNormParts * sizeof(double));
  p.sums = take(std::max({p.gram.partBytes(), p.square.partBytes(), p.update.partBytes()}));
  p.counters = take(4 * std::max({p.gram.counters(), p.square.counters(), p.update.counters()}));
  p.total = at;
  return p;
}

int ortho_check(const char* who, int K, int D, int count, int steps) {
  if (K < 0 || D < 0 || count < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative tensor extent", who);
  if (steps < 0 || steps > 100) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the number of steps is not between 0 and 100", who);
  if (K > (1 << 20) || D > (1 << 20) || std::min(K, D) > (1 << 15) || count > 65535) return fail(MCN_UNSUPPORTED, "%s: matrix too large", who);
  return MCN_SUCCESS;
}

template <bool ACROSS>
int close_gram(hipStream_t s, const char* who, const Matrix& X, const OrthoPlan& p, const Scratch& scratch, const ClosingEnd& e, int count) {
  if (p.gram.tile == kTile64)
    return run_product<Tile64<kPairs>, ACROSS, ACROSS>(s, who, "ortho_gram", X, X, p.m, p.m, count, true, p.gram, scratch, e);
  if (p.gram.alone()) return run_product<Tile128Alone<kPairs>, ACROSS, ACROSS>(s, who, "ortho_gram", X, X, p.m, p.m, count, true, p.gram, scratch, e);
  return run_product<Tile128<kPairs>, ACROSS, ACROSS>(s, who, "ortho_gram", X, X, p.m, p.m, count, true, p.gram, scratch, e);
}

int orthogonalise(hipStream_t s, const char* who, const OrthoPlan& p, float* y, const float* x, int K, int D, int count, int steps, char* ws) {
  double* parts = (double*)(ws + p.parts);
  {
    KernelTimer timer("ortho_squares", s);
    hipLaunchKernelGGL(ortho_squares, dim3((unsigned)p.normParts, (unsigned)count), dim3(256), 0, s, parts, x, (size_t)K * D,
                       (unsigned*)(ws + p.counters), (int)std::max({p.gram.counters(), p.square.counters(), p.update.counters()}));
  }
  {
    KernelTimer timer("ortho_pack", s);
    hipLaunchKernelGGL(ortho_pack, dim3((unsigned)((K * (p.pitch / 16) + 255) / 256), (unsigned)count), dim3(256), 0, s, (unsigned short*)(ws + p.x[0]), x,
                       parts, p.normParts, K, D, p.pitch);
  }
  int rc = check_launch(who);
  const bool tall = K > D;
  const Scratch scratch = {(float*)(ws + p.sums), (unsigned*)(ws + p.counters)};
  const Matrix A = {ws + p.a, p.mPitch, p.m * p.mPitch, p.m};
  const Matrix B = {ws + p.b, p.mPitch, p.m * p.mPitch, p.m};
  for (int step = 0; step < steps && !rc; ++step) {
    const Matrix X = {ws + p.x[step & 1], p.pitch, K * p.pitch, K};
    if (p.closes) {
      const ClosingEnd closing = {(unsigned short*)(ws + p.b), p.mPitch, p.m * p.mPitch, p.m};
      rc = tall ? close_gram<true>(s, who, X, p, scratch, closing, count) : close_gram<false>(s, who, X, p, scratch, closing, count);
    } else {
      OrthoEnd e = {(unsigned short*)(ws + p.a), nullptr, nullptr, p.mPitch, p.m * p.mPitch, p.m, p.m, 0.f, kUnscale, 0.f, 1};
      rc = tall ? product<kPairs, true, true>(s, who, "ortho_gram", X, X, p.m, p.m, p.gram, scratch, e, count, true)
                : product<kPairs, false, false>(s, who, "ortho_gram", X, X, p.m, p.m, p.gram, scratch, e, count, true);
      if (rc) break;
      e.out = (unsigned short*)(ws + p.b);
      e.c = (const unsigned short*)A.base;
      e.add = kB;
      e.times = kC * kUnscale;
      e.identity = kA * kScale;
      rc = product<kPairs, false, false>(s, who, "ortho_square", A, A, p.m, p.m, p.square, scratch, e, count, true);
    }
    if (rc) break;
    const OrthoEnd e = {(unsigned short*)(ws + p.x[~step & 1]), step == steps - 1 ? y : nullptr, nullptr, p.pitch, K * p.pitch, K, D, 0.f, kUnscale, 0.f, 0};
    rc = tall ? product<kPairs, false, false>(s, who, "ortho_update", X, B, K, D, p.update, scratch, e, count)
              : product<kPairs, false, true>(s, who, "ortho_update", B, X, K, D, p.update, scratch, e, count);
  }
  return rc;
}

// steps == 0: the normalised matrix alone
__global__ __launch_bounds__(256) void ortho_normalise(float* __restrict__ y, const float* __restrict__ x, const double* __restrict__ parts, int used,
                                                       size_t size) {
  const double factor = norm_factor(norm_square(parts, blockIdx.y, used), 1.0);
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (size_t)gridDim.x * 256)
    y[(size_t)blockIdx.y * size + i] = (float)((double)x[(size_t)blockIdx.y * size + i] * factor);
}

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_orthogonalise_workspace_bytes(int K, int D, int count) {
  if (K <= 0 || D <= 0 || count <= 0) return 0;
  return ortho_plan(K, D, count).total;
}

int mcn_orthogonalise(mcn_stream_t stream, float* y, const float* x, int K, int D, int count, int steps, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_orthogonalise";
  int rc = ortho_check(who, K, D, count, steps);
  if (rc || K == 0 || D == 0 || count == 0) return rc;
  if (!y || !x) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null tensor", who);
  const OrthoPlan p = ortho_plan(K, D, count);
  if (!workspace || workspaceBytes < p.total)
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: workspace too small (%zu < %zu bytes)", who, workspaceBytes, p.total);
  if (!aligned16(workspace)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the workspace is not 16-byte aligned", who);
  hipStream_t s = as_stream(stream);
  if (steps == 0) {
    double* parts = (double*)((char*)workspace + p.parts);
    hipLaunchKernelGGL(ortho_squares, dim3((unsigned)p.normParts, (unsigned)count), dim3(256), 0, s, parts, x, (size_t)K * D, (unsigned*)nullptr, 0);
    hipLaunchKernelGGL(ortho_normalise, dim3((unsigned)p.normParts, (unsigned)count), dim3(256), 0, s, y, x, parts, p.normParts, (size_t)K * D);
    return check_launch(who);
  }
  const int m = std::min(K, D), n = std::max(K, D);
  if (m <= kNarrowRows && n <= kNarrowColumns && !tunable("ortho_no_narrow", 0)) {
    const int lds = kNarrowRows * ((n + 63) / 64 * 256) + kSquareBytes;
    static std::atomic<unsigned long long> raised[3];
    const int form = K > D ? 2 : n % 4 == 0 && aligned16(x) && aligned16(y) ? 0 : 1;
    const auto kernel = form == 2 ? ortho_narrow<2> : form == 1 ? ortho_narrow<1> : ortho_narrow<0>;
    rc = allow_lds(who, (const void*)kernel, kNarrowRows * (kNarrowColumns * 4) + kSquareBytes, raised[form]);
    if (rc) return rc;
    KernelTimer timer("ortho_narrow", s);
    hipLaunchKernelGGL(kernel, dim3((unsigned)count), dim3(kNarrowThreads), lds, s, y, x, m, n, steps);
    return check_launch(who);
  }
  return orthogonalise(s, who, p, y, x, K, D, count, steps, (char*)workspace);
}

}  // extern "C"
