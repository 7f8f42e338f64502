// Orthogonalised updates: a matrix G of K filters x D values is replaced by (nearly) the closest one with orthonormal rows or columns, U V'
// of its singular value decomposition U S V', by matrix products alone:
//   X = G/|G|,  five times (or as asked)  X <- a X + (b A + c A^2) X,  A = X X'      (A = X'X and products from the right if K > D)
// Every singular value s goes through p(s) = a s + b s^3 + c s^5; with a = 3.4445, b = -4.7750, c = 2.0315 values from 0.005 on end within
// [0.68, 1.21] after five steps, and none ever passes 1.22.  So X, A and b A + c A^2 stay below 2.9 in magnitude, and the operands of the
// products are pairs of half-precision values (product.hpp) at a scale that is always the same, 2^14 (2.9 * 2^14 < 65504).
// A step is three products: A and A^2 are symmetric, of them only the tiles on and below the diagonal are made and written twice;
// 3 m^2 n + m^3 operations for an m x n matrix, m <= n.  All of a call's matrices (of one size) go through one launch per product.
#include "product.hpp"

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
  // (the products' counters are cleared on the way)
  for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < nCounters; i += gridDim.x * gridDim.y * 256) counters[i] = 0;
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
                                                  int used, int rows, int cols, long long pitch, int wide) {
  const int matrix = blockIdx.y, per = (int)(pitch / 16);
  const double factor = norm_factor(norm_square(parts, matrix, used), (double)kScale);
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)rows * per) return;
  const int row = (int)(i / per), c = (int)(i - (size_t)row * per) * 8;
  const float* from = x + ((size_t)matrix * rows + row) * cols;
  float v[8];
  load8(v, from, c, cols, wide);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (float)((double)v[k] * factor);
  store8_pairs(out + ((size_t)matrix * rows + row) * pitch, c, v);
}

// ---------------------------------------------------------------------------------------------- products

// D = add * C + times * A B, as pairs or as single-precision values
struct OrthoEnd {
  unsigned short* out;      // pairs, at outPitch / outSize
  float* result;            // not null: single precision, rows of `cols` values
  const unsigned short* c;  // pairs of the output's shape; null: nothing is added
  long long pitch, size;
  int rows, cols;
  float add, times;         // (times: with the scales of the two operands)
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

struct OrthoPlan {
  int m;                          // the shorter side
  int normParts;
  long long pitch, mPitch;
  ProductPlan gram, square, update;   // A = X X', B = b A + c A A, X <- a X + B X
  size_t x[2], a, b, parts, sums, counters, total;
};

OrthoPlan ortho_plan(int K, int D, int count) {
  OrthoPlan p;
  p.m = std::min(K, D);
  p.gram = plan_product(kPairs, p.m, p.m, std::max(K, D), count, true);
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
                       parts, p.normParts, K, D, p.pitch, (int)(D % 4 == 0 && aligned16(x)));
  }
  int rc = check_launch(who);
  const bool tall = K > D;
  const Scratch scratch = {(float*)(ws + p.sums), (unsigned*)(ws + p.counters)};
  const Matrix A = {ws + p.a, p.mPitch, p.m * p.mPitch, p.m};
  const Matrix B = {ws + p.b, p.mPitch, p.m * p.mPitch, p.m};
  for (int step = 0; step < steps && !rc; ++step) {
    const Matrix X = {ws + p.x[step & 1], p.pitch, K * p.pitch, K};
    OrthoEnd e = {(unsigned short*)(ws + p.a), nullptr, nullptr, p.mPitch, p.m * p.mPitch, p.m, p.m, 0.f, kUnscale, 1};
    rc = tall ? product<kPairs, true, true>(s, who, "ortho_gram", X, X, p.m, p.m, p.gram, scratch, e, count, true)
              : product<kPairs, false, false>(s, who, "ortho_gram", X, X, p.m, p.m, p.gram, scratch, e, count, true);
    if (rc) break;
    e.out = (unsigned short*)(ws + p.b);
    e.c = (const unsigned short*)A.base;
    e.add = kB;
    e.times = kC * kUnscale;
    rc = product<kPairs, false, false>(s, who, "ortho_square", A, A, p.m, p.m, p.square, scratch, e, count, true);
    if (rc) break;
    e = {(unsigned short*)(ws + p.x[~step & 1]), step == steps - 1 ? y : nullptr, (const unsigned short*)X.base, p.pitch, K * p.pitch, K, D, kA, kUnscale, 0};
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
  hipStream_t s = as_stream(stream);
  if (steps == 0) {
    double* parts = (double*)((char*)workspace + p.parts);
    hipLaunchKernelGGL(ortho_squares, dim3((unsigned)p.normParts, (unsigned)count), dim3(256), 0, s, parts, x, (size_t)K * D, (unsigned*)nullptr, 0);
    hipLaunchKernelGGL(ortho_normalise, dim3((unsigned)p.normParts, (unsigned)count), dim3(256), 0, s, y, x, parts, p.normParts, (size_t)K * D);
    return check_launch(who);
  }
  return orthogonalise(s, who, p, y, x, K, D, count, steps, (char*)workspace);
}

}  // extern "C"
