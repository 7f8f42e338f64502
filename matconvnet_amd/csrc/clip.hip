// The norm of all gradients of a network and the gradients clipped to it.
//   n = sqrt(sum over all tensors of g^2),  f = most/n where n > most, 1 otherwise,  y = f g
// Bound by memory: g is read once for the norm and once for the product, y written.  Squares are summed in double from the first on
// (gradients of 1e20 or 1e-30 neither overflow nor vanish, and hundreds of millions of terms lose nothing).
//
// A launch takes a table of up to kTable entries in its arguments, so that nothing has to reach the device ahead of it and a captured
// graph holds it all.  Every tensor is cut into runs of one length, a workgroup takes a run and leaves one partial sum; runs are as
// long as makes about kRuns of them in all.  The second launch's workgroups each add up all partial sums, in one order, rather than
// wait for a launch that does only that: 2048 values of 8 bytes out of the L2 for each.
// Measured: ResNet-50's 161 tensors of 25.6 million values, single, 53 us (two launches; most of what is read a second time comes out of the
// caches); 300 tensors of 600 million values in all, bfloat16 and single, 0.99 ms, 4.4 TB/s with g read twice.
#include "mcn_internal.hpp"

#include <algorithm>
#include <cmath>

namespace mcn {
namespace {

typedef unsigned uintx4loose __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes that may start at any value

constexpr int kTable = 164, kFew = 32, kRuns = 2048;
constexpr size_t kLeast = 8192;   // values of a run at least: 256 threads, 32 each
constexpr unsigned kBf16Bit = 1u << 31;
constexpr size_t kPiece = 1ull << 30;   // larger tensors are several entries
constexpr size_t kMost = 1ull << 40;    // values of all tensors: a run is no longer than a piece

// 24 bytes an entry: as many as the 4 KB hold that arguments may take, or few, whose launch has less to copy (10
// tensors of 70000 values: 12.9 us instead of 15.8)
template <int ENTRIES>
struct Table {
  static constexpr int most = ENTRIES;
  const void* der[ENTRIES];
  void* out[ENTRIES];
  unsigned count[ENTRIES];   // with kBf16Bit
  unsigned first[ENTRIES];   // its first workgroup in this launch
  int n;
};
static_assert(sizeof(Table<kTable>) + 48 <= 4096, "arguments");

// (every lane looks at some entries: a search by halves is eight loads one behind the other)
template <class T>
__device__ __forceinline__ int entry_of(const T& t, unsigned block) {
  const int lane = threadIdx.x & 63;
  int k = -1;
#pragma unroll
  for (int i = 0; i < T::most; i += 64) {
    const bool here = i + lane < t.n && t.first[std::min(i + lane, T::most - 1)] <= block;
    k += (int)__popcll(__ballot(here));
  }
  return __builtin_amdgcn_readfirstlane(k);
}

__device__ __forceinline__ double block_sum(double v, double* slots) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  return slots[0] + slots[1] + slots[2] + slots[3];
}

// (functions of a value: __builtin_bit_cast of a vector's element itself gives the vector's first one)
__device__ __forceinline__ float whole(unsigned v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ float low(unsigned v) { return __builtin_bit_cast(float, v << 16); }
__device__ __forceinline__ float high(unsigned v) { return __builtin_bit_cast(float, v & 0xffff0000u); }
__device__ __forceinline__ double square(float v) { return (double)v * (double)v; }

template <bool BF16>
__device__ __forceinline__ double squares(const void* base, size_t first, size_t last) {
  constexpr int V = BF16 ? 8 : 4;
  double s = 0.0;
  size_t i = first + (size_t)threadIdx.x * V;
  const auto load = [&](size_t at) __attribute__((always_inline)) {
    return *(const uintx4loose*)((const char*)base + at * (BF16 ? 2 : 4));
  };
  const auto add = [&](uintx4loose v) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (BF16) s += square(low(v[k])) + square(high(v[k]));
      else s += square(whole(v[k]));
    }
  };
  for (; i + 3 * 256 * V + V <= last; i += 4 * 256 * V) {   // four loads at a time
    const uintx4loose a = load(i), b = load(i + 256 * V), c = load(i + 512 * V), d = load(i + 768 * V);
    add(a);
    add(b);
    add(c);
    add(d);
  }
  for (; i + V <= last; i += 256 * V) add(load(i));
  for (int k = 0; k < V && i + k < last; ++k)
    s += square(BF16 ? low(((const unsigned short*)base)[i + k]) : ((const float*)base)[i + k]);
  return s;
}

template <int ENTRIES>
__global__ __launch_bounds__(256) void clip_squares(double* __restrict__ partials, Table<ENTRIES> t, size_t run) {
  __shared__ double slots[4];
  const int k = entry_of(t, blockIdx.x);
  const size_t count = t.count[k] & ~kBf16Bit, first = (size_t)(blockIdx.x - t.first[k]) * run, last = std::min(first + run, count);
  const double s = block_sum(t.count[k] & kBf16Bit ? squares<true>(t.der[k], first, last) : squares<false>(t.der[k], first, last), slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// the norm (times scale) from the partial sums: the same additions in every workgroup
__device__ __forceinline__ double join_norm(const double* __restrict__ partials, int parts, double scale, double* slots) {
  double s = 0.0;
  int i = threadIdx.x;
  for (; i + 3 * 256 < parts; i += 4 * 256) {
    const double a = partials[i], b = partials[i + 256], c = partials[i + 512], d = partials[i + 768];
    s += (a + b) + (c + d);
  }
  for (; i < parts; i += 256) s += partials[i];
  return sqrt(block_sum(s, slots)) * scale;
}
__device__ __forceinline__ double factor_of(double norm, double most) { return norm > most ? most / norm : 1.0; }

template <bool BF16>
__device__ __forceinline__ void scale_run(void* out, const void* base, size_t first, size_t last, double f) {
  // (the product in double: gradients of 1e25 and a largest norm of 1e-32 make a factor below single precision's smallest)
  const auto scaled = [&](float v) __attribute__((always_inline)) { return (float)((double)v * f); };
  constexpr int V = BF16 ? 8 : 4, SIZE = BF16 ? 2 : 4;
  const auto load = [&](size_t at) __attribute__((always_inline)) { return *(const uintx4loose*)((const char*)base + at * SIZE); };
  const auto store = [&](size_t at, uintx4loose v) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (BF16) {
        const unsigned a = __builtin_bit_cast(unsigned short, (__bf16)scaled(low(v[k]))), b = __builtin_bit_cast(unsigned short, (__bf16)scaled(high(v[k])));
        v[k] = a | b << 16;
      } else {
        v[k] = __builtin_bit_cast(unsigned, scaled(whole(v[k])));
      }
    }
    *(uintx4loose*)((char*)out + at * SIZE) = v;
  };
  size_t i = first + (size_t)threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= last; i += 4 * 256 * V) {
    const uintx4loose a = load(i), b = load(i + 256 * V), c = load(i + 512 * V), d = load(i + 768 * V);
    store(i, a);
    store(i + 256 * V, b);
    store(i + 512 * V, c);
    store(i + 768 * V, d);
  }
  for (; i + V <= last; i += 256 * V) store(i, load(i));
  for (int k = 0; k < V && i + k < last; ++k) {
    if (BF16) ((unsigned short*)out)[i + k] = __builtin_bit_cast(unsigned short, (__bf16)scaled(low(((const unsigned short*)base)[i + k])));
    else ((float*)out)[i + k] = scaled(((const float*)base)[i + k]);
  }
}

// (out may be der: a thread writes what it alone has read)
template <int ENTRIES>
__global__ __launch_bounds__(256) void clip_scale(float* __restrict__ norm, const double* __restrict__ partials, int parts, Table<ENTRIES> t, size_t run,
                                                  double most) {
  __shared__ double slots[4];
  const double n = join_norm(partials, parts, 1.0, slots);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double f = factor_of(n, most);
  const int k = entry_of(t, blockIdx.x);
  if (f == 1.0 && t.out[k] == t.der[k]) return;
  const size_t count = t.count[k] & ~kBf16Bit, first = (size_t)(blockIdx.x - t.first[k]) * run, last = std::min(first + run, count);
  if (t.count[k] & kBf16Bit) scale_run<true>(t.out[k], t.der[k], first, last, f);
  else scale_run<false>(t.out[k], t.der[k], first, last, f);
}

__global__ __launch_bounds__(256) void clip_join(float* __restrict__ norm, double* __restrict__ factor, const double* __restrict__ partials, int parts,
                                                 double scale, double most) {
  __shared__ double slots[4];
  const double n = join_norm(partials, parts, fabs(scale), slots);
  if (threadIdx.x) return;
  if (norm) *norm = (float)n;
  if (factor) *factor = n > most ? scale * factor_of(n, most) : (double)(float)scale;   // (not clipped: the step's own scale)
}

size_t run_of(size_t total) { return std::max(kLeast, (total / kRuns + kLeast - 1) / kLeast * kLeast); }

// the entries of one launch, from `at` on, which is left behind them: tensors and what of them is done; its workgroups
struct Place {
  int tensor = 0;
  size_t done = 0;
};
template <int ENTRIES>
void fill(Table<ENTRIES>* t, Place* at, int n, void* const* out, const void* const* ders, const size_t* counts, const int* types, size_t run, unsigned* blocks) {
  const size_t piece = std::max<size_t>(1, kPiece / run) * run;
  t->n = 0;
  *blocks = 0;
  while (at->tensor < n && t->n < ENTRIES) {
    const int i = at->tensor;
    const size_t size = types[i] == MCN_BFLOAT16 ? 2 : 4, count = std::min(piece, counts[i] - at->done);
    if (count) {
      t->der[t->n] = (const char*)ders[i] + at->done * size;
      t->out[t->n] = out ? (char*)out[i] + at->done * size : nullptr;
      t->count[t->n] = (unsigned)count | (types[i] == MCN_BFLOAT16 ? kBf16Bit : 0);
      t->first[t->n] = *blocks;
      *blocks += (unsigned)((count + run - 1) / run);
      ++t->n;
      at->done += count;
    }
    if (at->done < counts[i]) continue;
    ++at->tensor;
    at->done = 0;
  }
}

struct Sizes {
  size_t total, run, parts;
};
Sizes sizes_of(const size_t* counts, int n) {
  Sizes s = {0, 0, 0};
  for (int i = 0; i < n; ++i) s.total += counts[i];
  s.run = run_of(s.total);
  for (int i = 0; i < n; ++i) s.parts += (counts[i] + s.run - 1) / s.run;
  return s;
}

int check(const char* who, const void* const* ders, const size_t* counts, const int* types, int n) {
  if (n < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative number of tensors", who);
  if (n && (!ders || !counts || !types)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null argument", who);
  size_t total = 0;
  for (int i = 0; i < n; ++i) {
    if (types[i] != MCN_FLOAT && types[i] != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d of tensor %d", who, types[i], i);
    if (counts[i] > kMost - total) return fail(MCN_UNSUPPORTED, "%s: tensor %d too large", who, i);
    total += counts[i];
    if (!counts[i]) continue;
    if (!ders[i]) return fail(MCN_ILLEGAL_ARGUMENT, "%s: tensor %d is null", who, i);
    if ((uintptr_t)ders[i] % (types[i] == MCN_BFLOAT16 ? 2 : 4)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: tensor %d is not aligned", who, i);
  }
  return MCN_SUCCESS;
}

template <int ENTRIES>
int squares_of(const char* who, hipStream_t s, double* partials, const void* const* ders, const size_t* counts, const int* types, int n, size_t run) {
  for (Place at; at.tensor < n;) {
    Table<ENTRIES> t;
    unsigned blocks;
    fill(&t, &at, n, nullptr, ders, counts, types, run, &blocks);
    if (!blocks) continue;
    {
      KernelTimer timer("clip_squares", s);
      hipLaunchKernelGGL(clip_squares<ENTRIES>, dim3(blocks), dim3(256), 0, s, partials, t, run);
    }
    const int rc = check_launch(who);
    if (rc) return rc;
    partials += blocks;
  }
  return MCN_SUCCESS;
}
int squares_of_all(const char* who, hipStream_t s, double* partials, const void* const* ders, const size_t* counts, const int* types, int n, size_t run) {
  return n <= kFew ? squares_of<kFew>(who, s, partials, ders, counts, types, n, run) : squares_of<kTable>(who, s, partials, ders, counts, types, n, run);
}

template <int ENTRIES>
int scale_of(const char* who, hipStream_t s, void* const* outs, float* norm, const double* partials, const void* const* ders, const size_t* counts,
             const int* types, int n, const Sizes& z, double most) {
  int rc = MCN_SUCCESS;
  for (Place at; at.tensor < n && !rc;) {
    Table<ENTRIES> t;
    unsigned blocks;
    fill(&t, &at, n, outs, ders, counts, types, z.run, &blocks);
    if (!blocks) continue;
    KernelTimer timer("clip_scale", s);
    hipLaunchKernelGGL(clip_scale<ENTRIES>, dim3(blocks), dim3(256), 0, s, norm, partials, (int)z.parts, t, z.run, most);
    rc = check_launch(who);
  }
  return rc;
}

}  // namespace

// for the solver's step (eltwise.hip): *factor (device) = derScale * factor of the norm of derScale * der
size_t clip_factor_workspace(size_t count) { return sizes_of(&count, 1).parts * sizeof(double) + 16; }
int clip_factor(const char* who, hipStream_t s, float* norm, double** factor, const float* der, size_t count, double derScale, double most, void* workspace,
                size_t workspaceBytes) {
  const Sizes z = sizes_of(&count, 1);
  int rc = check_workspace(who, workspace, workspaceBytes, clip_factor_workspace(count));
  if (rc) return rc;
  double* partials = (double*)((char*)workspace + 16);
  *factor = (double*)workspace;
  const void* ders[1] = {der};
  const int types[1] = {MCN_FLOAT};
  rc = squares_of_all(who, s, partials, ders, &count, types, 1, z.run);
  if (rc) return rc;
  KernelTimer timer("clip_join", s);
  hipLaunchKernelGGL(clip_join, dim3(1), dim3(256), 0, s, norm, *factor, partials, (int)z.parts, derScale, most);
  return check_launch(who);
}

}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_clip_workspace_bytes(const size_t* counts, int n) {
  if (!counts || n <= 0) return 0;
  return sizes_of(counts, n).parts * sizeof(double);
}

int mcn_gradient_norm(mcn_stream_t stream, float* norm, const void* const* ders, const size_t* counts, const int* dataTypes, int n, void* workspace,
                      size_t workspaceBytes) {
  const char* who = "mcn_gradient_norm";
  int rc = check(who, ders, counts, dataTypes, n);
  if (rc) return rc;
  if (!norm) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null norm", who);
  const Sizes z = sizes_of(counts, n);
  rc = check_workspace(who, workspace, workspaceBytes, z.parts * sizeof(double));
  if (rc) return rc;
  hipStream_t s = as_stream(stream);
  rc = squares_of_all(who, s, (double*)workspace, ders, counts, dataTypes, n, z.run);
  if (rc) return rc;
  KernelTimer timer("clip_join", s);
  hipLaunchKernelGGL(clip_join, dim3(1), dim3(256), 0, s, norm, (double*)nullptr, (const double*)workspace, (int)z.parts, 1.0, 0.0);
  return check_launch(who);
}

int mcn_clip_gradients(mcn_stream_t stream, void* const* outs, float* norm, const void* const* ders, const size_t* counts, const int* dataTypes, int n,
                       double maxNorm, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_clip_gradients";
  int rc = check(who, ders, counts, dataTypes, n);
  if (rc) return rc;
  if (!(maxNorm >= 0)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the largest norm is negative", who);
  if (n && !outs) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null argument", who);
  for (int i = 0; i < n; ++i) {
    if (!counts[i]) continue;
    if (!outs[i]) return fail(MCN_ILLEGAL_ARGUMENT, "%s: output %d is null", who, i);
    const size_t size = dataTypes[i] == MCN_BFLOAT16 ? 2 : 4;
    if ((uintptr_t)outs[i] % size) return fail(MCN_ILLEGAL_ARGUMENT, "%s: output %d is not aligned", who, i);
  }
  const Sizes z = sizes_of(counts, n);
  if (z.parts == 0) {   // nothing but empty tensors
    if (!norm) return MCN_SUCCESS;
    hipLaunchKernelGGL(clip_join, dim3(1), dim3(256), 0, as_stream(stream), norm, (double*)nullptr, (const double*)nullptr, 0, 1.0, 0.0);
    return check_launch(who);
  }
  rc = check_workspace(who, workspace, workspaceBytes, z.parts * sizeof(double));
  if (rc) return rc;
  hipStream_t s = as_stream(stream);
  rc = squares_of_all(who, s, (double*)workspace, ders, counts, dataTypes, n, z.run);
  if (rc) return rc;
  return n <= kFew ? scale_of<kFew>(who, s, outs, norm, (const double*)workspace, ders, counts, dataTypes, n, z, maxNorm)
                   : scale_of<kTable>(who, s, outs, norm, (const double*)workspace, ders, counts, dataTypes, n, z, maxNorm);
}

}  // extern "C"
