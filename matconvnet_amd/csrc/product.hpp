// Matrix products on 16-bit operands, D[m][n] = sum_k A(m, k) B(n, k), for the operators whose work is one
// (fcloss.hip, ortho.hip).
//
// Operands.  Rows of 16-bit values in global memory, 16-byte aligned.  An operand is read ALONG its rows (the reduction
// index is the one that runs along a row: the row index is m or n) or ACROSS them (the reduction index counts the rows).
//   kBf16   bfloat16 as it stands.
//   kPairs  a single-precision value v as two half-precision ones, h = half(s v) and l = half(s v - h), s a power of two that puts the
//           largest magnitude of the tensor (or row) into [2^14, 2^15).  h + l keeps 22 bits and the sign of l one more: v to 2^-24
//           of itself down to 2^-29 of the largest magnitude, to 2^-40 of that magnitude below (l is subnormal there; the matrix
//           instruction takes subnormals).  A product of two such values is the sum of three, hh + hl + lh; the dropped ll is
//           at most 2^-24 and 1e-8 on average of it, a sixth of single precision's own rounding.  Three half-precision
//           matrix instructions do what the six of a split into three bfloat16 do, which needs no scale.
//           Of each 32 values of a row first the 32 h, then the 32 l: one row of a stage is 128 bytes in either type.
//
// One workgroup makes a BM x BN tile of D, a wavefront 32 TM x 32 TN of it by v_mfma_f32_32x32x16 with the operands exchanged, so that
// a lane holds one row m and four neighbouring columns n per four registers: a row's sums need one exchange between two lanes, and
// stores along rows are 8 or 16 bytes.  A stage is 64 (kBf16) or 32 (kPairs) reduction indices, 128 bytes per row of tile, brought
// straight into LDS while the previous one is multiplied.
#pragma once

#include "mcn_internal.hpp"

#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

namespace mcn {

enum { kBf16 = 0, kPairs = 1 };

typedef float floatx16p __attribute__((ext_vector_type(16)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4p __attribute__((ext_vector_type(4)));
typedef unsigned uintx2p __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned short to_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
__device__ __forceinline__ float from_bf16(unsigned short v) { return __builtin_bit_cast(float, (unsigned)v << 16); }

// reduction indices per stage, and 16-bit values a row of `n` takes
constexpr int stage_depth(int type) { return type == kPairs ? 32 : 64; }
constexpr long long row_halves(int type, long long n) { return type == kPairs ? (n + 31) / 32 * 64 : (n + 63) / 64 * 64; }

struct Operand {
  const void* base;
  long long pitch;   // 16-bit values from row to row (a multiple of 64)
  long long rows;    // rows that exist: what is behind them reads as zero
};

template <int TYPE, int BM_, int BN_, int WM_, int WN_>
struct ProductShape {
  static constexpr int type = TYPE;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;      // tile, wavefronts along m and n
  static constexpr int threads = 64 * WM * WN;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;         // blocks of 32 x 32 per wavefront
  static constexpr int stageBytes = (BM + BN) * 128;
  static constexpr int ldsBytes = 2 * stageBytes;
};

typedef __attribute__((address_space(3))) char* lds_bytes;

// Where 16 bytes of a stage lie.  ALONG: row r's eight chunks are exchanged by r & 7, so that eight lanes that read the same chunk
// of eight rows meet all banks.  ACROSS: a row of the stage is one reduction index, R values; 64-byte granules (32 values of m, h
// or l) are exchanged so that the four indices a transposing read takes lie in different banks.
template <int TYPE, bool ACROSS, int R>
struct Stage {
  static constexpr int granules = TYPE == kPairs ? R / 16 : R / 32;    // per row of the stage, ACROSS
  static constexpr int rowBytes = ACROSS ? granules * 64 : 128;
  static constexpr int chunks = R * 128 / 16;                          // 16-byte chunks of the whole stage
  __device__ static __forceinline__ int turn(int k) { return granules >= 4 ? (k & 3) : ((k >> 1) & (granules - 1)); }
  // chunk t of LDS: which row of the stage and which 16 bytes of that row it holds
  __device__ static __forceinline__ void source(int t, int* row, int* chunk) {
    if (ACROSS) {
      *row = t / (granules * 4);
      const int c = t % (granules * 4);
      *chunk = c ^ (turn(*row) << 2);
    } else {
      *row = t >> 3;
      *chunk = (t & 7) ^ (*row & 7);
    }
  }
  // eight reduction indices from 16 s + 8 (lane / 32) of row 32 b + lane % 32, part (0: h, 1: l)
  __device__ static __forceinline__ uintx4p fragment(const char* lds, int lane, int b, int s, int part) {
    if (!ACROSS) {
      const int chunk = (TYPE == kPairs ? 4 * part : 0) + 2 * s + (lane >> 5);
      return *(const uintx4p*)(lds + (lane & 31) * 128 + ((chunk ^ (lane & 7)) << 4) + b * 4096);
    } else {
      // a group of 16 lanes gives four indices x 16 values of m and takes, lane by lane, one m and four indices
      const int k = 16 * s + 8 * (lane >> 5) + ((lane >> 2) & 3);
      const int granule = TYPE == kPairs ? 2 * b + part : b;
      const int within = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
      typedef __attribute__((address_space(3))) shortx4* lds_shorts;
      const uintx2p a = __builtin_bit_cast(uintx2p, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_shorts)(lds + k * rowBytes + ((granule ^ turn(k)) << 6) + within)));
      const uintx2p c = __builtin_bit_cast(uintx2p, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_shorts)(lds + (k + 4) * rowBytes + ((granule ^ turn(k + 4)) << 6) + within)));
      return (uintx4p){a.x, a.y, c.x, c.y};
    }
  }
};

template <int TYPE>
__device__ __forceinline__ floatx16p multiply(uintx4p a, uintx4p b, floatx16p c) {
  if (TYPE == kPairs)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfx8, a), __builtin_bit_cast(bfx8, b), c, 0, 0, 0);
}

// One operand's loads.  A workgroup's wavefront w brings chunks [64 (w + i W), + 64) of a stage for every i.
template <class S, bool ACROSS, int R>
struct Loader {
  typedef Stage<S::type, ACROSS, R> St;
  static constexpr int loads = St::chunks / S::threads;
  static_assert(St::chunks % S::threads == 0, "whole loads");
  unsigned offset[loads];
  const char* base;
  unsigned long long left;   // bytes from base to the end of the operand
  unsigned long long step;

  // first: first row (ALONG) or first value of m (ACROSS) of the tile; stage0: first stage
  __device__ __forceinline__ void begin(const Operand& o, long long first, long long stage0, int tid) {
#pragma unroll
    for (int i = 0; i < loads; ++i) {
      int row, chunk;
      St::source(i * S::threads + tid, &row, &chunk);
      offset[i] = (unsigned)(row * o.pitch * 2 + chunk * 16);
    }
    const unsigned long long all = (unsigned long long)o.rows * o.pitch * 2;
    const unsigned long long at = ACROSS ? (unsigned long long)stage0 * stage_depth(S::type) * o.pitch * 2 + (S::type == kPairs ? 4 : 2) * first
                                         : (unsigned long long)first * o.pitch * 2 + stage0 * 128;
    base = (const char*)o.base + at;
    left = at < all ? all - at : 0;
    step = ACROSS ? (unsigned long long)stage_depth(S::type) * o.pitch * 2 : 128;
  }
  __device__ __forceinline__ void load(char* lds, int wave) {
    typedef __attribute__((address_space(3))) void* lds_ptr;
    const unsigned records = left > 0xfffffff0ull ? 0xfffffff0u : (unsigned)left;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)records, 0x00020000);
#pragma unroll
    for (int i = 0; i < loads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (i * S::threads + wave * 64) * 16), 16, (int)offset[i], 0, 0, 0);
    base += step;
    left = left > step ? left - step : 0;
  }
};

// (a function of its own with `restrict` pointers: that the loads fill another buffer than the one read is what lets the reads go
// without waiting for them)
template <class S, bool A_ACROSS, bool B_ACROSS, class LA, class LB>
__device__ __forceinline__ void product_stage(const char* __restrict__ from, char* __restrict__ to, bool more, LA& la, LB& lb, int wave, int lane,
                                              int wm, int wn, floatx16p (&acc)[S::TM][S::TN]) {
  if (more) {
    la.load(to, wave);
    lb.load(to + S::BM * 128, wave);
  }
  typedef Stage<S::type, A_ACROSS, S::BM> SA;
  typedef Stage<S::type, B_ACROSS, S::BN> SB;
  constexpr int parts = S::type == kPairs ? 2 : 1;
#pragma unroll
  for (int s = 0; s < stage_depth(S::type) / 16; ++s) {
    uintx4p a[parts][S::TM], b[parts][S::TN];
#pragma unroll
    for (int q = 0; q < parts; ++q) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i) a[q][i] = SA::fragment(from, lane, wm * S::TM + i, s, q);
#pragma unroll
      for (int j = 0; j < S::TN; ++j) b[q][j] = SB::fragment(from + S::BM * 128, lane, wn * S::TN + j, s, q);
    }
#pragma unroll
    for (int t = parts == 2 ? 0 : 2; t < 3; ++t)   // lh, hl, hh: the small ones first
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
          acc[i][j] = multiply<S::type>(b[parts == 2 && t == 1 ? 1 : 0][j], a[parts == 2 && t == 0 ? 1 : 0][i], acc[i][j]);
  }
}

// acc[i][j][r]: row m0 + 32 (wm TM + i) + lane % 32, column n0 + 32 (wn TN + j) + 8 (r / 4) + 4 (lane / 32) + r % 4.
// lds: S::ldsBytes, free again behind the last barrier.
template <class S, bool A_ACROSS, bool B_ACROSS>
__device__ __forceinline__ void product_tile(const Operand& A, const Operand& B, long long m0, long long n0, long long stage0, int stages, char* lds,
                                             floatx16p (&acc)[S::TM][S::TN]) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave % S::WM, wn = wave / S::WM;
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  Loader<S, A_ACROSS, S::BM> la;
  Loader<S, B_ACROSS, S::BN> lb;
  la.begin(A, m0, stage0, tid);
  lb.begin(B, n0, stage0, tid);
  if (stages > 0) {
    la.load(lds, wave);
    lb.load(lds + S::BM * 128, wave);
  }
  int at = 0;
  for (int s = 1; s <= stages; ++s) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    product_stage<S, A_ACROSS, B_ACROSS>(lds + at, lds + (S::stageBytes - at), s < stages, la, lb, wave, lane, wm, wn, acc);
    at = S::stageBytes - at;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The tiles of a grid of workgroups: consecutive workgroups of one XCD take kTileRows rows of tiles by as many columns as fit, so that
// the tiles in flight on an XCD share operands in its L2.
struct TileGrid {
  int tilesM, tilesN;
  int slices;          // independent products, or cuts of the reduction, one behind the other
};
constexpr int kTileRows = 4;
__device__ __forceinline__ void tile_of(const TileGrid& g, int* tm, int* tn, int* slice) {
  const int per = g.tilesM * g.tilesN;
  const int id = xcd_contiguous_id((int)blockIdx.x, (int)gridDim.x);
  *slice = id / per;
  const int t = id - *slice * per;
  const int band = kTileRows * g.tilesN;
  const int first = t / band * kTileRows, rows = min(kTileRows, g.tilesM - first);
  const int within = t - t / band * band;
  *tm = first + within % rows;
  *tn = within / rows;
}

// The power of two s that puts a magnitude (its bits) into [2^14, 2^15), and 1 / s.  1 for zero and what is not finite.
__device__ __forceinline__ float pair_scale(unsigned bits) {
  const int e = (int)(bits >> 23 & 255);
  if (bits == 0 || e == 255) return 1.f;
  return __builtin_bit_cast(float, (unsigned)(127 + min(126, 14 - (e - 127))) << 23);
}
__device__ __forceinline__ float pair_unscale(unsigned bits) {
  const int e = (int)(bits >> 23 & 255);
  if (bits == 0 || e == 255) return 1.f;
  return __builtin_bit_cast(float, (unsigned)(127 - min(126, 14 - (e - 127))) << 23);
}
// v (already scaled) as its two halves, in the bits of an unsigned: h below, l above
__device__ __forceinline__ unsigned split_pair(float v) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(v - (float)h);
  return (unsigned)__builtin_bit_cast(unsigned short, h) | (unsigned)__builtin_bit_cast(unsigned short, l) << 16;
}
__device__ __forceinline__ float half_bits(unsigned short b) { return (float)__builtin_bit_cast(_Float16, b); }

// eight neighbours (from a multiple of eight on) of a row of D values; zeros behind its end
template <class V>
__device__ __forceinline__ void load8(float (&v)[8], const V* __restrict__ row, int c, int D, bool wide) {
  if (wide && c + 8 <= D) {
    if (sizeof(V) == 4) {
      const float4 a = ((const float4*)(row + c))[0], b = ((const float4*)(row + c))[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uintx4p a = *(const uintx4p*)(row + c);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = from_bf16((unsigned short)a[k]);
        v[2 * k + 1] = from_bf16((unsigned short)(a[k] >> 16));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < D ? (sizeof(V) == 4 ? ((const float*)row)[c + k] : from_bf16(((const unsigned short*)row)[c + k])) : 0.f;
  }
}
__device__ __forceinline__ void store8_pairs(unsigned short* row, int c, const float (&v)[8]) {
  uintx4p h, l;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned a = split_pair(v[2 * k]), b = split_pair(v[2 * k + 1]);
    h[k] = (a & 0xffffu) | b << 16;
    l[k] = a >> 16 | (b & 0xffff0000u);
  }
  uintx4p* at = (uintx4p*)(row + (c / 32) * 64 + c % 32);
  at[0] = h;
  at[4] = l;
}

// What to do with a finished tile is E's: e.finish<S>(acc, tile row, tile column, slice, lane, wavefront along m, along n, LDS).
template <class S, bool A_ACROSS, bool B_ACROSS, class E>
__global__ __launch_bounds__(S::threads, 2) void product_kernel(Operand A, Operand B, TileGrid g, int stages, int perSlice, E e) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  int tm, tn, slice;
  tile_of(g, &tm, &tn, &slice);
  const int s0 = slice * perSlice;
  floatx16p acc[S::TM][S::TN];
  product_tile<S, A_ACROSS, B_ACROSS>(A, B, (long long)tm * S::BM, (long long)tn * S::BN, s0, max(0, min(perSlice, stages - s0)), lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  e.template finish<S>(acc, tm, tn, slice, lane, wave % S::WM, wave / S::WM, lds);
}

// ---------------------------------------------------------------------------------------------- host

// Which tile: the largest that still gives every compute unit one
enum { kTile256, kTile128, kTile64 };
inline int choose_tile(long long M, long long N, int count = 1, bool symmetric = false) {
  const int cus = std::max(1, device_compute_units());
  const auto tiles = [&](int t) {
    const long long rows = (M + t - 1) / t;
    return count * (symmetric ? rows * (rows + 1) / 2 : rows * ((N + t - 1) / t));
  };
  if (tiles(256) >= cus) return kTile256;
  if (tiles(128) >= cus) return kTile128;
  return kTile64;
}

// A kernel with more than 64 KiB of local memory has to be told so once per device.
template <class S>
int allow_lds(const char* who, const void* kernel) {
  if (S::ldsBytes <= 65536) return MCN_SUCCESS;
  static std::mutex mutex;
  static std::set<std::pair<const void*, int>> raised;
  const int dev = current_device();
  if (dev < 0) return fail(MCN_DEVICE_ERROR, "%s: no device", who);
  std::lock_guard<std::mutex> lock(mutex);
  if (raised.count({kernel, dev})) return MCN_SUCCESS;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, S::ldsBytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(MCN_DEVICE_ERROR, "%s: local memory", who);
  }
  raised.insert({kernel, dev});
  return MCN_SUCCESS;
}

template <class S, bool A_ACROSS, bool B_ACROSS, class E>
int run_product(hipStream_t s, const char* who, const char* name, const Operand& A, const Operand& B, long long M, long long N, int stages, int slices, const E& e) {
  TileGrid g = {div_up(M, S::BM), div_up(N, S::BN), slices};
  const long long blocks = (long long)g.tilesM * g.tilesN * slices;
  if (blocks >= (1ll << 31)) return fail(MCN_UNSUPPORTED, "%s: tensor too large", who);
  const auto kernel = product_kernel<S, A_ACROSS, B_ACROSS, E>;
  int rc = allow_lds<S>(who, (const void*)kernel);
  if (rc) return rc;
  KernelTimer timer(name, s);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(S::threads), S::ldsBytes, s, A, B, g, stages, div_up(stages, slices), e);
  return check_launch(who);
}

template <int TYPE, bool A_ACROSS, bool B_ACROSS, class E>
int product(hipStream_t s, const char* who, const char* name, const Operand& A, const Operand& B, long long M, long long N, long long depth, int slices, const E& e, int tile) {
  const int stages = (int)((depth + stage_depth(TYPE) - 1) / stage_depth(TYPE));
  switch (tile) {
    case kTile256: return run_product<ProductShape<TYPE, 256, 256, 2, 4>, A_ACROSS, B_ACROSS>(s, who, name, A, B, M, N, stages, slices, e);
    case kTile128: return run_product<ProductShape<TYPE, 128, 128, 2, 2>, A_ACROSS, B_ACROSS>(s, who, name, A, B, M, N, stages, slices, e);
    default: return run_product<ProductShape<TYPE, 64, 64, 2, 2>, A_ACROSS, B_ACROSS>(s, who, name, A, B, M, N, stages, slices, e);
  }
}
constexpr int kTileSize[3] = {256, 128, 64};

}  // namespace mcn
