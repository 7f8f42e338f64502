// Matrix products on 16-bit operands, D[m][n] = sum_k A(m, k) B(n, k), for the operators whose work is one
// (fcloss.hip, ortho.hip).
//
// Operands.  Rows of 16-bit values in global memory, 16-byte aligned.  An operand is read ALONG its rows (the reduction
// index is the one that runs along a row: the row index is m or n) or ACROSS them (the reduction index counts the rows).
//   kBf16   bfloat16 as it stands.
//   kPairs  a single-precision value v as two half-precision ones, h = half(s v) and l = half(s v - h), s a power of two that puts the
//           largest magnitude of what shares it into [2^14, 2^15).  h + l is v to 2^-23 of itself down to 2^-16 of that magnitude, and to
//           2^-39 of that magnitude below (l is subnormal there; the matrix instruction takes subnormals): a bit is lost per power of
//           two.  A product of two such values is the sum of three, hh + hl + lh; the dropped ll is at most 2^-22 of it.
//           All told a product is off by 2^-21 of itself at most and 7e-8 in the mean square (a single-precision multiplication: 2^-24 and
//           2.5e-8); sums are in single precision.  Three half-precision matrix instructions do what the six of a split into three
//           bfloat16 do, which needs no scale.
//           Of each 32 values of a row first the 32 h, then the 32 l: one row of a stage is 128 bytes in either type.
//
// One workgroup makes a BM x BN tile of D, a wavefront 32 TM x 32 TN of it by v_mfma_f32_32x32x16 with the operands exchanged, so that
// a lane holds one row m and four neighbouring columns n per four registers: a row's sums need one exchange between two lanes, and
// stores along rows are 8 or 16 bytes.  A stage is 64 (kBf16) or 32 (kPairs) reduction indices, 128 bytes per row of tile, brought
// straight into LDS while the previous one is multiplied.
#pragma once

#include "mcn_internal.hpp"

#include <algorithm>
#include <atomic>

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

template <int TYPE, int BM_, int BN_, int WM_, int WN_, int BUFFERS>
struct ProductShape {
  static constexpr int type = TYPE;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;      // tile, wavefronts along m and n
  static constexpr int threads = 64 * WM * WN;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;         // blocks of 32 x 32 per wavefront
  static constexpr int stageBytes = (BM + BN) * 128;
  static constexpr int buffers = BUFFERS;                            // stages in LDS at a time
  static constexpr int ldsBytes = BUFFERS * stageBytes;
};

typedef __attribute__((address_space(3))) char* lds_bytes;

// Where 16 bytes of a stage lie.  ALONG: row r's eight chunks are exchanged by r / 2 % 8, so that sixteen lanes that read the same chunk
// of sixteen rows meet all 64 banks (by r % 8 rows r and r + 8 met: half of the cycles of these reads were conflicts).  ACROSS: a row of the stage is one reduction index, R values; 64-byte granules (32 values of m, h
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
      *chunk = (t & 7) ^ (*row >> 1 & 7);
    }
  }
  // eight reduction indices from 16 s + 8 (lane / 32) of row 32 b + lane % 32, part (0: h, 1: l)
  __device__ static __forceinline__ uintx4p fragment(const char* lds, int lane, int b, int s, int part) {
    if (!ACROSS) {
      const int chunk = (TYPE == kPairs ? 4 * part : 0) + 2 * s + (lane >> 5);
      return *(const uintx4p*)(lds + (lane & 31) * 128 + ((chunk ^ (lane >> 1 & 7)) << 4) + b * 4096);
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

// One operand's loads.  A workgroup's wavefront w brings chunks [64 (w + i W), + 64) of a stage for every i.  REPEAT: how many stages of the
// product each stage of the operand serves, one behind the other (against another operand whose values stand in two parts, a stage of the first
// part and one of the second in turn).
template <class S, bool ACROSS, int R, int REPEAT>
struct Loader {
  typedef Stage<S::type, ACROSS, R> St;
  static constexpr int loads = St::chunks / S::threads;
  static_assert(St::chunks % S::threads == 0, "whole loads");
  unsigned offset[loads];
  const char* base;
  unsigned long long left;   // bytes from base to the end of the operand
  unsigned long long step;
  int turn;                  // how often the stage that is due has been brought
  int more;                  // stages to come: the loads behind the last one go out all the same (their number is what is waited for) and
                             // find nothing

  // first: first row (ALONG) or first value of m (ACROSS) of the tile; productStage: the product's first stage
  __device__ __forceinline__ void begin(const Operand& o, long long first, long long productStage, int stages, int tid) {
    const long long stage0 = productStage / REPEAT;
    turn = (int)(productStage % REPEAT);
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
    more = stages;
    step = ACROSS ? (unsigned long long)stage_depth(S::type) * o.pitch * 2 : 128;
  }
  // load i of a stage; after the last one the next stage's are due
  __device__ __forceinline__ void load(char* lds, int wave, int i) {
    typedef __attribute__((address_space(3))) void* lds_ptr;
    const unsigned records = more <= 0 ? 0u : left > 0xfffffff0ull ? 0xfffffff0u : (unsigned)left;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)records, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (i * S::threads + wave * 64) * 16), 16, (int)offset[i], 0, 0, 0);
    if (i == loads - 1) {
      --more;
      if (REPEAT > 1 && ++turn < REPEAT) return;
      turn = 0;
      base += step;
      left = left > step ? left - step : 0;
    }
  }
  __device__ __forceinline__ void load_all(char* lds, int wave) {
#pragma unroll
    for (int i = 0; i < loads; ++i) load(lds, wave, i);
  }
};

// The fragments of one step of 16 reduction indices
template <class S>
struct Fragments {
  static constexpr int parts = S::type == kPairs ? 2 : 1;
  uintx4p a[parts][S::TM], b[parts][S::TN];
  template <bool A_ACROSS, bool B_ACROSS>
  __device__ __forceinline__ void read(const char* lds, int lane, int wm, int wn, int s) {
#pragma unroll
    for (int q = 0; q < parts; ++q) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i) a[q][i] = Stage<S::type, A_ACROSS, S::BM>::fragment(lds, lane, wm * S::TM + i, s, q);
#pragma unroll
      for (int j = 0; j < S::TN; ++j) b[q][j] = Stage<S::type, B_ACROSS, S::BN>::fragment(lds + S::BM * 128, lane, wn * S::TN + j, s, q);
    }
  }
  // the matrix instructions of a step, with load(0), load(1) ... load(LOADS - 1) spread among them
  template <int LOADS, class Load>
  __device__ __forceinline__ void multiply_into(floatx16p (&acc)[S::TM][S::TN], Load load) const {
    constexpr int products = parts == 2 ? 3 : 1, all = products * S::TM * S::TN, every = all / (LOADS + 1) > 0 ? all / (LOADS + 1) : 1;
    int done = 0, loaded = 0;
#pragma unroll
    for (int t = 0; t < products; ++t)   // lh, hl, hh: the small ones first
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) {
          acc[i][j] = multiply<S::type>(b[parts == 2 && t == 1 ? 1 : 0][j], a[parts == 2 && t == 0 ? 1 : 0][i], acc[i][j]);
          if (++done % every == 0 && loaded < LOADS) {
            __builtin_amdgcn_sched_barrier(0);
            load(loaded++);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
    for (; loaded < LOADS; ++loaded) load(loaded);
  }
};

// One stage: `f` holds the fragments of its first step and is left with those of the next stage's.  The reads of a step go out before the
// matrix instructions of the step before it; the barrier, which every wavefront reaches with its last reads of this stage done,
// stands before the last step's, behind it the stage's buffer (`to`) is filled again: with A's share among the matrix
// instructions of the last step, B's among those of the next stage's first.  (All of a stage's loads in a row behind the
// barrier held the wavefronts up for as long as the CU's 64 bytes a clock take: 8192 x 8192 x 4096 bfloat16 475 -> 446 us.)
// (A function of its own with `restrict` pointers: that the loads fill none of what is read is what lets the reads go without waiting
// for them.  `to` is `from`, filled behind the barrier that ends its reads; `filled` holds what the barrier then waits for.)
template <class S, bool A_ACROSS, bool B_ACROSS, class LA, class LB>
__device__ __forceinline__ void product_stage(const char* __restrict__ from, const char* __restrict__ next, char* __restrict__ to, char* __restrict__ filled,
                                              LA& la, LB& lb, int wave, int lane, int wm, int wn, Fragments<S>& f, floatx16p (&acc)[S::TM][S::TN]) {
  constexpr int steps = stage_depth(S::type) / 16;
#pragma unroll
  for (int s = 1; s < steps; ++s) {
    Fragments<S> g;
    g.template read<A_ACROSS, B_ACROSS>(from, lane, wm, wn, s);
    __builtin_amdgcn_sched_barrier(0);   // (the compiler would move the reads down to their first use)
    if (s == 1) f.template multiply_into<LB::loads>(acc, [&](int i) __attribute__((always_inline)) { lb.load(filled + S::BM * 128, wave, i); });
    else f.template multiply_into<0>(acc, [](int) {});
    __builtin_amdgcn_sched_barrier(0);
    f = g;
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S::buffers - 2) * (LA::loads + LB::loads)) : "memory");
  Fragments<S> g;
  g.template read<A_ACROSS, B_ACROSS>(next, lane, wm, wn, 0);
  __builtin_amdgcn_sched_barrier(0);
  f.template multiply_into<LA::loads>(acc, [&](int i) __attribute__((always_inline)) { la.load(to, wave, i); });
  __builtin_amdgcn_sched_barrier(0);
  f = g;
}

// acc[i][j][r]: row m0 + 32 (wm TM + i) + lane % 32, column n0 + 32 (wn TN + j) + 8 (r / 4) + 4 (lane / 32) + r % 4.
// lds: S::ldsBytes, free again behind the last barrier.
template <class S, bool A_ACROSS, bool B_ACROSS, int A_REPEAT>
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
  Loader<S, A_ACROSS, S::BM, A_REPEAT> la;
  Loader<S, B_ACROSS, S::BN, 1> lb;
  la.begin(A, m0, stage0, stages, tid);
  lb.begin(B, n0, stage0, stages, tid);
#pragma unroll
  for (int k = 0; k < S::buffers; ++k) {
    la.load_all(lds + k * S::stageBytes, wave);
    if (k < S::buffers - 1) lb.load_all(lds + k * S::stageBytes + S::BM * 128, wave);
  }
  Fragments<S> f;
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S::buffers - 2) * (la.loads + lb.loads) + la.loads) : "memory");
  f.template read<A_ACROSS, B_ACROSS>(lds, lane, wm, wn, 0);
  int at = 0, filled = S::ldsBytes - S::stageBytes;
  for (int s = 0; s < stages; ++s) {
    const int next = at + S::stageBytes == S::ldsBytes ? 0 : at + S::stageBytes;
    product_stage<S, A_ACROSS, B_ACROSS>(lds + at, lds + next, lds + at, lds + filled, la, lb, wave, lane, wm, wn, f, acc);
    filled = at;
    at = next;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The exponent of a magnitude (its bits): 2^e <= magnitude < 2^(e + 1), subnormal ones included; -1 for zero and what is not finite.  A
// value as pairs is brought up by kPairExponent - e.
constexpr int kPairExponent = 14;
__device__ __forceinline__ int exponent_of(unsigned bits) { return __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, bits)) - 1; }
// v (already scaled) as its two halves, in the bits of an unsigned: h below, l above
__device__ __forceinline__ unsigned split_pair(float v) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(v - (float)h);
  return (unsigned)__builtin_bit_cast(unsigned short, h) | (unsigned)__builtin_bit_cast(unsigned short, l) << 16;
}
__device__ __forceinline__ float half_bits(unsigned short b) { return (float)__builtin_bit_cast(_Float16, b); }

// eight neighbours (from a multiple of eight on) of a row of D values; zeros behind its end.  Rows may start anywhere: 16-byte loads ask for
// no alignment here (rows of odd lengths by single values: 21841 x 1001 bfloat16 values packed in 37 us, 22 so)
typedef unsigned uintx4loose __attribute__((ext_vector_type(4), aligned(2)));
typedef float floatx4loose __attribute__((ext_vector_type(4), aligned(4)));
template <class V>
__device__ __forceinline__ void load8(float (&v)[8], const V* __restrict__ row, int c, int D) {
  if (c + 8 <= D) {
    if (sizeof(V) == 4) {
      const floatx4loose a = *(const floatx4loose*)(row + c), b = *(const floatx4loose*)(row + c + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = a[k];
        v[4 + k] = b[k];
      }
    } else {
      const uintx4loose a = *(const uintx4loose*)(row + c);
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

// A reduction cut into slices (of the tiles from `full` on): every workgroup of a tile leaves its part in memory, the one that comes last adds them up in the order of the
// slices (its own among them: the same bits whichever is last) and goes on to finish the tile.  `counters`: one per tile, zero
// before and after.  The XCDs' L2s are not coherent: the parts are written and read by relaxed atomic accesses at the scope of the
// device, which go past them, and are counted once they have arrived.  (Plain accesses, and a count that releases and acquires, write
// back and empty an L2 per workgroup: a quarter of a microsecond each, one at a time on an XCD.)
struct Slices {
  float* parts;
  unsigned* counters;
  int slices, perSlice;   // (slices == 1: neither pointer is used)
  int full;               // tiles before the first that is cut
};
template <class S>
__device__ __forceinline__ bool join_slices(const Slices& j, int tile, int slice, floatx16p (&acc)[S::TM][S::TN], char* lds) {
  if (j.slices == 1) return true;
  constexpr size_t size = (size_t)S::BM * S::BN / 2;   // in pairs of values
  typedef unsigned long long two;
  two* mine = (two*)j.parts + ((size_t)tile * j.slices + slice) * size + threadIdx.x;
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int k = 0; k < S::TN; ++k)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float2 v = make_float2(acc[i][k][2 * q], acc[i][k][2 * q + 1]);
        __hip_atomic_store(mine + ((i * S::TN + k) * 8 + q) * S::threads, __builtin_bit_cast(two, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the parts have arrived where every XCD reads them,
  __syncthreads();                                     // those of all wavefronts,
  if (threadIdx.x == 0) {                              // before they are counted
    const unsigned before = __hip_atomic_fetch_add(j.counters + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = before == (unsigned)j.slices - 1u;
    if (last) __hip_atomic_store(j.counters + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *(unsigned*)lds = last;
  }
  __syncthreads();
  const bool last = *(volatile unsigned*)lds != 0;
  __syncthreads();   // (the LDS is the finishing code's again)
  if (!last) return false;
  two* from = (two*)j.parts + (size_t)tile * j.slices * size + threadIdx.x;
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int k = 0; k < S::TN; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][k][r] = 0.f;
  for (int s = 0; s < j.slices; ++s)
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int k = 0; k < S::TN; ++k) {
        two v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          v[q] = __hip_atomic_load(from + s * size + ((i * S::TN + k) * 8 + q) * S::threads, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float2 f = __builtin_bit_cast(float2, v[q]);
          acc[i][k][2 * q] += f.x;
          acc[i][k][2 * q + 1] += f.y;
        }
      }
  return true;
}

// Rows out through LDS.  A lane holds four neighbouring columns of a row here and there: stored as they are they are 8 or 16 bytes in each of
// 32 rows.  A wavefront turns 32 rows of `bytes` in a corner of LDS of its own (nobody waits for anybody) and takes them back 16 bytes
// a lane along the rows.
template <int BYTES>
struct RowTurn {
  static constexpr int pitch = BYTES + 16, size = 32 * pitch;   // (16 bytes more: sixteen lanes that write a column meet all banks)
  char* base;
  __device__ __forceinline__ RowTurn(char* lds, int wave) : base(lds + wave * size) {}
  __device__ __forceinline__ char* at(int row, int offset) const { return base + row * pitch + offset; }
  // take(row, offset, 16 bytes) for all of the 32 rows
  template <class Take>
  __device__ __forceinline__ void each(int lane, Take take) const {
    order();
#pragma unroll
    for (int k = 0; k < BYTES / 32; ++k) {
      const int chunk = lane + 64 * k, row = chunk / (BYTES / 16), offset = chunk % (BYTES / 16) * 16;
      take(row, offset, *(const uintx4p*)at(row, offset));
    }
    order();
  }
  // take(row, column, value) for all of the single-precision values
  template <class Take>
  __device__ __forceinline__ void single(int lane, Take take) const {
    order();
#pragma unroll 4
    for (int k = 0; k < BYTES / 8; ++k) {
      const int i = lane + 64 * k, row = i / (BYTES / 4), column = i % (BYTES / 4);
      take(row, column, *(const float*)at(row, 4 * column));
    }
    order();
  }
  // (what a wavefront's lanes have written its other lanes may read: LDS accesses of a wavefront are in order, the compiler's too)
  __device__ static __forceinline__ void order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
};
// blocks of 32 columns that are turned together: 256 bytes a row where there are as many
template <class S, int SIZE>
constexpr int turned_blocks() { return S::TN * 32 * SIZE <= 256 ? S::TN : 256 / (32 * SIZE); }

// The matrices of a grid of products: one or more of one shape, `size` 16-bit values apart
struct Matrix {
  const void* base;
  long long pitch, size;
  long long rows;
  __device__ __forceinline__ Operand of(int k) const { return {(const char*)base + k * size * 2, pitch, rows}; }
};

struct TileGrid {
  int tilesM, tilesN;
  int count;           // products of one shape
  int triangle;        // only the tiles on and below the diagonal
};
// Consecutive workgroups of one XCD take kTileRows rows of tiles by as many columns as fit, so that the tiles in flight on an XCD share
// operands in its L2; the slices of a tile are neighbours.
constexpr int kTileRows = 4;

// What to do with a finished tile is E's: e.finish<S>(acc, tile row, tile column, which product, lane, wavefront along m, along n, LDS).
template <class S, bool A_ACROSS, bool B_ACROSS, int A_REPEAT, class E>
__global__ __launch_bounds__(S::threads, 2) void product_kernel(Matrix A, Matrix B, TileGrid g, int stages, Slices j, E e) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const bool whole = (int)blockIdx.x < j.full;
  const int id = whole ? xcd_contiguous_id((int)blockIdx.x, j.full) : xcd_contiguous_id((int)blockIdx.x - j.full, (int)gridDim.x - j.full);
  const int cut = whole ? 0 : id / j.slices, slice = whole ? 0 : id - cut * j.slices, tile = whole ? id : j.full + cut;
  const int per = g.triangle ? g.tilesM * (g.tilesM + 1) / 2 : g.tilesM * g.tilesN;
  const int which = tile / per, t = tile - which * per;
  int tm, tn;
  if (g.triangle) {
    tm = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > t) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
    tn = t - tm * (tm + 1) / 2;
  } else {
    const int band = kTileRows * g.tilesN;
    const int first = t / band * kTileRows, rows = min(kTileRows, g.tilesM - first);
    const int within = t - t / band * band;
    tm = first + within % rows;
    tn = within / rows;
  }
  const int s0 = slice * j.perSlice, mine = whole ? stages : max(0, min(j.perSlice, stages - s0));
  floatx16p acc[S::TM][S::TN];
  product_tile<S, A_ACROSS, B_ACROSS, A_REPEAT>(A.of(which), B.of(which), (long long)tm * S::BM, (long long)tn * S::BN, s0, mine, lds, acc);
  if (!whole && !join_slices<S>(j, cut, slice, acc, lds)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  e.template finish<S>(acc, tm, tn, which, lane, wave % S::WM, wave / S::WM, lds);
}

// ---------------------------------------------------------------------------------------------- host

enum { kTile256, kTile128, kTile64 };
constexpr int kTileSize[3] = {256, 128, 64};

// How a product is cut: the tile, how many tiles are made whole (as many rounds of the chip as there are full ones), and how many workgroups
// share the reduction of each of the others.
struct ProductPlan {
  int tile, slices, perSlice, stages;
  long long tiles, full;
  double cost;   // as the model below has it
  long long rest() const { return tiles - full; }
  long long groups() const { return full + rest() * slices; }
  size_t partBytes() const { return slices > 1 ? (size_t)rest() * slices * kTileSize[tile] * kTileSize[tile] * 4 : 0; }
  size_t counters() const { return slices > 1 ? (size_t)rest() : 0; }
  bool alone() const { return groups() <= device_compute_units(); }   // a workgroup to a CU
  // the same cut for fewer rows or columns
  ProductPlan of(long long M, long long N) const {
    ProductPlan p = *this;
    p.tiles = (M + kTileSize[tile] - 1) / kTileSize[tile] * ((N + kTileSize[tile] - 1) / kTileSize[tile]);
    p.full = std::min(full, p.tiles);
    return p;
  }
};

// The cheapest of the cuts by a model in microseconds, measured on products of 2^10 to 2^13 indices: a stage takes `alone` where a
// workgroup has its CU (nearly) to itself, `shared` per workgroup where several keep it busy; `ends` is what a tile's first loads and
// its end cost; a join costs kJoin, its parts' way to memory and back (all together at 5 TB/s, a tile's at 0.1).  (bfloat16, tiles of
// 64 / 128 / 256: 650 / 1040 / 1240 TFLOP/s with the chip full; pairs: 850 / 1140 / 1260.  P f of 2048 x 1024 over 16000 classes, pairs,
// in us: 891, 288, 225 by tiles of 256 in 1, 4, 8 slices, 412, 196, 244 by tiles of 128, 234, 338, 497 by tiles of 64; chosen: 128 in 4.)
// What is left over behind whole rounds of the chip (one workgroup of 256 to a CU, two of the smaller ones) is cut finer: 528 tiles of
// 128 by 128 stages of pairs 266 -> 210 us.
struct StageCost { double alone, shared, ends; };
constexpr StageCost kStageCost[2][3] = {{{1.5, 1.6, 8.0}, {0.48, 0.50, 3.0}, {0.29, 0.20, 1.0}},     // kBf16: 256, 128, 64
                                        {{2.3, 2.5, 8.0}, {0.65, 0.70, 3.0}, {0.30, 0.24, 1.0}}};    // kPairs
constexpr int kResident[3] = {1, 2, 2};
constexpr double kJoin = 4.0;
constexpr int kMostSlices = 32;
inline ProductPlan plan_product(int type, long long M, long long N, long long depth, int count = 1, bool triangle = false, int smallest = 0) {
  const int cus = std::max(1, device_compute_units());
  // (an unknown tile is none; a forced cut is held to what the loop below reaches)
  const int asked = tunable("product_tile", 0), forced = asked == 64 || asked == 128 || asked == 256 ? asked : 0;
  const int cut = std::max(0, std::min(tunable("product_slices", 0), kMostSlices));
  const int stages = (int)((depth + stage_depth(type) - 1) / stage_depth(type));
  ProductPlan best = {};
  double least = 1e300;
  for (int tile = 0; tile < 3; ++tile) {
    if (forced ? forced != kTileSize[tile] : kTileSize[tile] < smallest) continue;
    const long long rows = (M + kTileSize[tile] - 1) / kTileSize[tile], columns = (N + kTileSize[tile] - 1) / kTileSize[tile];
    const long long tiles = count * (triangle ? rows * (rows + 1) / 2 : rows * columns);
    const StageCost& c = kStageCost[type][tile];
    const double part = 4.0 * kTileSize[tile] * kTileSize[tile];
    const long long round = (long long)cus * kResident[tile];
    const long long full = cut ? 0 : tiles / round * round, rest = tiles - full;
    const double before = full / round * (stages * kResident[tile] * c.shared + c.ends);
    for (int slices = 1; slices <= kMostSlices && slices <= std::max(1, stages); ++slices) {
      if (cut && slices != div_up(std::max(1, stages), div_up(std::max(1, stages), cut))) continue;
      const int perSlice = std::max(1, div_up(stages, slices));
      if (slices > 1 && ((slices - 1) * perSlice >= stages || (!cut && rest * slices > 4ll * cus))) continue;   // (no empty slice; parts stay small)
      const double waves = (double)((rest * slices + cus - 1) / cus);
      const double cost = rest == 0 ? before
                                    : before + perSlice * std::max(c.alone, waves * c.shared) + c.ends * std::max(1.0, waves / 2) +
                                          (slices > 1 ? kJoin + slices * part * (2.0 * rest / 5.0e6 + 1.0 / 1.0e5) : 0.0);
      if (cost < least) {
        least = cost;
        best = {tile, slices, perSlice, stages, tiles, full, cost};
      }
    }
  }
  return best;
}

// A kernel with more than 64 KiB of local memory has to be told so once per device (`raised`: the devices where that is done, a bit each).
inline int allow_lds(const char* who, const void* kernel, int bytes, std::atomic<unsigned long long>& raised) {
  if (bytes <= 65536) return MCN_SUCCESS;
  const int dev = current_device();
  if (dev < 0) return fail(MCN_DEVICE_ERROR, "%s: no device", who);
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (raised.load(std::memory_order_relaxed) & bit) return MCN_SUCCESS;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(MCN_DEVICE_ERROR, "%s: local memory", who);
  }
  raised.fetch_or(bit, std::memory_order_relaxed);
  return MCN_SUCCESS;
}

// Where a call's products leave their parts
struct Scratch {
  float* parts;
  unsigned* counters;
};

template <class S, bool A_ACROSS, bool B_ACROSS, int A_REPEAT = 1, class E>
int run_product(hipStream_t s, const char* who, const char* name, const Matrix& A, const Matrix& B, long long M, long long N, int count, bool triangle,
                const ProductPlan& p, const Scratch& scratch, const E& e) {
  if (p.groups() >= (1ll << 32) / S::threads) return fail(MCN_UNSUPPORTED, "%s: tensor too large", who);
  const TileGrid g = {div_up(M, S::BM), div_up(N, S::BN), count, triangle};
  const auto kernel = product_kernel<S, A_ACROSS, B_ACROSS, A_REPEAT, E>;
  static std::atomic<unsigned long long> raised;
  const int rc = allow_lds(who, (const void*)kernel, S::ldsBytes, raised);
  if (rc) return rc;
  KernelTimer timer(name, s);
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.groups()), dim3(S::threads), S::ldsBytes, s, A, B, g, p.stages,
                     Slices{scratch.parts, scratch.counters, p.slices, p.perSlice, (int)p.full}, e);
  return check_launch(who);
}

template <int TYPE> using Tile256 = ProductShape<TYPE, 256, 256, 4, 2, 2>;
template <int TYPE> using Tile128 = ProductShape<TYPE, 128, 128, 2, 2, 2>;
// (a workgroup that has its CU to itself takes eight wavefronts and four stages: 256 tiles by 64 stages of pairs 50 us instead of 62, 32
// tiles 35 instead of 52; where two share a CU, 512 tiles, it is 99 us against 96, of 16 stages 33 against 31)
template <int TYPE> using Tile128Alone = ProductShape<TYPE, 128, 128, 4, 2, 4>;
template <int TYPE> using Tile64 = ProductShape<TYPE, 64, 64, 2, 2, 4>;

template <int TYPE, bool A_ACROSS, bool B_ACROSS, int A_REPEAT = 1, class E>
int product(hipStream_t s, const char* who, const char* name, const Matrix& A, const Matrix& B, long long M, long long N, const ProductPlan& p,
            const Scratch& scratch, const E& e, int count = 1, bool triangle = false) {
  if (p.tile == kTile256) return run_product<Tile256<TYPE>, A_ACROSS, B_ACROSS, A_REPEAT>(s, who, name, A, B, M, N, count, triangle, p, scratch, e);
  if (p.tile == kTile64) return run_product<Tile64<TYPE>, A_ACROSS, B_ACROSS, A_REPEAT>(s, who, name, A, B, M, N, count, triangle, p, scratch, e);
  if (p.alone()) return run_product<Tile128Alone<TYPE>, A_ACROSS, B_ACROSS, A_REPEAT>(s, who, name, A, B, M, N, count, triangle, p, scratch, e);
  return run_product<Tile128<TYPE>, A_ACROSS, B_ACROSS, A_REPEAT>(s, who, name, A, B, M, N, count, triangle, p, scratch, e);
}

}  // namespace mcn
