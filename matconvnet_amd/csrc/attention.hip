// Attention of the positions of packed sequences, heads in groups that share keys and values.
//   s_ij = scale q_i . k_j,  L_i = log sum_j exp s_ij,  p_ij = exp(s_ij - L_i),  o_i = sum_j p_ij v_j
//   backward: delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//             dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// Bound by the matrix pipe where sequences are long (4 D operations a pair of positions forward, 10 D backward) and by reading k and v where
// few queries meet many keys.  No tensor of scores: the softmax is taken along with the products, its largest score and its sum
// running.
//
// Rows.  A key head's queries are the rows r = i G + g of one matrix, i the position, g the head of the group of G: one query a sequence
// is a tile of G rows that reads its keys once, and dk, dv of a group are sums inside one workgroup.
//
// Products are v_mfma_f32_32x32x16_bf16, or 32x32x2_f32 in single precision, always with the operands such that a result's lane holds one
// index of the side that stays (a query forward and for dq, a key for dk and dv) and sixteen of the 32 of the side that is walked:
// 8 (r / 4) + 4 (lane / 32) + r % 4.  A row's maximum and sum then need one exchange between two lanes, and p or ds goes into the next
// product straight from the registers: the order of a reduction is free, so the other operand is read from LDS in the same order.
//
// The walked side comes through LDS, brought there by the DMA a tile ahead, one barrier a tile.  Rows lie there 16 bytes by 16 bytes, exchanged
// by the row so that neither reads along a row nor transposing reads across rows meet in a bank (counted: no conflict in any of the kernels).
//
// Measured (bfloat16, times of the kernels; operations counted over the pairs that are seen).  One causal sequence of 16384, 32 heads over 8 of
// 128: forward 2.12 ms, 1040 TFLOP/s; dq 3.64 and dk, dv 4.36 ms, 690 TFLOP/s, 1100 with all products counted that are made (scores and do.v in
// both kernels, dq's product twice).  32 x 196 positions, 12 heads of 64, not causal: 17, 25 and 24 us.  64 queries, one a sequence, 262144 keys in
// all, 8 heads of 128: k and v read at 4.6 TB/s (233 us).
#include "mcn_internal.hpp"

#include <algorithm>
#include <cmath>

namespace mcn {
namespace {

typedef unsigned short bf16;
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMostD = 128;
constexpr unsigned kNowhere = 0x80000000u;   // an offset behind every buffer, and so is what is a tile's size further on: reads zero

__device__ __forceinline__ float bits_float(unsigned v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ unsigned float_bits(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ unsigned short round_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bfx2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2){a, b}, bfx2));
}
__device__ __forceinline__ float power2(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ bool finite(float v) { return (float_bits(v) & 0x7f800000u) != 0x7f800000u; }

// the other half's value of the 64 lanes (lane ^ 32)
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, kWave); }
// Whether both lanes of a row (or key) find it good.  (As numbers: a lane's own bit of a ballot takes a 64-bit shift by the lane, whose result was
// wrong in half of a wavefront now and then where the compiler kept the amount in the last register that a wavefront has, v255 in dq; the slow
// sums behind the loop hid that but for their time.)
__device__ __forceinline__ bool both_good(bool good) {
  const float bad = good ? 0.f : 1.f;
  return bad + other_half(bad) == 0.f;
}

struct Tensor3 {            // heads where they lie, strides in bytes
  char* data;
  long long position, head;
};

struct AttentionP {
  Tensor3 q, k, v, o, dO, dq, dk, dv;
  float *logSums, *parts, *partSums;     // parts: a slice's o (normalised) and log sums; backward, of groupParts: [M][keyHeads][2][DW] of dk and dv
  int groupParts, headsOfPart;           // dk, dv: the group's heads in so many workgroups
  float *statL, *statD;                  // backward, [heads][N]: -L (negative_sum), -delta
  const int *qStarts, *kStarts;
  int sequences, each, eachKeys;         // without starts: queries and keys of a sequence
  int D, G, heads, keyHeads, N, M, causal;
  int slices, vector;                    // vector: outputs may be stored four values at a time
  FastDiv byG, byTiles, bySequences;     // (tiles of a sequence, sequences: without starts)
  float scale, c;                        // c = scale log2 e
};

template <class V> struct Matrix;
template <> struct Matrix<bf16> {
  static constexpr int perChunk = 8;
  // 16 bytes a lane along the reduction: lane / 32 says which of two neighbouring runs of eight
  __device__ static __forceinline__ floatx16 along(uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfx8, a), __builtin_bit_cast(bfx8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ float dot(uintx4 a, uintx4 b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += bits_float(a[e] << 16) * bits_float(b[e] << 16) + bits_float(a[e] & 0xffff0000u) * bits_float(b[e] & 0xffff0000u);
    return s;
  }
};
template <> struct Matrix<float> {
  static constexpr int perChunk = 4;
  __device__ static __forceinline__ floatx16 along(uintx4 a, uintx4 b, floatx16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(bits_float(a[e]), bits_float(b[e]), c, 0, 0, 0);
    return c;
  }
  __device__ static __forceinline__ float dot(uintx4 a, uintx4 b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += bits_float(a[e]) * bits_float(b[e]);
    return s;
  }
};

// Keeps what follows from the lane's number inside a loop's body: addresses made ahead of the loop take registers that the backward kernels of 128
// channels do not have (kept in memory, every read of one waits for the tile that is on its way).  What those kernels keep in memory all the same, 2 to
// 13 registers, is read outside of the loops over tiles but for dk and dv with two wavefronts to a block, which reads three offsets of its loads a tile.
template <class V, int DW>
__device__ __forceinline__ int fresh(int lane) {
  if (sizeof(V) == 2 && DW == 128) asm volatile("" : "+v"(lane));
  return lane;
}

// A tile in LDS: rows of DP values, of which the products take DW; chunk c (16 bytes) of a row at c ^ turn(row).  bfloat16: four rows that a transposing read takes lie in four
// 64-byte runs of banks, and sixteen rows put a chunk in sixteen places; single precision: the latter.
template <class V, int DW>
struct Tile {
  static constexpr int DP = DW <= 64 ? 64 : 128;
  static constexpr int rowBytes = DP * (int)sizeof(V), chunks = rowBytes / 16, steps = DW * (int)sizeof(V) / 32, blocks = DW / 32;
  __device__ static __forceinline__ int turn(int row) {
    if (sizeof(V) == 4) return row & 15;
    return chunks == 16 ? ((row & 3) << 2 | (row >> 2 & 3)) : ((row >> 1 & 1) << 2 | (row >> 2 & 3));
  }
  // chunks 2 s + lane / 32 of row first + lane % 32
  __device__ static __forceinline__ uintx4 along(const char* lds, int first, int s, int lane) {
    const int row = lane & 31;   // (first is a multiple of 32: the turn is the lane's own)
    return *(const uintx4*)(lds + (first + row) * rowBytes + (((2 * s) ^ (turn(row) ^ (lane >> 5))) << 4));
  }
  // (bfloat16) rows first .. first + 15 as the other operand of `across`, the 32 columns from 32 b on
  __device__ static __forceinline__ uintx4 turned(const char* lds, int first, int b, int lane) {
    typedef __attribute__((address_space(3))) shortx4* lds_shorts;
    const int quarter = (lane >> 5) * 4 + (lane >> 2 & 3), chunk = 4 * b + (lane >> 4 & 1) * 2 + (lane >> 1 & 1), within = (lane & 1) * 8;
    const int r0 = first + quarter, r1 = r0 + 8;
    const uintx2 a0 = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_shorts)(lds + r0 * rowBytes + ((chunk ^ turn(quarter)) << 4) + within)));
    const uintx2 a1 = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_shorts)(lds + r1 * rowBytes + ((chunk ^ turn(quarter + 8)) << 4) + within)));
    return (uintx4){a0.x, a0.y, a1.x, a1.y};
  }
  // acc += (rows first .. first + 31 of the tile)' x p, the 32 columns from 32 b on: p in the order of a result's registers
  __device__ static __forceinline__ floatx16 across(const char* lds, int first, int b, int lane, const uintx4 (&p)[sizeof(V) == 4 ? 4 : 2], floatx16 acc) {
    if (sizeof(V) == 2) {
#pragma unroll
      for (int s = 0; s < 2; ++s) acc = Matrix<bf16>::along(turned(lds, first + 16 * s, b, lane), p[s], acc);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = 8 * (r / 4) + 4 * (lane >> 5) + r % 4, column = 32 * b + (lane & 31);
        const float a = *(const float*)(lds + (first + row) * rowBytes + ((column / 4 ^ turn(row)) << 4) + (column & 3) * 4);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, bits_float(p[r / 4 & 3][r % 4]), acc, 0, 0, 0);
      }
    }
    return acc;
  }
  // a result's sixteen values as the operand of `across`
  __device__ static __forceinline__ void operand(uintx4 (&p)[sizeof(V) == 4 ? 4 : 2], const float (&v)[16]) {
    if (sizeof(V) == 2) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[s][e] = pack_bf16(v[8 * s + 2 * e], v[8 * s + 2 * e + 1]);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r / 4 & (sizeof(V) == 4 ? 3 : 1)][r % 4] = float_bits(v[r]);
    }
  }
};

// Brings ROWS rows of a tile into LDS: wavefront w the 1024-byte pieces w, w + NW, ...  A lane's offsets are made once; where the rows of its
// pieces are 16 apart (the turn's period) they follow from the first.  What is behind the rows that are left, or behind D, reads as zero.
template <class V, int DW, int ROWS, int NW>
struct Loader {
  typedef Tile<V, DW> T;
  static constexpr int pieces = ROWS * T::rowBytes / 1024 / NW, rowsOfPiece = 1024 / T::rowBytes;
  static constexpr bool periodic = NW * rowsOfPiece % 16 == 0;
  static_assert(ROWS * T::rowBytes % (1024 * NW) == 0, "whole pieces");
  unsigned offset[periodic ? 1 : pieces];
  unsigned pitch, width;   // bytes from row to row, and of a row
  __device__ __forceinline__ void begin(const Tensor3& t, int D, int wave, int lane) {
    pitch = (unsigned)t.position;
    width = (unsigned)(D * (int)sizeof(V) + 15) / 16 * 16;   // (rows that were packed are whole pieces of 16 bytes)
#pragma unroll
    for (int i = 0; i < (periodic ? 1 : pieces); ++i) {
      const int slot = (i * NW + wave) * 64 + lane, row = slot / T::chunks, chunk = (slot % T::chunks) ^ T::turn(row);
      offset[i] = chunk * Matrix<V>::perChunk >= D ? kNowhere : row * pitch + chunk * 16u;
    }
  }
  // from: the tile's first row; left: rows from there on (may be none)
  __device__ __forceinline__ void bring(char* lds, const char* from, int left, int wave) const {
    typedef __attribute__((address_space(3))) void* lds_ptr;
    const unsigned records = left <= 0 ? 0u : (unsigned)(std::min(left, ROWS) - 1) * pitch + width;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, (int)records, 0x00020000);
#pragma unroll
    for (int i = 0; i < pieces; ++i) {
      const unsigned at = periodic ? offset[0] + i * (NW * rowsOfPiece) * pitch : offset[i];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (i * NW + wave) * 1024), 16, (int)at, 0, 0, 0);
    }
  }
};

// N matrix instructions, step i of them on what read(i) brought from LDS DEPTH steps before: left to itself the compiler reads one step ahead, and
// every instruction waits for most of a read's latency.  Vector instructions may move among the steps.
template <int DEPTH, int N, class Read, class Step>
__device__ __forceinline__ void steps_ahead(Read read, Step step) {
  uintx4 a[DEPTH];
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) a[i] = read(i);
  __builtin_amdgcn_sched_barrier(6);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    step(i, a[i % DEPTH]);
    if (i + DEPTH < N) a[i % DEPTH] = read(i + DEPTH);
    __builtin_amdgcn_sched_barrier(6);
  }
}

// 16 bytes of a row in global memory, zero where there is none
template <class V>
__device__ __forceinline__ uintx4 chunk_of(const char* row, int chunk, int D, bool live) {
  uintx4 v = {0u, 0u, 0u, 0u};
  if (live && chunk * Matrix<V>::perChunk < D) v = *(const uintx4*)(row + chunk * 16);
  return v;
}

// The sums of a row of D values times a weight onto a result's lane: the columns that the lane holds
template <class V, int DW>
__device__ __forceinline__ void add_row(floatx16 (&acc)[DW / 32], const char* row, float weight, int D, int lane) {
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int at = 32 * d + 2 * r + 4 * (lane >> 5);
      if (at >= D) continue;   // (rows are whole pieces of 16 bytes)
      if (sizeof(V) == 2) {
        const uintx2 v = *(const uintx2*)(row + 2 * at);
        acc[d][r] += weight * bits_float(v.x << 16);
        acc[d][r + 1] += weight * bits_float(v.x & 0xffff0000u);
        acc[d][r + 2] += weight * bits_float(v.y << 16);
        acc[d][r + 3] += weight * bits_float(v.y & 0xffff0000u);
      } else {
        const uintx4 v = *(const uintx4*)(row + 4 * at);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][r + e] += weight * bits_float(v[e]);
      }
      if (r % 8 == 4) __builtin_amdgcn_sched_barrier(0);
    }
}
// All finite, in both lanes of a row (or key)
template <int N>
__device__ __forceinline__ bool all_finite(const floatx16 (&v)[N]) {
  bool good = true;
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) good = good && finite(v[d][r]);
  return both_good(good);
}
// The product of two rows in global memory, by a lane and its other half.  (From memory again, and two loads at a time: what the slow sums
// behind a loop keep in registers the loop does not have.)
template <class V, int DW>
__device__ __forceinline__ float row_product(const char* a, const char* b, int D, int lane) {
  float s = 0.f;
#pragma unroll 1
  for (int k = 0; k < Tile<V, DW>::steps; ++k) s += Matrix<V>::dot(chunk_of<V>(a, 2 * k + (lane >> 5), D, true), chunk_of<V>(b, 2 * k + (lane >> 5), D, true));
  return s + other_half(s);
}
// The first (LAST: the last) row of [from, to) that holds what is not finite; none: behind (ahead of) all.  All lanes look, some rows at a time.
__device__ __forceinline__ bool two_finite(unsigned v) { return (v & 0x7f800000u) != 0x7f800000u && (v & 0x7f80u) != 0x7f80u; }
template <class V, int DW, bool LAST>
__device__ __forceinline__ int bad_row(const char* rows, long long pitch, int D, int from, int to, int lane) {
  constexpr int chunks = Tile<V, DW>::chunks, step = 64 / chunks;
#pragma unroll 1
  for (int j = 0; j < to - from; j += step) {
    const int at = j + lane / chunks, row = LAST ? to - 1 - at : from + at;
    const uintx4 v = chunk_of<V>(rows + row * pitch, lane % chunks, D, at < to - from);
    bool good = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) good = good && (sizeof(V) == 2 ? two_finite(v[e]) : finite(bits_float(v[e])));
    const unsigned long long bad = __ballot(!good);
    if (bad) {
      const int found = j + __builtin_ctzll(bad) / chunks;
      return LAST ? to - 1 - found : from + found;
    }
  }
  return LAST ? -1 : 0x7fffffff;
}
template <class V>
__device__ __forceinline__ float as_operand(float v) { return sizeof(V) == 2 ? bits_float((unsigned)round_bf16(v) << 16) : v; }

// Four neighbouring values of a row out
template <class V>
__device__ __forceinline__ void store4(char* row, int d, int D, int vector, float a, float b, float c, float e) {
  if (vector) {
    if (d >= D) return;
    if (sizeof(V) == 2) *(uintx2*)(row + 2 * d) = (uintx2){pack_bf16(a, b), pack_bf16(c, e)};
    else *(uintx4*)(row + 4 * d) = (uintx4){float_bits(a), float_bits(b), float_bits(c), float_bits(e)};
    return;
  }
  const float v[4] = {a, b, c, e};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (d + k >= D) return;
    if (sizeof(V) == 2) ((bf16*)row)[d + k] = round_bf16(v[k]);
    else ((float*)row)[d + k] = v[k];
  }
}

// ------------------------------------------------------------------------------------------ which sequence

struct Span {
  int q0, n, k0, m;   // the sequence's queries and keys
  int first;          // first row (or key) of the tile, -1: nothing to do
};

__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// of all lanes: sixteen by the vector instructions' own lane exchange, the four of these as scalars (shuffles go through LDS and are waited for)
template <int CONTROL>
__device__ __forceinline__ int exchanged(int v) { return __builtin_amdgcn_update_dpp(0, v, CONTROL, 0xf, 0xf, true); }
template <class F>
__device__ __forceinline__ int over_wave(int v, F f) {
  v = f(v, exchanged<0xB1>(v));    // lane ^ 1
  v = f(v, exchanged<0x4E>(v));    // lane ^ 2
  v = f(v, exchanged<0x141>(v));   // the other four of eight, mirrored
  v = f(v, exchanged<0x140>(v));   // the other eight of sixteen, mirrored
  return f(f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)), f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_total(int v) { return over_wave(v, [](int a, int b) { return a + b; }); }
__device__ __forceinline__ int wave_most(int v) { return over_wave(v, [](int a, int b) { return a > b ? a : b; }); }

// Tile `tile` of SIZE rows (KEYS: keys) of all sequences'.  Causal tiles differ in their work (rows: the last of a sequence see the most keys;
// keys: the first are seen by the most rows), so they are taken in the order of falling work, over all sequences: of the
// `level`-th most first.  (13 sequences of up to 1100 positions, dk and dv: a sequence's tiles one after the other left a tail of a third.)
// With starts on the device and more than 64 sequences, sequence s has the tiles from before(s)/SIZE + s on, before(s) the rows ahead
// of it: no tile holds two sequences, floor(b/SIZE) + 1 numbers are enough for any, so the number of all tiles is known without the starts;
// the sequence is found 64 candidates at a time, all loads of a step at once.
template <int SIZE, bool KEYS>
__device__ __forceinline__ Span find(const AttentionP& p, int tile, int lane) {
  Span s;
  int t = -1, lo;
  if (!p.qStarts) {
    int seq;
    const int tiles = p.byTiles.d;
    if (p.causal) {
      p.bySequences.divmod(tile, &t, &seq);
      if (!KEYS) t = tiles - 1 - t;
    } else {
      p.byTiles.divmod(tile, &seq, &t);
    }
    s.q0 = seq * p.each; s.n = p.each;
    s.k0 = seq * p.eachKeys; s.m = p.eachKeys;
    const int rows = KEYS ? s.m : s.n * p.G;
    s.first = t >= 0 && t * SIZE < rows ? t * SIZE : -1;
    return s;
  }
  if (p.causal && p.sequences <= 64) {
    int q0 = 0, n = 0, k0 = 0, m = 0;   // of sequence `lane`
    if (lane < p.sequences) {
      const int a = p.qStarts[lane], b = p.qStarts[lane + 1], c = p.kStarts[lane], d = p.kStarts[lane + 1];
      q0 = clamped(a, p.N);
      n = std::max(0, clamped(b, p.N) - q0);
      k0 = clamped(c, p.M);
      m = std::max(0, clamped(d, p.M) - k0);
    }
    const int count = ((KEYS ? m : n * p.G) + SIZE - 1) / SIZE;   // its tiles
    // level l: tiles with l - 1 lighter ones in their sequence; those of level `low` or above are more than `tile`
    int low = 1, high = wave_most(count) + 1;
    int above = 0;               // tiles of level `high` or above
    if (wave_total(count) <= tile) low = 0;
    else
      while (high - low > 1) {
        const int mid = (low + high) / 2, total = wave_total(std::max(0, count - mid + 1));
        if (total > tile) low = mid;
        else {
          high = mid;
          above = total;
        }
      }
    const unsigned long long some = __ballot(count >= low && lane < p.sequences);
    const int rank = __builtin_amdgcn_mbcnt_hi((unsigned)(some >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)some, 0));
    const unsigned long long one = __ballot(count >= low && lane < p.sequences && rank == tile - above);
    lo = __builtin_amdgcn_readfirstlane(one && low ? __builtin_ctzll(one) : 0);
    const int tiles = __builtin_amdgcn_readlane(count, lo);
    t = !low || !one ? -1 : KEYS ? tiles - low : low - 1;
    s.q0 = __builtin_amdgcn_readlane(q0, lo);
    s.n = __builtin_amdgcn_readlane(n, lo);
    s.k0 = __builtin_amdgcn_readlane(k0, lo);
    s.m = __builtin_amdgcn_readlane(m, lo);
    t = __builtin_amdgcn_readfirstlane(t);
    s.first = t < 0 || t >= tiles ? -1 : t * SIZE;
    return s;
  }
  const auto before = [&](int i) { return (KEYS ? clamped(p.kStarts[i], p.M) : clamped(p.qStarts[i], p.N) * p.G) / SIZE + i; };
  int n = p.sequences;
  lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const unsigned long long below = __ballot(lane * step < n && before(i) <= tile);
    const int found = below ? 63 - __builtin_clzll(below) : 0;
    lo += found * step;
    n = std::min(step, n - found * step);
  }
  t = tile - before(lo);
  lo = __builtin_amdgcn_readfirstlane(lo);
  t = __builtin_amdgcn_readfirstlane(t);
  s.q0 = clamped(p.qStarts[lo], p.N);
  s.n = std::max(0, clamped(p.qStarts[lo + 1], p.N) - s.q0);
  s.k0 = clamped(p.kStarts[lo], p.M);
  s.m = std::max(0, clamped(p.kStarts[lo + 1], p.M) - s.k0);
  const int rows = KEYS ? s.m : s.n * p.G, tiles = (rows + SIZE - 1) / SIZE;
  if (p.causal && !KEYS && p.sequences > 64 && t >= 0) t = tiles - 1 - t;   // (within a sequence, at least)
  s.first = t < 0 || t >= tiles ? -1 : t * SIZE;
  return s;
}

// ------------------------------------------------------------------------------------------ forward

constexpr int kAhead = 2;   // tiles in LDS at a time: the one that is walked, the one that comes

// KB blocks of 32 keys of a tile: fragments of 32 queries (q) against them.  `next` is filled meanwhile.  (A function of its own with `restrict` pointers:
// that the loads fill none of what is read is what lets the reads go without waiting for them.)
template <class V, int DW, int KB, class Bring>
__device__ __forceinline__ void forward_tile(const char* __restrict__ keys, const char* __restrict__ values, char* __restrict__ next, Bring bring_next,
                                             const uintx4 (&q)[Tile<V, DW>::steps], floatx16 (&o)[DW / 32], float& most, float& sum, int j0, int limit,
                                             bool edge, float c, int lane) {
  typedef Tile<V, DW> T;
  bring_next(next);
  floatx16 s[KB];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
  // masks, the running maximum; then exponentials
  const auto largest = [&]() __attribute__((always_inline)) {
    if (edge) {
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (j0 + 32 * b + 8 * (r / 4) + 4 * (lane >> 5) + r % 4 >= limit) s[b][r] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, s[b][r]);
    m = fmaxf(m, other_half(m));
    // The reference of the exponentials is raised only when a score lies more than 2^8 above it: what is summed stays below 2^8 a key, and the
    // outputs are scaled anew a few times in all instead of every tile.
    const bool raise = m * c > most * c + 8.f || (most == -INFINITY && m > -INFINITY);
    if (__any(raise)) {
      const float to = raise ? m : most;
      const float f = raise ? (most == -INFINITY ? 0.f : power2((most - to) * c)) : 1.f;
      most = to;
      sum *= f;
#pragma unroll
      for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
  };
  uintx4 operand[KB][sizeof(V) == 4 ? 4 : 2];
  // (bfloat16: each is rounded for its product with v, and not in the sum.  The roundings are independent and partly cancel over the keys: o is off by
  // 0.0021 of itself where its own rounding alone leaves 0.0017; a second bfloat16 part of each would be half as many products again.)
  const auto exponentials = [&](int b) __attribute__((always_inline)) {
    const float shift = most == -INFINITY ? 0.f : most * c;
    float e[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) e[r] = power2(s[b][r] * c - shift);
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += e[r];
    T::operand(operand[b], e);
  };
  if constexpr (sizeof(V) == 2) {
    constexpr int S = T::steps, P = DW / 32 * 2;   // steps of a block of 32 keys: scores, outputs
    steps_ahead<S, KB * (S + P)>(
        [&](int i) __attribute__((always_inline)) {
          if (i < KB * S) return T::along(keys, 32 * (i / S), i % S, lane);
          i -= KB * S;
          return T::turned(values, 32 * (i / P) + 16 * (i % 2), i % P / 2, lane);
        },
        [&](int i, uintx4 a) __attribute__((always_inline)) {
          if (i < KB * S) {
            s[i / S] = Matrix<V>::along(a, q[i % S], s[i / S]);
            return;
          }
          i -= KB * S;
          if (i == 0) {
            largest();
#pragma unroll
            for (int b = 0; b < KB; ++b) exponentials(b);
          }
          o[i % P / 2] = Matrix<V>::along(a, operand[i / P][i % 2], o[i % P / 2]);
        });
  } else {
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int k = 0; k < T::steps; ++k) s[b] = Matrix<V>::along(T::along(keys, 32 * b, k, lane), q[k], s[b]);
    largest();
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      exponentials(b);
#pragma unroll
      for (int d = 0; d < DW / 32; ++d) o[d] = T::across(values, 32 * b, d, lane, operand[b], o[d]);
    }
  }
}

// NB blocks of 32 rows, tiles of KT keys; NS wavefronts share a block, each takes its blocks of 32 keys of every tile, and what they have is put
// together through LDS.
template <class V, int DW, int NB, int NS, int KT>
__global__ __launch_bounds__(64 * NB * NS, NB * NS == 1 ? 1 : 2) void attention_forward(AttentionP p) {
  typedef Tile<V, DW> T;
  constexpr int NW = NB * NS, KB = KT / 32 / NS, tileBytes = KT * T::rowBytes;
  __shared__ __attribute__((aligned(16))) char lds[kAhead * 2 * tileBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = wave % NB, share0 = wave / NB * KB * 32;
  int id = blockIdx.x;
  const int head = id % p.keyHeads;
  id /= p.keyHeads;
  const int slice = id % p.slices;
  const Span span = find<32 * NB, false>(p, id / p.slices, lane);
  if (span.first < 0) return;
  const int rows = span.n * p.G, off = span.m - span.n;
  const int row = span.first + 32 * block + (lane & 31);
  const bool live = row < rows;
  int i, g;
  p.byG.divmod(live ? row : 0, &i, &g);
  const int limit = !live ? 0 : p.causal ? std::max(0, std::min(span.m, i + off + 1)) : span.m;
  // keys that some row of the workgroup sees
  int end = span.m;
  if (p.causal) end = std::max(0, std::min(end, p.byG.div(std::min(rows, span.first + 32 * NB) - 1) + off + 1));
  int begin = 0;
  if (p.slices > 1) {
    const int share = ((end + p.slices - 1) / p.slices + KT - 1) / KT * KT;
    begin = std::min(end, slice * share);
    end = std::min(end, begin + share);
  }
  // ... that all rows of the wavefront see (those of its first row), and the last that some row sees
  const int all = p.causal ? std::max(0, std::min(span.m, p.byG.div(std::min(rows - 1, span.first + 32 * block)) + off + 1)) : span.m;
  const int some = span.first + 32 * block >= rows ? 0
                   : p.causal ? std::max(0, std::min(span.m, p.byG.div(std::min(rows, span.first + 32 * block + 32) - 1) + off + 1)) : span.m;

  const long long position = span.q0 + i;
  const int column = head * p.G + g;
  uintx4 q[T::steps];
  {
    const char* at = p.q.data + position * p.q.position + column * p.q.head;
#pragma unroll
    for (int s = 0; s < T::steps; ++s) q[s] = chunk_of<V>(at, 2 * s + (lane >> 5), p.D, live);
  }
  const char* keys = p.k.data + (long long)span.k0 * p.k.position + head * p.k.head;
  const char* values = p.v.data + (long long)span.k0 * p.v.position + head * p.v.head;
  Loader<V, DW, KT, NW> loadK, loadV;
  loadK.begin(p.k, p.D, wave, lane);
  loadV.begin(p.v, p.D, wave, lane);
  const char* nextK = keys + (long long)begin * p.k.position;   // the tile that is brought next
  const char* nextV = values + (long long)begin * p.v.position;
  const auto bring_tile = [&](char* to, int left) __attribute__((always_inline)) {
    loadK.bring(to, nextK, left, wave);
    loadV.bring(to + tileBytes, nextV, left, wave);
    nextK += (long long)KT * p.k.position;
    nextV += (long long)KT * p.v.position;
  };
  floatx16 o[DW / 32];
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float most = -INFINITY, sum = 0.f;
  if (begin < end) bring_tile(lds, end - begin);
  int turn = 0;
  for (int j0 = begin; j0 < end; j0 += KT) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    char* from = lds + turn * 2 * tileBytes;
    char* to = lds + (turn ^ 1) * 2 * tileBytes;
    turn ^= 1;
    const auto bring_next = [&](char* at) __attribute__((always_inline)) {
      if (j0 + KT < end) bring_tile(at, end - j0 - KT);
    };
    const int j = j0 + share0;
    if (j < std::min(some, end))
      forward_tile<V, DW, KB>(from + share0 * T::rowBytes, from + tileBytes + share0 * T::rowBytes, to, bring_next, q, o, most, sum, j, std::min(limit, end),
                              j + 32 * KB > std::min(all, end), p.c, lane);
    else bring_next(to);
  }
  sum += other_half(sum);
  if (NS == 2) {
    constexpr int values = DW / 32 * 16 + 2;
    static_assert(NS == 1 || NB * values * 256 <= (int)sizeof(lds), "room");
    float* room = (float*)lds + block * values * 64 + lane;
    __syncthreads();
    if (share0) {
#pragma unroll
      for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) room[(16 * d + r) * 64] = o[d][r];
      room[(values - 2) * 64] = most;
      room[(values - 1) * 64] = sum;
    }
    __syncthreads();
    if (share0) return;
    const float most1 = room[(values - 2) * 64], to = fmaxf(most, most1);
    const float f = most == -INFINITY ? 0.f : power2((most - to) * p.c), f1 = most1 == -INFINITY ? 0.f : power2((most1 - to) * p.c);
    sum = sum * f + room[(values - 1) * 64] * f1;
    most = to;
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f + room[(16 * d + r) * 64] * f1;
  }
  // A key that a row does not see has p = 0, but 0 times an infinity or a NaN of its values is NaN.  A row that is not finite, and that some key of the
  // tiles it walked which it does not see, and none that it sees, may have made so, is added up key by key over those it sees; the others keep
  // what they have.  (Found out behind the loop, from the values themselves: what the loop would have to note on the way takes registers of
  // it, and is lost where two wavefronts share a block.)
  if (p.causal) {
    bool mend = live && !all_finite(o);
    const int last = std::min(end, some + 32 * KB - 1);   // behind the last key of these tiles
    if (__any(mend)) {   // (all lanes look)
      const int row = bad_row<V, DW, true>(values, p.v.position, p.D, std::max(begin, all), last, lane);
      mend = mend && row >= limit;
    }
    if (__any(mend)) {
      const int row = bad_row<V, DW, false>(values, p.v.position, p.D, begin, last, lane);
      mend = mend && row >= limit;
    }
    if (__any(mend)) {
      if (mend) {
#pragma unroll
        for (int d = 0; d < DW / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
      }
      const float shift = most == -INFINITY ? 0.f : most * p.c;
      const char* query = p.q.data + position * p.q.position + column * p.q.head;
#pragma unroll 1
      for (int j = begin; j < std::min(some, end); ++j) {
        const float e = power2(row_product<V, DW>(query, keys + (long long)j * p.k.position, p.D, lane) * p.c - shift);
        if (mend && j < limit) add_row<V, DW>(o, values + (long long)j * p.v.position, as_operand<V>(e), p.D, lane);
      }
    }
  }
  if (!live) return;
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float total = sum == 0.f ? -INFINITY : most * p.scale + logf(sum);
  const long long index = position * p.heads + column;
  if (p.slices == 1) {
    if (lane < 32 && p.logSums) p.logSums[index] = total;
    char* at = p.o.data + position * p.o.position + column * p.o.head;
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store4<V>(at, 32 * d + 8 * (r / 4) + 4 * (lane >> 5), p.D, p.vector, o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv);
  } else {
    const long long part = (long long)slice * p.N * p.heads + index;
    if (lane < 32) p.partSums[part] = total;
    char* at = (char*)(p.parts + part * DW);
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store4<float>(at, 32 * d + 8 * (r / 4) + 4 * (lane >> 5), DW, 1, o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv);
  }
}

// The slices of a row put together: o = sum_s exp(L_s - L) o_s.  A wavefront per row and head; rows of no sequence are passed over.
template <class V, int DW>
__global__ __launch_bounds__(256) void attention_join(AttentionP p) {
  const int lane = threadIdx.x & 63;
  const long long index = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), all = (long long)p.N * p.heads;
  if (index >= all) return;
  const int position = (int)(index / p.heads), column = (int)(index % p.heads);
  if (p.qStarts && (position < clamped(p.qStarts[0], p.N) || position >= clamped(p.qStarts[p.sequences], p.N))) return;
  const float mine = lane < p.slices ? p.partSums[lane * all + index] : -INFINITY;
  float most = mine;
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) most = fmaxf(most, __shfl_xor(most, k, kWave));
  // (a NaN of one slice is a NaN of the row)
  const float weight = most == -INFINITY && mine == mine ? 0.f : power2((mine - most) * kLog2e);
  const float sum = wave_sum(weight);
  constexpr int W = (DW + 63) / 64;
  float o[W];
#pragma unroll
  for (int w = 0; w < W; ++w) o[w] = 0.f;
  for (int s = 0; s < p.slices; ++s) {
    const float f = __shfl(weight, s, kWave);
    if (f == 0.f) continue;
    const float* at = p.parts + (s * all + index) * DW + lane;
#pragma unroll
    for (int w = 0; w < W; ++w) o[w] += f * (DW % 64 == 0 || lane + 64 * w < DW ? at[64 * w] : 0.f);
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (lane == 0 && p.logSums) p.logSums[index] = sum == 0.f ? -INFINITY : most + logf(sum);
  char* at = p.o.data + position * p.o.position + column * p.o.head;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int d = lane + 64 * w;
    if (d >= p.D) continue;
    if (sizeof(V) == 2) ((bf16*)at)[d] = round_bf16(o[w] * inv);
    else ((float*)at)[d] = o[w] * inv;
  }
}

// ------------------------------------------------------------------------------------------ dq, and delta for dk and dv

// p = exp(scale q.k - L).  bfloat16: the sum of products starts at -L/scale, which saves an addition; in single precision that would round every
// partial sum to the places that L/scale leaves, so there it starts at 0 (dq of heads of 75 channels: off by 5e-7 instead of 1.1e-6).
template <class V>
__device__ constexpr bool starts_at_sum() { return sizeof(V) == 2; }
template <class V>
__device__ __forceinline__ float negative_sum(float logSum, float scale) {   // (a row that sees nothing: what it gives is masked)
  return logSum == -INFINITY ? 0.f : starts_at_sum<V>() ? -logSum / scale : -logSum * kLog2e;
}
template <class V>
__device__ __forceinline__ float probability(float s, float negL, float c) { return starts_at_sum<V>() ? power2(s * c) : power2(s * c + negL); }

template <class V, int DW, int KB, class Bring>
__device__ __forceinline__ void dq_tile(const char* __restrict__ keys, const char* __restrict__ values, char* __restrict__ next, Bring bring_next,
                                        const uintx4 (&q)[Tile<V, DW>::steps], const uintx4 (&dO)[Tile<V, DW>::steps], floatx16 (&dq)[DW / 32], float& rest,
                                        float negL, float negDelta, int j0, int limit, int last, bool edge, float c, int lane) {
  typedef Tile<V, DW> T;
  bring_next(next);
  lane = fresh<V, DW>(lane);
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    if (b && j0 + 32 * b >= last) break;
    floatx16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = starts_at_sum<V>() ? negL : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = negDelta;
    uintx4 operand[sizeof(V) == 4 ? 4 : 2], low[2];
    const auto scores = [&]() __attribute__((always_inline)) {
      float e[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) e[r] = probability<V>(s[r], negL, c) * dp[r];
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (j0 + 32 * b + 8 * (r / 4) + 4 * (lane >> 5) + r % 4 >= limit) e[r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) rest += e[r];
      T::operand(operand, e);
      // ds as two bfloat16 values: its sums over the keys are small beside its terms (they add up to zero against equal keys), and what one rounding
      // of each leaves is as large as the result's own
      if (sizeof(V) == 2) {
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const unsigned high = operand[r / 8 & 1][r % 8 / 2];
          e[r] -= bits_float(high << 16);
          e[r + 1] -= bits_float(high & 0xffff0000u);
          low[r / 8 & 1][r % 8 / 2] = pack_bf16(e[r], e[r + 1]);
        }
      }
    };
    if constexpr (sizeof(V) == 2) {
      constexpr int S = T::steps, P = DW / 32 * 2;
      steps_ahead<3, 2 * S + P>(
          [&](int i) __attribute__((always_inline)) {
            if (i < S) return T::along(keys, 32 * b, i, lane);
            if (i < 2 * S) return T::along(values, 32 * b, i - S, lane);
            return T::turned(keys, 32 * b + 16 * (i % 2), (i - 2 * S) / 2, lane);
          },
          [&](int i, uintx4 a) __attribute__((always_inline)) {
            if (i < S) s = Matrix<V>::along(a, q[i], s);
            else if (i < 2 * S) dp = Matrix<V>::along(a, dO[i - S], dp);
            else {
              if (i == 2 * S) scores();
              dq[(i - 2 * S) / 2] = Matrix<V>::along(a, operand[i % 2], dq[(i - 2 * S) / 2]);
              dq[(i - 2 * S) / 2] = Matrix<V>::along(a, low[i % 2], dq[(i - 2 * S) / 2]);
            }
          });
    } else {
#pragma unroll
      for (int k = 0; k < T::steps; ++k) s = Matrix<V>::along(T::along(keys, 32 * b, k, lane), q[k], s);
#pragma unroll
      for (int k = 0; k < T::steps; ++k) dp = Matrix<V>::along(T::along(values, 32 * b, k, lane), dO[k], dp);
      scores();
#pragma unroll
      for (int d = 0; d < DW / 32; ++d) dq[d] = T::across(keys, 32 * b, d, lane, operand, dq[d]);
    }
  }
}

// (NB, NS, KT: as in the forward pass)
template <class V, int DW, int NB, int NS, int KT>
__global__ __launch_bounds__(64 * NB * NS, sizeof(V) == 4 ? 1 : 2) void attention_dq(AttentionP p) {
  typedef Tile<V, DW> T;
  constexpr int NW = NB * NS, KB = KT / 32 / NS, tileBytes = KT * T::rowBytes;
  __shared__ __attribute__((aligned(16))) char lds[kAhead * 2 * tileBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = wave % NB, share0 = wave / NB * KB * 32;
  const int head = blockIdx.x % p.keyHeads;
  const Span span = find<32 * NB, false>(p, blockIdx.x / p.keyHeads, lane);
  if (span.first < 0) return;
  const int rows = span.n * p.G, off = span.m - span.n;
  const int row = span.first + 32 * block + (lane & 31);
  const bool live = row < rows;
  int i, g;
  p.byG.divmod(live ? row : 0, &i, &g);
  const int limit = !live ? 0 : p.causal ? std::max(0, std::min(span.m, i + off + 1)) : span.m;
  int end = span.m;
  if (p.causal) end = std::max(0, std::min(end, p.byG.div(std::min(rows, span.first + 32 * NB) - 1) + off + 1));
  const int all = p.causal ? std::max(0, std::min(span.m, p.byG.div(std::min(rows - 1, span.first + 32 * block)) + off + 1)) : span.m;
  const int some = span.first + 32 * block >= rows ? 0
                   : p.causal ? std::max(0, std::min(span.m, p.byG.div(std::min(rows, span.first + 32 * block + 32) - 1) + off + 1)) : span.m;
  const long long position = span.q0 + i;
  const int column = head * p.G + g;
  uintx4 q[T::steps], dO[T::steps];
  float negDelta = 0.f;
  {
    const char* at = p.q.data + position * p.q.position + column * p.q.head;
    const char* dAt = p.dO.data + position * p.dO.position + column * p.dO.head;
    const char* oAt = p.o.data + position * p.o.position + column * p.o.head;
#pragma unroll
    for (int s = 0; s < T::steps; ++s) dO[s] = chunk_of<V>(dAt, 2 * s + (lane >> 5), p.D, live);
#pragma unroll
    for (int s = 0; s < T::steps; ++s) negDelta -= Matrix<V>::dot(dO[s], chunk_of<V>(oAt, 2 * s + (lane >> 5), p.D, live));
#pragma unroll
    for (int s = 0; s < T::steps; ++s) q[s] = chunk_of<V>(at, 2 * s + (lane >> 5), p.D, live);
  }
  negDelta += other_half(negDelta);
  const float negL = live ? negative_sum<V>(p.logSums[position * p.heads + column], p.scale) : 0.f;
  float rest = 0.f;
  if (!p.dq.data && !p.dk.data) {   // (dv needs the log sums alone)
    if (live && lane < 32 && !share0) {
      const long long at = (long long)column * p.N + position;
      p.statL[at] = negL;
      p.statD[at] = negDelta;   // (what dk is made of and left out of)
    }
    return;
  }
  const char* keys = p.k.data + (long long)span.k0 * p.k.position + head * p.k.head;
  const char* values = p.v.data + (long long)span.k0 * p.v.position + head * p.v.head;
  Loader<V, DW, KT, NW> loadK, loadV;
  loadK.begin(p.k, p.D, wave, lane);
  loadV.begin(p.v, p.D, wave, lane);
  const char* nextK = keys;   // the tile that is brought next
  const char* nextV = values;
  const auto bring_tile = [&](char* to, int left) __attribute__((always_inline)) {
    loadK.bring(to, nextK, left, wave);
    loadV.bring(to + tileBytes, nextV, left, wave);
    nextK += (long long)KT * p.k.position;
    nextV += (long long)KT * p.v.position;
  };
  floatx16 dq[DW / 32];
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  if (end > 0) bring_tile(lds, end);
  int turn = 0;
  for (int j0 = 0; j0 < end; j0 += KT) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    char* from = lds + turn * 2 * tileBytes;
    char* to = lds + (turn ^ 1) * 2 * tileBytes;
    turn ^= 1;
    const auto bring_next = [&](char* at) __attribute__((always_inline)) {
      if (j0 + KT < end) bring_tile(at, end - j0 - KT);
    };
    const int j = j0 + share0;
    if (j < std::min(some, end))
      dq_tile<V, DW, KB>(from + share0 * T::rowBytes, from + tileBytes + share0 * T::rowBytes, to, bring_next, q, dO, dq, rest, negL, negDelta, j,
                         limit, std::min(some, end), j + 32 * KB > std::min(all, end), p.c, lane);
    else bring_next(to);
  }
  if (NS == 2) {
    constexpr int values = DW / 32 * 16 + 1;
    static_assert(NS == 1 || NB * values * 256 <= (int)sizeof(lds), "room");
    float* room = (float*)lds + block * values * 64 + lane;
    __syncthreads();
    if (share0) {
#pragma unroll
      for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) room[(16 * d + r) * 64] = dq[d][r];
      room[(values - 1) * 64] = rest;
    }
    __syncthreads();
    if (share0) return;
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] += room[(16 * d + r) * 64];
    rest += room[(values - 1) * 64];
  }
  // delta is the sum of p (do.v) over the keys, o in do.o is rounded: what ds adds up to, instead of zero, is what delta was off by
  rest += other_half(rest);
  if (live && lane < 32) {
    const long long at = (long long)column * p.N + position;
    p.statL[at] = negL;
    p.statD[at] = negDelta - rest;
  }
  if (!p.dq.data) return;
  // (as in the forward pass, with the keys in the place of the values)
  if (p.causal) {
    bool mend = live && !all_finite(dq);
    const int last = std::min(end, some + 32 * KB - 1);
    if (__any(mend)) {
      const int row = bad_row<V, DW, true>(keys, p.k.position, p.D, all, last, lane);
      mend = mend && row >= limit;
    }
    if (__any(mend)) {
      const int row = bad_row<V, DW, false>(keys, p.k.position, p.D, 0, last, lane);
      mend = mend && row >= limit;
    }
    if (__any(mend)) {
      if (mend) {
#pragma unroll
        for (int d = 0; d < DW / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
      }
      const char* query = p.q.data + position * p.q.position + column * p.q.head;
      const char* der = p.dO.data + position * p.dO.position + column * p.dO.head;
#pragma unroll 1
      for (int j = 0; j < std::min(some, end); ++j) {
        const char* key = keys + (long long)j * p.k.position;
        const float e = probability<V>((starts_at_sum<V>() ? negL : 0.f) + row_product<V, DW>(query, key, p.D, lane), negL, p.c) *
                        (negDelta + row_product<V, DW>(der, values + (long long)j * p.v.position, p.D, lane));
        if (mend && j < limit) add_row<V, DW>(dq, key, e, p.D, lane);
      }
    }
  }
  if (!live) return;
  char* at = p.dq.data + position * p.dq.position + column * p.dq.head;
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      store4<V>(at, 32 * d + 8 * (r / 4) + 4 * (lane >> 5), p.D, p.vector, dq[d][r] * p.scale, dq[d][r + 1] * p.scale, dq[d][r + 2] * p.scale,
                dq[d][r + 3] * p.scale);
}

// ------------------------------------------------------------------------------------------ dk, dv

// 32 positions of a head against a wavefront's 32 keys
// (AHEAD: LDS is read three steps ahead, where the registers for it are there and cost no wavefront: heads of 96, and of 64 where two wavefronts
// share a block.  2 x 1024 positions, 8 heads of 64: 20.9 -> 19.0 us; with four wavefronts alone, of which three fit a SIMD as it is, 32 x 196
// positions, 12 heads of 64: 23 -> 26.)
template <class V, int DW, bool AHEAD, class Bring>
__device__ __forceinline__ void dkv_tile(const char* __restrict__ queries, const char* __restrict__ ders, const float* __restrict__ statL,
                                         const float* __restrict__ statD, char* __restrict__ next, Bring bring_next, const uintx4 (&k)[Tile<V, DW>::steps],
                                         const uintx4 (&v)[Tile<V, DW>::steps], floatx16 (&dk)[DW / 32], floatx16 (&dv)[DW / 32], int i0, int n, int firstOf,
                                         bool edge, float c, int lane) {
  typedef Tile<V, DW> T;
  bring_next(next);
  lane = fresh<V, DW>(lane);
  floatx16 s, dp;
  float e[16];
  uintx4 operand[sizeof(V) == 4 ? 4 : 2];
  const auto start = [&](floatx16& v, const float* stat) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const float4 l = *(const float4*)(stat + 2 * r + 4 * (lane >> 5));
      v[r] = l.x; v[r + 1] = l.y; v[r + 2] = l.z; v[r + 3] = l.w;
    }
  };
  start(s, statL);
  const floatx16 sums = s;   // (used in single precision)
  if (!starts_at_sum<V>()) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
  }
  const auto masked = [&]() __attribute__((always_inline)) {   // (firstOf: the first position that sees this lane's key)
    if (!edge) return;
    const int here = i0 + 4 * (lane >> 5), low = firstOf - here, high = n - here;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) + r % 4 < low || 8 * (r / 4) + r % 4 >= high) e[r] = 0.f;
  };
  // (bfloat16: p is rounded for dv and ds for dk, once each, as p is forward: both are off by 0.0023 of themselves)
  const auto probabilities = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) e[r] = probability<V>(s[r], sums[r], c);
    masked();
    T::operand(operand, e);
  };
  const auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) e[r] *= dp[r];
    masked();
    T::operand(operand, e);
  };
  if constexpr (AHEAD) {
    constexpr int S = T::steps, P = DW / 32 * 2;   // steps of the products with rows as they lie, and with rows turned
    start(dp, statD);
    steps_ahead<3, 2 * (S + P)>(
        [&](int i) __attribute__((always_inline)) {
          const char* rows = (i < S || i >= 2 * S + P) ? queries : ders;
          if (i < S || (i >= S + P && i < 2 * S + P)) return T::along(rows, 0, i < S ? i : i - S - P, lane);
          i -= i < S + P ? S : 2 * S + P;
          return T::turned(rows, 16 * (i % 2), i / 2, lane);
        },
        [&](int i, uintx4 a) __attribute__((always_inline)) {
          if (i < S) s = Matrix<V>::along(a, k[i], s);
          else if (i < S + P) {
            if (i == S) probabilities();
            dv[(i - S) / 2] = Matrix<V>::along(a, operand[i % 2], dv[(i - S) / 2]);
          } else if (i < 2 * S + P) dp = Matrix<V>::along(a, v[i - S - P], dp);
          else {
            if (i == 2 * S + P) scores();
            dk[(i - 2 * S - P) / 2] = Matrix<V>::along(a, operand[i % 2], dk[(i - 2 * S - P) / 2]);
          }
        });
    return;
  }
#pragma unroll
  for (int t = 0; t < T::steps; ++t) s = Matrix<V>::along(T::along(queries, 0, t, lane), k[t], s);
  probabilities();
#pragma unroll
  for (int d = 0; d < DW / 32; ++d) dv[d] = T::across(ders, 0, d, lane, operand, dv[d]);
  start(dp, statD);
#pragma unroll
  for (int t = 0; t < T::steps; ++t) dp = Matrix<V>::along(T::along(ders, 0, t, lane), v[t], dp);
  scores();
#pragma unroll
  for (int d = 0; d < DW / 32; ++d) dk[d] = T::across(queries, 0, d, lane, operand, dk[d]);
}

// NB blocks of 32 keys; they walk over the positions of one head of the group after the other.  NS wavefronts share a block, each takes its 32
// positions of every tile, and their sums are added up through LDS.
template <class V, int DW, int NB, int NS>
__global__ __launch_bounds__(64 * NB * NS, sizeof(V) == 4 ? 1 : 2) void attention_dkv(AttentionP p) {
  typedef Tile<V, DW> T;
  constexpr int NW = NB * NS, RT = 32 * NS;
  constexpr int tileBytes = RT * T::rowBytes, statBytes = RT * 4, bufferBytes = 2 * tileBytes + 2 * statBytes;
  static_assert(RT <= 64, "one load brings the statistics of a tile");
  __shared__ __attribute__((aligned(16))) char lds[kAhead * bufferBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = wave % NB, share0 = wave / NB * 32;
  int id = blockIdx.x;
  const int head = id % p.keyHeads;
  id /= p.keyHeads;
  const int part = id % p.groupParts, firstHead = part * p.headsOfPart, heads = std::min(p.headsOfPart, p.G - firstHead);
  const Span span = find<32 * NB, true>(p, id / p.groupParts, lane);
  if (span.first < 0) return;
  const int off = span.m - span.n;
  const int key = span.first + 32 * block + (lane & 31);
  const bool live = key < span.m;
  // the first position that sees the lane's key, the workgroup's first key (from a tile's border on), the wavefront's first and its last one
  const int firstOf = p.causal ? key - off : 0;
  const int begin = p.causal ? std::max(0, span.first - off) / RT * RT : 0;
  const int some = p.causal ? span.first + 32 * block - off : 0;
  const int all = p.causal ? span.first + 32 * block + 31 - off : 0;

  uintx4 k[T::steps], v[T::steps];
  {
    const char* at = p.k.data + (long long)(span.k0 + (live ? key : 0)) * p.k.position + head * p.k.head;
    const char* vAt = p.v.data + (long long)(span.k0 + (live ? key : 0)) * p.v.position + head * p.v.head;
#pragma unroll
    for (int s = 0; s < T::steps; ++s) k[s] = chunk_of<V>(at, 2 * s + (lane >> 5), p.D, live);
#pragma unroll
    for (int s = 0; s < T::steps; ++s) v[s] = chunk_of<V>(vAt, 2 * s + (lane >> 5), p.D, live);
  }
  const char* queries = p.q.data + (long long)span.q0 * p.q.position + ((long long)head * p.G + firstHead) * p.q.head;
  const char* ders = p.dO.data + (long long)span.q0 * p.dO.position + ((long long)head * p.G + firstHead) * p.dO.head;
  const float* statL = p.statL + ((long long)head * p.G + firstHead) * p.N + span.q0;
  const float* statD = p.statD + ((long long)head * p.G + firstHead) * p.N + span.q0;
  Loader<V, DW, RT, NW> loadQ, loadD;
  loadQ.begin(p.q, p.D, wave, lane);
  loadD.begin(p.dO, p.D, wave, lane);
  // the tile that is brought next: position nextI of the head whose first positions are at headQ, headD, headStat
  const char *headQ = queries, *headD = ders;
  const int each = begin < span.n ? (span.n - begin + RT - 1) / RT : 0, tiles = each * heads, last = begin + (each - 1) * RT;
  const char *nextQ = queries + (long long)last * p.q.position, *nextD = ders + (long long)last * p.dO.position;
  const float* headStat = wave ? statD : statL;   // (of the first two wavefronts)
  int nextI = last;
  const auto bring_tile = [&](char* to) __attribute__((always_inline)) {
    loadQ.bring(to, nextQ, span.n - nextI, wave);
    loadD.bring(to + tileBytes, nextD, span.n - nextI, wave);
    typedef __attribute__((address_space(3))) void* lds_ptr;
    if (wave < 2 && lane < RT) {
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(headStat + nextI), 0, std::min(span.n - nextI, RT) * 4, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(to + 2 * tileBytes + wave * statBytes), 4, lane * 4, 0, 0, 0);
    }
    nextI -= RT;
    nextQ -= (long long)RT * p.q.position;
    nextD -= (long long)RT * p.dO.position;
    if (nextI < begin) {   // the next head
      nextI = last;
      headQ += p.q.head;
      headD += p.dO.head;
      headStat += p.N;
      nextQ = headQ + (long long)last * p.q.position;
      nextD = headD + (long long)last * p.dO.position;
    }
  };
  floatx16 dk[DW / 32], dv[DW / 32];
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
  if (tiles) bring_tile(lds);
  int turn = 0, i0 = last;   // the tile that is due: its buffer, its first position
  for (int t = 0; t < tiles; ++t) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    char* from = lds + turn * bufferBytes;
    char* to = lds + (turn ^ 1) * bufferBytes;
    turn ^= 1;
    const auto bring_next = [&](char* at) __attribute__((always_inline)) {
      if (t + 1 < tiles) bring_tile(at);
    };
    const int i = i0 + share0;
    if (i + 32 > some && i < span.n)
      dkv_tile<V, DW, sizeof(V) == 2 && (DW == 96 || (DW == 64 && NS == 2))>(from + share0 * T::rowBytes, from + tileBytes + share0 * T::rowBytes, (const float*)(from + 2 * tileBytes) + share0,
                      (const float*)(from + 2 * tileBytes + statBytes) + share0, to, bring_next, k, v, dk, dv, i, span.n, firstOf, i < all || i + 32 > span.n, p.c,
                      lane);
    else bring_next(to);
    i0 -= RT;
    if (i0 < begin) i0 = last;
  }
  if (NS == 2) {
    constexpr int values = DW / 32 * 16;
    static_assert(NS == 1 || NB * 2 * values * 256 <= (int)sizeof(lds), "room");
    float* room = (float*)lds + block * 2 * values * 64 + lane;
    __syncthreads();
    if (share0) {
#pragma unroll
      for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          room[(16 * d + r) * 64] = dk[d][r];
          room[(values + 16 * d + r) * 64] = dv[d][r];
        }
    }
    __syncthreads();
    if (share0) return;
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[d][r] += room[(16 * d + r) * 64];
        dv[d][r] += room[(values + 16 * d + r) * 64];
      }
  }
  // Rows that do not see a key have p = ds = 0, which times an infinity or a NaN of theirs is NaN: as in the forward pass, with the queries for dk and the
  // outputs' derivatives for dv.  (Each by itself: neither's bits depend on whether the other is asked for.)
  if (p.causal) {
    const auto to_mend = [&](const floatx16 (&sums)[DW / 32], const char* rows, const Tensor3& t) __attribute__((always_inline)) {
      bool mend = live && !all_finite(sums);
      if (!__any(mend)) return false;
      bool unseen = false, seen = false;
#pragma unroll 1
      for (int h = 0; h < heads; ++h) {
        const int row = bad_row<V, DW, false>(rows + h * t.head, t.position, p.D, std::max(0, some - 31), std::min(span.n, all), lane);
        unseen = unseen || row < firstOf;
      }
      mend = mend && unseen;
#pragma unroll 1
      for (int h = 0; h < heads && __any(mend && !seen); ++h) {
        const int row = bad_row<V, DW, true>(rows + h * t.head, t.position, p.D, std::max(0, some), span.n, lane);
        seen = seen || row >= std::max(0, firstOf);
      }
      return mend && !seen;
    };
    const bool mendK = p.dk.data && to_mend(dk, queries, p.q), mendV = p.dv.data && to_mend(dv, ders, p.dO);
    if (__any(mendK || mendV)) {
#pragma unroll
      for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (mendK) dk[d][r] = 0.f;
          if (mendV) dv[d][r] = 0.f;
        }
      const char* keyRow = p.k.data + (long long)(span.k0 + (live ? key : 0)) * p.k.position + head * p.k.head;
      const char* valueRow = p.v.data + (long long)(span.k0 + (live ? key : 0)) * p.v.position + head * p.v.head;
#pragma unroll 1
      for (int h = 0; h < heads; ++h)
#pragma unroll 1
        for (int i = std::max(0, some); i < span.n; ++i) {
          const char* query = queries + (long long)i * p.q.position + h * p.q.head;
          const char* der = ders + (long long)i * p.dO.position + h * p.dO.head;
          const float negL = statL[(long long)h * p.N + i];
          const float e = probability<V>((starts_at_sum<V>() ? negL : 0.f) + row_product<V, DW>(keyRow, query, p.D, lane), negL, p.c);
          const float f = e * (statD[(long long)h * p.N + i] + row_product<V, DW>(valueRow, der, p.D, lane));
          if (i < firstOf) continue;
          if (mendV) add_row<V, DW>(dv, der, as_operand<V>(e), p.D, lane);
          if (mendK) add_row<V, DW>(dk, query, as_operand<V>(f), p.D, lane);
        }
    }
  }
  if (!live) return;
  if (p.groupParts > 1) {
    char* at = (char*)(p.parts + (((long long)part * p.M + span.k0 + key) * p.keyHeads + head) * 2 * DW);
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int first = 32 * d + 8 * (r / 4) + 4 * (lane >> 5);
        store4<float>(at, first, DW, 1, dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]);
        store4<float>(at + DW * 4, first, DW, 1, dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]);
      }
    return;
  }
#pragma unroll
  for (int d = 0; d < DW / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int at = 32 * d + 8 * (r / 4) + 4 * (lane >> 5);
      if (p.dk.data)
        store4<V>(p.dk.data + (long long)(span.k0 + key) * p.dk.position + head * p.dk.head, at, p.D, p.vector, dk[d][r] * p.scale, dk[d][r + 1] * p.scale,
                  dk[d][r + 2] * p.scale, dk[d][r + 3] * p.scale);
      if (p.dv.data)
        store4<V>(p.dv.data + (long long)(span.k0 + key) * p.dv.position + head * p.dv.head, at, p.D, p.vector, dv[d][r], dv[d][r + 1], dv[d][r + 2],
                  dv[d][r + 3]);
    }
}

// dk and dv of a group whose heads were in several workgroups: the parts added up in their order.  A thread per key, head and four channels.
template <class V, int DW>
__global__ __launch_bounds__(256) void attention_dkv_join(AttentionP p) {
  constexpr int kFours = 2 * DW / 4;
  const long long index = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)p.M * p.keyHeads;
  const long long item = index / kFours;
  if (item >= all) return;
  const int four = (int)(index % kFours), key = (int)(item / p.keyHeads), head = (int)(item % p.keyHeads);
  if (p.kStarts && (key < clamped(p.kStarts[0], p.M) || key >= clamped(p.kStarts[p.sequences], p.M))) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int part = 0; part < p.groupParts; ++part) {
    const float4 v = *(const float4*)(p.parts + (part * all + item) * 2 * DW + 4 * four);
    sum.x += v.x;
    sum.y += v.y;
    sum.z += v.z;
    sum.w += v.w;
  }
  const bool isK = four < kFours / 2;
  const Tensor3& out = isK ? p.dk : p.dv;
  if (!out.data) return;
  const float f = isK ? p.scale : 1.f;
  store4<V>(out.data + key * out.position + head * out.head, 4 * (four % (kFours / 2)), p.D, p.vector, sum.x * f, sum.y * f, sum.z * f, sum.w * f);
}

// ------------------------------------------------------------------------------------------ operands that do not start at 16 bytes

struct PackP {
  const char* from[5];
  char* to[5];
  long long position[5], head[5], items[5];   // (strides in bytes) heads of all positions
  int positions[5];
  int D, chunks;
};

// Heads of any D and strides, each a whole number of 16 bytes, zero behind D: a thread per 16 bytes.  A head's positions lie one behind the other,
// so that a tile's rows are near each other however many heads there are (their offsets and the tile's size are 32-bit numbers).
template <class V>
__global__ __launch_bounds__(256) void attention_pack(PackP p) {
  constexpr int W = 16 / sizeof(V);
  const int which = blockIdx.y;
  const long long all = p.items[which] * p.chunks;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < all; t += (long long)gridDim.x * 256) {
    const long long item = t / p.chunks, head = item / p.positions[which];
    const int chunk = (int)(t % p.chunks), position = (int)(item % p.positions[which]);
    const V* from = (const V*)(p.from[which] + position * p.position[which] + head * p.head[which]) + chunk * W;
    V v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = chunk * W + e < p.D ? from[e] : V(0);
    uintx4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[e] = sizeof(V) == 4 ? __builtin_bit_cast(unsigned, (float)v[e]) : (unsigned)v[2 * e % W] | (unsigned)v[(2 * e + 1) % W] << 16;
    *(uintx4*)(p.to[which] + t * 16) = out;
  }
}

// ------------------------------------------------------------------------------------------ rows that are zero

struct ClearP {
  char* data[4];
  long long position[4], head[4];   // strides in bytes
  const int* starts[4];
  int positions[4], heads[4], width[4], size[4];   // (width: values of a head)
  int n, sequences, inside;
};

// Zeros for the rows before the first sequence's and behind the last one's; inside: for those of the sequences (without starts: all)
__global__ __launch_bounds__(256) void attention_clear(ClearP p) {
  for (int t = 0; t < p.n; ++t) {
    const int first = p.starts[t] ? clamped(p.starts[t][0], p.positions[t]) : 0;
    const int last = p.starts[t] ? std::max(first, clamped(p.starts[t][p.sequences], p.positions[t])) : p.positions[t];
    const long long rows = p.inside ? last - first : first + p.positions[t] - last, each = (long long)p.heads[t] * p.width[t];
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * each; i += (long long)gridDim.x * 256) {
      const long long r = i / each;
      const int within = (int)(i % each), head = within / p.width[t], d = within % p.width[t];
      char* at = p.data[t] + (p.inside ? first + r : r < first ? r : last + r - first) * p.position[t] + head * p.head[t];
      if (p.size[t] == 4) ((unsigned*)at)[d] = 0u;
      else ((unsigned short*)at)[d] = 0;
    }
  }
}

// ---------------------------------------------------------------------------------------------- host

constexpr long long kMostThreads = 1ll << 32;   // of a launch
constexpr size_t kAlign = 256;
size_t rounded(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

int check_geom(const char* who, const mcn_attention_geom* g) {
  if (!g) return fail(MCN_ILLEGAL_ARGUMENT, "%s: null geometry", who);
  if (g->dataType != MCN_FLOAT && g->dataType != MCN_BFLOAT16) return fail(MCN_ILLEGAL_ARGUMENT, "%s: unknown data type %d", who, g->dataType);
  if (g->D < 0 || g->heads < 0 || g->keyHeads < 0 || g->N < 0 || g->M < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative extent", who);
  if (g->D > kMostD) return fail(MCN_UNSUPPORTED, "%s: heads of more than %d channels", who, kMostD);
  if (g->sequences < 0) return fail(MCN_ILLEGAL_ARGUMENT, "%s: negative number of sequences", who);
  if (g->sequences > 1 << 28) return fail(MCN_UNSUPPORTED, "%s: too many sequences", who);
  if (g->heads && (g->keyHeads == 0 || g->heads % g->keyHeads)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: %d heads over %d key heads", who, g->heads, g->keyHeads);
  if (!(g->scale >= 0) || std::isinf(g->scale)) return fail(MCN_ILLEGAL_ARGUMENT, "%s: the scale is negative or no number", who);
  // (log sums are divided by it)
  if (g->scale > 0 && (g->scale < 1e-30 || g->scale > 1e30)) return fail(MCN_UNSUPPORTED, "%s: a scale outside of 1e-30 to 1e30", who);
  // (rows of heads, and 256 positions behind the last one, are counted in 31 bits)
  if (((long long)g->N + 256) * g->heads >= (1ll << 31) || (long long)g->M + 256 >= (1ll << 31)) return fail(MCN_UNSUPPORTED, "%s: too many positions", who);
  return MCN_SUCCESS;
}

struct Operand {
  const mcn_heads* t;
  int positions, heads;
};

// read as they lie: 16 bytes at a time, rows one behind the other, those of a tile within 2^30 bytes
bool lies_well(const Operand& o, int D, int size) {
  const int V = 16 / size;
  return D % V == 0 && aligned16(o.t->data) && o.t->position % V == 0 && o.t->head % V == 0 && o.t->position * size <= (1ll << 30) / 64 &&
         (o.positions <= 1 || o.t->position >= D);
}

size_t packed_bytes(int positions, int heads, int D, int size) { return rounded((size_t)positions * heads * (((size_t)D * size + 15) / 16 * 16)); }

struct Plan {
  int DW, size, G, blocks, slices;
  int dqBlocks, dkvBlocks, groupParts, headsOfPart;   // backward
  size_t partsAt, sumsAt, statAt, packAt, bytes;
};

// Whether two wavefronts share a block of 32 rows or keys.  They make twice as many workgroups of half the length, which bring twice as many
// tiles.  Rows: where the chip is not filled otherwise (causal, bfloat16, calls with four wavefronts alone -> two to a block.  4 sequences of 512, 16
// heads of 128: forward 16.5 -> 16.0 us, dq 24.6 -> 23.1; 2 of 1024, 8 heads of 64: 21.5 -> 20.2, 22.1 -> 17.2; 9 sequences, 6 heads of 75 over 2 in
// single precision: 87 -> 71, 142 -> 104; one of 4096, 4 heads of 128 over one: dq 112 -> 73, but forward, which slices of keys fill the chip for as
// well, 45 -> 50; on the other side 4 of 2048, 16 heads of 128: 89 -> 104, 137 -> 154; 196 positions x 32 x 12 heads of 64: dq 23 -> 30).  Keys,
// whole backward: 4 of 2048 as above 293 -> 327, the one sequence 277 -> 217, 13 packed ones of up to 1100, 32 heads over 8, 331 -> 317, and the 196
// positions, whose last tiles hold more that is not there, 45 -> 53; the rule loses on 32 heads over 8 of 4096, 559 -> 591, and of 4 x 512, 88 -> 96.
bool split(const char* name, bool rule) {
  const int forced = tunable(name, 0);
  return forced ? forced == 2 : rule;
}

// How a forward call is cut.  Rows of a sequence on average up to 32: one wavefront a workgroup, and keys are cut into slices until four of
// those are there for every compute unit; otherwise four wavefronts, and slices until there are two workgroups for each.  A slice has four
// tiles at least, eight where a tile takes the least time: the partial results are written, read and put together by a launch (bfloat16, heads of 128,
// causal, slices of two workgroups a compute unit against one slice: one sequence of 8192 of 2 heads 73 and 112 us, of 2048 of 32 heads over 8
// the same 52, but 2 of 1024 of 8 heads of 64 21 and 15; with four workgroups a compute unit 67 and 75, and 9 sequences of 6 heads of 75 over 2 in single
// precision 90 instead of 72).
Plan plan_of(const mcn_attention_geom* g, int backward) {
  Plan l = {};
  l.size = g->dataType == MCN_BFLOAT16 ? 2 : 4;
  l.DW = g->D <= 64 ? 64 : g->D <= 96 ? 96 : 128;
  l.G = g->keyHeads ? g->heads / g->keyHeads : 1;
  const int sequences = std::max(1, g->sequences);
  const long long rows = (long long)g->N * l.G;
  l.slices = 1;
  if (!backward) {
    l.blocks = rows <= 32ll * sequences ? 1 : split("attention_forward_split", (rows / 128 + sequences) * g->keyHeads < 2ll * device_compute_units()) ? 2 : 4;
    const long long groups = (long long)div_up(rows, 32 * l.blocks) * g->keyHeads, want = (l.blocks == 1 ? 4ll : 2ll) * std::max(1, device_compute_units());
    const int tile = l.size == 2 ? 64 : 32;
    const long long most = std::max<long long>(1, g->M / sequences / ((l.blocks == 1 || l.size == 4 ? 4 : 8) * tile));
    l.slices = (int)std::max<long long>(1, std::min<long long>({64, most, want / std::max<long long>(1, groups)}));
  }
  l.groupParts = 1;
  l.headsOfPart = l.G;
  if (backward) {
    const long long cus = std::max(1, device_compute_units());
    l.dqBlocks = split("attention_dq_split", (rows / 128 + sequences) * g->keyHeads < 2 * cus) ? 2 : 4;
    l.dkvBlocks = split("attention_dkv_split", (g->M / 128 + sequences) * (long long)g->keyHeads < (g->N < 512ll * sequences ? 2 : 4) * cus) ? 2 : 4;
    // The heads of a group in several workgroups, whose sums are put together by one more launch, where there are not four workgroups a compute
    // unit otherwise, two in single precision (whole backward of one sequence of 4096, causal, bfloat16, heads of 128: 4 over one 538 -> 217 us in
    // four parts, 32 over 8 721 -> 590 in two; 13 packed sequences of 32 over 8, whose workgroups are enough, 317 -> 381 in two)
    const long long groups = std::max(1ll, ((long long)g->M / (32 * l.dkvBlocks) + sequences) * g->keyHeads), want = (l.size == 2 ? 4 : 2) * cus;
    const int forced = tunable("attention_group_parts", 0);
    const int parts = forced ? std::min(forced, l.G) : (int)std::max<long long>(1, std::min<long long>(l.G, (want + groups - 1) / groups));
    l.headsOfPart = div_up(l.G, parts);
    l.groupParts = div_up(l.G, l.headsOfPart);
  }
  size_t at = 0;
  if (l.groupParts > 1) {
    l.partsAt = at;
    at += rounded((size_t)l.groupParts * g->M * g->keyHeads * 2 * l.DW * sizeof(float));
  }
  if (l.slices > 1) {
    l.partsAt = at;
    at += rounded((size_t)l.slices * g->N * g->heads * l.DW * sizeof(float));
    l.sumsAt = at;
    at += rounded((size_t)l.slices * g->N * g->heads * sizeof(float));
  }
  if (backward) {
    l.statAt = at;
    at += 2 * rounded((size_t)g->N * g->heads * sizeof(float));
  }
  l.packAt = at;
  at += packed_bytes(g->N, g->heads, g->D, l.size) * (backward ? 3 : 1) + 2 * packed_bytes(g->M, g->keyHeads, g->D, l.size);
  l.bytes = at;
  return l;
}

Tensor3 in_bytes(const mcn_heads* t, int size) {
  Tensor3 r = {};
  if (t && t->data) r = {(char*)t->data, t->position * size, t->head * size};
  return r;
}

bool stores_well(const mcn_heads* t) { return !t || !t->data || (((uintptr_t)t->data & 15) == 0 && t->position % 4 == 0 && t->head % 4 == 0); }

template <class V>
int pack(const char* who, hipStream_t s, const PackP& p, int n) {
  if (!n) return MCN_SUCCESS;
  long long most = 0;
  for (int i = 0; i < n; ++i) most = std::max(most, p.items[i] * p.chunks);
  KernelTimer timer("attention_pack", s);
  hipLaunchKernelGGL(attention_pack<V>, dim3((unsigned)std::min<long long>((most + 255) / 256, 8192), (unsigned)n), dim3(256), 0, s, p);
  return check_launch(who);
}

// The operands of a call where the kernels read them: as they lie, or packed into the workspace
int place(const char* who, hipStream_t s, const mcn_attention_geom* g, const Plan& l, const Operand* operands, Tensor3** to, int n, char* workspace) {
  PackP p = {};
  p.D = g->D;
  p.chunks = (g->D * l.size + 15) / 16;
  size_t at = l.packAt;
  int packs = 0;
  for (int i = 0; i < n; ++i) {
    const Operand& o = operands[i];
    if (lies_well(o, g->D, l.size)) {
      *to[i] = in_bytes(o.t, l.size);
      continue;
    }
    p.from[packs] = (const char*)o.t->data;
    p.to[packs] = workspace + at;
    p.position[packs] = o.t->position * l.size;
    p.head[packs] = o.t->head * l.size;
    p.items[packs] = (long long)o.positions * o.heads;
    p.positions[packs] = o.positions;
    *to[i] = {workspace + at, p.chunks * 16ll, p.chunks * 16ll * o.positions};
    at += packed_bytes(o.positions, o.heads, g->D, l.size);
    ++packs;
  }
  return g->dataType == MCN_BFLOAT16 ? pack<bf16>(who, s, p, packs) : pack<float>(who, s, p, packs);
}

void common(AttentionP* p, const mcn_attention_geom* g, const Plan& l, const int* qStarts, const int* kStarts) {
  p->qStarts = qStarts;
  p->kStarts = kStarts;
  p->sequences = g->sequences;
  p->each = g->sequences ? g->N / g->sequences : 0;
  p->eachKeys = g->sequences ? g->M / g->sequences : 0;
  p->D = g->D; p->G = l.G; p->heads = g->heads; p->keyHeads = g->keyHeads;
  p->N = g->N; p->M = g->M; p->causal = g->causal != 0;
  p->slices = l.slices;
  p->groupParts = l.groupParts;
  p->headsOfPart = l.headsOfPart;
  p->byG = FastDiv(l.G);
  const double scale = g->scale > 0 ? g->scale : 1.0 / std::sqrt((double)g->D);
  p->scale = (float)scale;
  p->c = (float)(scale * 1.4426950408889634);
}

// tiles of all sequences, of `size` rows or keys
long long tiles_of(AttentionP* p, int rowsEach, int size, long long rows) {
  if (p->qStarts) return rows / size + p->sequences;
  const int each = std::max(1, div_up(rowsEach, size));
  p->byTiles = FastDiv(each);
  p->bySequences = FastDiv(p->sequences);
  return (long long)each * p->sequences;
}

template <class V, int DW>
int forward(const char* who, hipStream_t s, AttentionP& p, const Plan& l) {
  constexpr int KT = sizeof(V) == 2 ? 64 : 32;
  const long long rows = (long long)p.N * p.G;
  const long long blocks = tiles_of(&p, p.each * p.G, 32 * l.blocks, rows) * p.keyHeads * p.slices;
  if (blocks * (l.blocks == 1 ? 64 : 256) >= kMostThreads) return fail(MCN_UNSUPPORTED, "%s: too many tiles", who);
  const dim3 grid((unsigned)blocks);
  {
    KernelTimer timer("attention_forward", s);
    if (l.blocks == 1) hipLaunchKernelGGL((attention_forward<V, DW, 1, 1, KT>), grid, dim3(64), 0, s, p);
    else if (l.blocks == 2) hipLaunchKernelGGL((attention_forward<V, DW, 2, 2, 64>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attention_forward<V, DW, 4, 1, KT>), grid, dim3(256), 0, s, p);
  }
  int rc = check_launch(who);
  if (rc || p.slices == 1) return rc;
  KernelTimer timer("attention_join", s);
  hipLaunchKernelGGL((attention_join<V, DW>), dim3((unsigned)div_up((long long)p.N * p.heads, 4)), dim3(256), 0, s, p);
  return check_launch(who);
}

template <class V, int DW>
int backward(const char* who, hipStream_t s, AttentionP& p, const Plan& l) {
  constexpr int KT = sizeof(V) == 2 ? 64 : 32;
  if (p.N) {
    const long long rows = (long long)p.N * p.G;
    const bool two = l.dqBlocks == 2;
    const long long blocks = tiles_of(&p, p.each * p.G, two ? 64 : 128, rows) * p.keyHeads;
    if (blocks * 256 >= kMostThreads) return fail(MCN_UNSUPPORTED, "%s: too many tiles", who);
    KernelTimer timer("attention_dq", s);
    if (two) hipLaunchKernelGGL((attention_dq<V, DW, 2, 2, 64>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attention_dq<V, DW, 4, 1, KT>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    const int rc = check_launch(who);
    if (rc) return rc;
  }
  if (!p.M || (!p.dk.data && !p.dv.data)) return MCN_SUCCESS;
  const bool two = l.dkvBlocks == 2;
  const long long blocks = tiles_of(&p, p.eachKeys, two ? 64 : 128, p.M) * p.keyHeads * p.groupParts;
  if (blocks * 256 >= kMostThreads) return fail(MCN_UNSUPPORTED, "%s: too many tiles", who);
  {
    KernelTimer timer("attention_dkv", s);
    if (two) hipLaunchKernelGGL((attention_dkv<V, DW, 2, 2>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attention_dkv<V, DW, 4, 1>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  }
  int rc = check_launch(who);
  if (rc || p.groupParts == 1) return rc;
  const long long threads = (long long)p.M * p.keyHeads * (2 * DW / 4);
  if (threads >= kMostThreads - 256) return fail(MCN_UNSUPPORTED, "%s: too many keys", who);
  KernelTimer timer("attention_dkv_join", s);
  hipLaunchKernelGGL((attention_dkv_join<V, DW>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, p);
  return check_launch(who);
}

template <class V>
int forward_of(const char* who, hipStream_t s, AttentionP& p, const Plan& l) {
  return l.DW == 64 ? forward<V, 64>(who, s, p, l) : l.DW == 96 ? forward<V, 96>(who, s, p, l) : forward<V, 128>(who, s, p, l);
}
template <class V>
int backward_of(const char* who, hipStream_t s, AttentionP& p, const Plan& l) {
  return l.DW == 64 ? backward<V, 64>(who, s, p, l) : l.DW == 96 ? backward<V, 96>(who, s, p, l) : backward<V, 128>(who, s, p, l);
}

struct Clear {
  ClearP p = {};
  void add(const Tensor3& t, const int* starts, int positions, int heads, int width, int size) {
    if (!t.data) return;
    const int i = p.n++;
    p.data[i] = t.data;
    p.position[i] = t.position;
    p.head[i] = t.head;
    p.starts[i] = starts;
    p.positions[i] = positions;
    p.heads[i] = heads;
    p.width[i] = width;
    p.size[i] = size;
  }
  int run(const char* who, hipStream_t s, const mcn_attention_geom* g, bool inside = false) {
    if (!p.n) return MCN_SUCCESS;
    p.sequences = g->sequences;
    p.inside = inside;
    KernelTimer timer("attention_clear", s);
    hipLaunchKernelGGL(attention_clear, dim3(256), dim3(256), 0, s, p);
    return check_launch(who);
  }
};

int check_starts(const char* who, const mcn_attention_geom* g, const int* qStarts, const int* kStarts) {
  if (!qStarts != !kStarts) return fail(MCN_ILLEGAL_ARGUMENT, "%s: starts of queries or of keys alone", who);
  if (!qStarts && g->sequences && (g->N % g->sequences || g->M % g->sequences))
    return fail(MCN_ILLEGAL_ARGUMENT, "%s: the positions are not %d sequences of one length", who, g->sequences);
  return MCN_SUCCESS;
}

}  // namespace
}  // namespace mcn

using namespace mcn;

extern "C" {

size_t mcn_attention_workspace_bytes(const mcn_attention_geom* g, int backward) {
  if (!g || g->D <= 0 || g->heads <= 0 || g->keyHeads <= 0 || g->heads % g->keyHeads || g->N < 0 || g->M < 0) return 0;   // (refused by the calls)
  return plan_of(g, backward != 0).bytes;
}

int mcn_attention_forward(mcn_stream_t stream, const mcn_attention_geom* g, const mcn_heads* o, float* logSums, const mcn_heads* q, const mcn_heads* k,
                          const mcn_heads* v, const int* queryStarts, const int* keyStarts, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_attention_forward";
  int rc = check_geom(who, g);
  if (!rc) rc = check_starts(who, g, queryStarts, keyStarts);
  if (!rc && g->D == 0 && g->N && g->heads && logSums) rc = fail(MCN_ILLEGAL_ARGUMENT, "%s: log sums of heads of no channels", who);
  if (rc || g->D == 0 || g->N == 0 || g->heads == 0 || (g->sequences == 0 && !(g->clear && queryStarts))) return rc;
  const int size = g->dataType == MCN_BFLOAT16 ? 2 : 4;
  rc = check_heads(who, "queries", q, g->heads, g->N, g->D, size, false);
  if (!rc && g->M) rc = check_heads(who, "keys", k, g->keyHeads, g->M, g->D, size, false);
  if (!rc && g->M) rc = check_heads(who, "values", v, g->keyHeads, g->M, g->D, size, false);
  if (!rc) rc = check_heads(who, "output", o, g->heads, g->N, g->D, size, true);
  const Plan l = plan_of(g, 0);
  if (!rc) rc = check_workspace(who, workspace, workspaceBytes, l.bytes);
  if (rc) return rc;
  AttentionP p = {};
  common(&p, g, l, queryStarts, keyStarts);
  hipStream_t s = as_stream(stream);
  Operand operands[3] = {{q, g->N, g->heads}, {k, g->M, g->keyHeads}, {v, g->M, g->keyHeads}};
  Tensor3* to[3] = {&p.q, &p.k, &p.v};
  rc = place(who, s, g, l, operands, to, g->M ? 3 : 1, (char*)workspace);
  if (rc) return rc;
  p.o = in_bytes(o, size);
  p.vector = g->D % 4 == 0 && stores_well(o);
  p.logSums = logSums;
  if (g->clear && queryStarts) {
    Clear clear;
    clear.add(p.o, queryStarts, g->N, g->heads, g->D, size);
    clear.add({(char*)logSums, 4ll * g->heads, 4}, queryStarts, g->N, g->heads, 1, 4);
    rc = clear.run(who, s, g);
    if (rc) return rc;
  }
  p.parts = (float*)((char*)workspace + l.partsAt);
  p.partSums = (float*)((char*)workspace + l.sumsAt);
  if (g->sequences == 0) return MCN_SUCCESS;
  return g->dataType == MCN_BFLOAT16 ? forward_of<bf16>(who, s, p, l) : forward_of<float>(who, s, p, l);
}

int mcn_attention_backward(mcn_stream_t stream, const mcn_attention_geom* g, const mcn_heads* derQ, const mcn_heads* derK, const mcn_heads* derV,
                           const mcn_heads* o, const float* logSums, const mcn_heads* q, const mcn_heads* k, const mcn_heads* v,
                           const mcn_heads* derOutput, const int* queryStarts, const int* keyStarts, void* workspace, size_t workspaceBytes) {
  const char* who = "mcn_attention_backward";
  int rc = check_geom(who, g);
  if (!rc) rc = check_starts(who, g, queryStarts, keyStarts);
  const bool wantQ = derQ && derQ->data, wantK = derK && derK->data, wantV = derV && derV->data;
  if (rc || g->D == 0 || (g->sequences == 0 && !(g->clear && queryStarts)) || (g->N == 0 && g->M == 0) || (!wantQ && !wantK && !wantV)) return rc;
  const int size = g->dataType == MCN_BFLOAT16 ? 2 : 4;
  if (g->heads == 0) {   // no query sees the keys
    Clear clear;
    const mcn_heads* ders[2] = {wantK ? derK : nullptr, wantV ? derV : nullptr};
    for (int i = 0; i < 2 && g->keyHeads && g->M; ++i) {
      if (!ders[i]) continue;
      rc = check_heads(who, i ? "values' derivative" : "keys' derivative", ders[i], g->keyHeads, g->M, g->D, size, true);
      if (rc) return rc;
      clear.add(in_bytes(ders[i], size), g->clear ? nullptr : keyStarts, g->M, g->keyHeads, g->D, size);
    }
    return clear.run(who, as_stream(stream), g, true);
  }
  if (g->N) {
    rc = check_heads(who, "queries", q, g->heads, g->N, g->D, size, false);
    if (!rc) rc = check_heads(who, "output", o, g->heads, g->N, g->D, size, false);
    if (!rc) rc = check_heads(who, "output's derivative", derOutput, g->heads, g->N, g->D, size, false);
    if (!rc && wantQ) rc = check_heads(who, "queries' derivative", derQ, g->heads, g->N, g->D, size, true);
    if (!rc && !logSums) rc = fail(MCN_ILLEGAL_ARGUMENT, "%s: null log sums", who);
  }
  if (g->M) {
    if (!rc) rc = check_heads(who, "keys", k, g->keyHeads, g->M, g->D, size, false);
    if (!rc) rc = check_heads(who, "values", v, g->keyHeads, g->M, g->D, size, false);
    if (!rc && wantK) rc = check_heads(who, "keys' derivative", derK, g->keyHeads, g->M, g->D, size, true);
    if (!rc && wantV) rc = check_heads(who, "values' derivative", derV, g->keyHeads, g->M, g->D, size, true);
  }
  const Plan l = plan_of(g, 1);
  if (!rc) rc = check_workspace(who, workspace, workspaceBytes, l.bytes);
  if (rc) return rc;
  AttentionP p = {};
  common(&p, g, l, queryStarts, keyStarts);
  hipStream_t s = as_stream(stream);
  Operand operands[5];
  Tensor3* to[5];
  int n = 0;
  const auto add = [&](const mcn_heads* t, int positions, int heads, Tensor3* where) {
    operands[n] = {t, positions, heads};
    to[n++] = where;
  };
  if (g->N) {
    add(q, g->N, g->heads, &p.q);
    add(o, g->N, g->heads, &p.o);
    add(derOutput, g->N, g->heads, &p.dO);
  }
  if (g->M) {
    add(k, g->M, g->keyHeads, &p.k);
    add(v, g->M, g->keyHeads, &p.v);
  }
  rc = place(who, s, g, l, operands, to, n, (char*)workspace);
  if (rc) return rc;
  p.dq = in_bytes(derQ, size);
  p.dk = in_bytes(derK, size);
  p.dv = in_bytes(derV, size);
  if (g->clear && queryStarts) {
    Clear clear;
    if (g->N) clear.add(p.dq, queryStarts, g->N, g->heads, g->D, size);
    if (g->M) clear.add(p.dk, keyStarts, g->M, g->keyHeads, g->D, size);
    if (g->M) clear.add(p.dv, keyStarts, g->M, g->keyHeads, g->D, size);
    rc = clear.run(who, s, g);
    if (rc) return rc;
  }
  p.vector = g->D % 4 == 0 && stores_well(derQ) && stores_well(derK) && stores_well(derV);
  p.logSums = const_cast<float*>(logSums);
  p.parts = (float*)((char*)workspace + l.partsAt);
  p.statL = (float*)((char*)workspace + l.statAt);
  p.statD = p.statL + rounded((size_t)g->N * g->heads * sizeof(float)) / sizeof(float);
  if (g->sequences == 0) return MCN_SUCCESS;
  return g->dataType == MCN_BFLOAT16 ? backward_of<bf16>(who, s, p, l) : backward_of<float>(who, s, p, l);
}

}  // extern "C"
