// gg_w4.hip -- products of a few rows with 4-bit weights, one matrix or one an
// expert:
//
//   y[i][j] = sum_g scales[j][g] * sum_{k in g} x[i][k] * (q[j][k] - zeros[j][g])
//
// With few rows the weights' bytes are what counts: they are read once, into registers, and turned into binary16
// there.  q - zero is an integer of at most 9 bits, which binary16 holds exactly; the matrix instructions
// (v_mfma_f32_16x16x32_f16: 16 rows of x by 16 columns j) sum exact products in float, and a group's scale
// multiplies its sum: no weight is ever rounded.
//
// Both operands go through LDS.  A load is coalesced among 16 neighbouring lanes, which in the instruction's order
// hold 16 rows: straight to registers each would take 64 cache accesses instead of 16, and that bounded the kernel (55
// accesses a load, three quarters of its cycles).  Weights are loaded 64 bytes of each of 16 rows of q at a time into
// registers, four steps ahead, then written to the wave's own LDS and read back in the instruction's order.  x is
// loaded by the workgroup straight into LDS, a chunk of K ahead.
//
// A workgroup of 8 or 16 waves computes 16 columns for each WK of them, of up to R rows: WK waves split K among them, step
// by step, so that a narrow matrix still gives every CU loads to wait for, and their sums are joined in LDS in the
// waves' order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gg_common.h"
#include "grouped_gemm_amd_kernels.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr int kCus = 256;
constexpr int kXcds = 8;  // neighbouring workgroups go to different ones, each with an L2 of its own
constexpr int kStep = 128;  // values of k a wave takes at once: 16 bytes of each of 16 rows of q in 4 lanes

// The 8 weights of a dword (nibble i: k + i) less a zero point, times 2^-9; minus_zero: the zero point times -2^-9.  An
// integer up to 15 as the bits of a binary16 is a subnormal, that many times 2^-24: the nibbles become halves by two
// masks and a byte permutation a pair, and the fused multiply-add that brings them to normal numbers and subtracts the
// zero point is exact.  (Subnormal operands themselves cost the matrix instruction bits: the sums' error
// was 5e-6 instead of 1e-7.)  The sums are multiplied by 2^9 at the end.
constexpr float kWeightUnit = 0.001953125f;  // 2^-9

__device__ __forceinline__ half8v unpack(uint32_t w, half2v minus_zero) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  const half2v up = {(_Float16)32768.0f, (_Float16)32768.0f};
  uint4v r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = __builtin_amdgcn_perm(odd, even, 0x0c040c00u + i * 0x00010001u);  // 0x0c: a byte of zeros
    r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, pair), up, minus_zero));
  }
  return __builtin_bit_cast(half8v, r);
}

// A launch: the call's arguments and what the host divides for the kernel.
struct Launch {
  ggk_w4_args a;
  int stride_groups, stride_rest;  // the groups from one load of a lane's scales to the next, and the rest in values
  uint32_t group_inverse;          // ceil(2^32 / group)
  int blocks;                      // of columns
  int stride_tiles, stride_blocks; // experts: from one item of a workgroup to the next
};

// The rows of one tile: the expert, its first place in the order, how many.
struct RowTile {
  int expert, first, rows;
};

// Places and row tiles of every expert, made once a workgroup: expert e has places [first[e], first[e + 1]) and tiles
// [tile[e], tile[e + 1]); "expert" a.experts has the places that the counts leave.  Counts are clamped to >= 0 and
// their sums to the rows there are.
template <int MOST>
struct Experts {
  int first[MOST + 2];
  int tile[MOST + 2];
  int waves[32];
};

// a + b, at most `limit` (which is at most 2^30, as a and b are).
__device__ __forceinline__ int add_up_to(int a, int b, int limit) { return (int)min((unsigned)a + (unsigned)b, (unsigned)limit); }

// Prefix sum of the values before this thread's, in thread order, and of all; both at most `limit`.
template <int THREADS>
__device__ int block_before(int v, int limit, int* s_waves, int* total) {
  constexpr int kWaves = THREADS / kWave;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x = add_up_to(x, y, limit);
  }
  int before = __shfl_up(x, 1, kWave);
  if (lane == 0) before = 0;
  if (lane == kWave - 1) s_waves[wave] = x;
  __syncthreads();
  int ahead = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) ahead = add_up_to(ahead, s_waves[w], limit);
    all = add_up_to(all, s_waves[w], limit);
  }
  __syncthreads();
  *total = all;
  return add_up_to(before, ahead, limit);
}

template <int THREADS, int ROWS, class Table>
__device__ void list_experts(const ggk_w4_args& a, Table& s) {
  int placed = 0, tiles = 0;
  for (int e0 = 0; e0 < a.experts; e0 += THREADS) {
    const int e = e0 + threadIdx.x;
    const int count = e < a.experts ? min(max(a.counts[e], 0), a.rows) : 0;
    int all, all_tiles;
    const int first = add_up_to(block_before<THREADS>(count, a.rows, s.waves, &all), placed, a.rows);
    const int rows = min(count, a.rows - first);
    const int mine = (rows + ROWS - 1) / ROWS;
    const int tile = block_before<THREADS>(mine, 0x3fffffff, s.waves, &all_tiles) + tiles;
    if (e < a.experts) {
      s.first[e] = first;
      s.tile[e] = tile;
    }
    placed = add_up_to(placed, all, a.rows);
    tiles += all_tiles;
  }
  if (threadIdx.x == 0) {
    s.first[a.experts] = placed;
    s.tile[a.experts] = tiles;
    s.first[a.experts + 1] = a.rows;
    s.tile[a.experts + 1] = tiles + (a.rows - placed + ROWS - 1) / ROWS;
  }
  __syncthreads();
}

template <int ROWS, class Table>
__device__ RowTile expert_tile(const ggk_w4_args& a, const Table& s, int tile) {
  const int lane = threadIdx.x % kWave;
  int before = 0;  // entries of s.tile at or below `tile`: the last of them is the one that holds it
  for (int e0 = 0; e0 <= a.experts; e0 += kWave) {
    before += __popcll(__ballot(e0 + lane <= a.experts && s.tile[min(e0 + lane, a.experts)] <= tile));
  }
  RowTile t;
  t.expert = before - 1;
  t.first = s.first[t.expert] + (tile - s.tile[t.expert]) * ROWS;
  t.rows = min(ROWS, s.first[t.expert + 1] - t.first);
  return t;
}

constexpr int kWaves = 8;       // of a workgroup, two on a CU,
constexpr int kManyWaves = 16;  // or of one on a CU
constexpr int kDepth = 4;  // steps of weights a wave has in flight

// Steps of every wave that a chunk of x holds: four, less where two chunks of R rows would not fit 64 KB (32 KB beside
// the full table of experts), so that a CU holds two workgroups.  A load instruction takes 512 values of one row.
template <int R, int WK, bool EXPERTS>
constexpr int kChunk = R * WK <= (EXPERTS && R < 32 ? 16 : 32) ? 4 : (EXPERTS ? 64 : 128) / (R * WK);

// Experts that the table of a kernel with R-row tiles holds: all, or as many as leave room for two workgroups.
template <int R>
constexpr int kTable = R < 32 ? GGK_MOE_MAX_EXPERTS : 256;

// Length in values of a row of x in LDS: 16 bytes more than its chunk, so that the 16 rows of an instruction's
// operand lie in distinct banks.
template <int R, int WK, bool EXPERTS>
constexpr int kRowLength = kChunk<R, WK, EXPERTS> * WK * kStep + 8;

// Bytes of two chunks of x, or of the waves' sums at the end.
template <int WAVES, int R, int WK, bool EXPERTS>
constexpr int kXBytes = 4 * R * kRowLength<R, WK, EXPERTS> > WAVES * (R < 16 ? 16 : R) * 64
                            ? 4 * R * kRowLength<R, WK, EXPERTS>
                            : WAVES * (R < 16 ? 16 : R) * 64;

// What a workgroup keeps in LDS: pointers to arrays of their own, so that accesses to one may pass those to another.
struct Shared {
  unsigned char* x;
  // A step's weights per wave: 64 bytes a column, the four pieces of 16 in an order that depends on the column
  // (piece), so that neither the write nor the read meets a bank twice.
  unsigned char (*w)[16 * 64];
  uint32_t (*sz)[16][4];  // scales and zero points, per wave and column
  int* slot;              // of the tile's rows, -1 for none
  int* x_row;
};

// Place of piece p (32 values of k) of a column in Shared::w.
__device__ __forceinline__ int piece(int column, int p) { return column * 64 + ((p ^ (column >> 2)) & 3) * 16; }

// One item's sums over the wave's steps of K, of up to R rows, times kWeightUnit.  FINE: groups that are not whole steps,
// each instruction's 32 values lie in one; else a step lies in one group.  Every load of weights is made without a
// condition, past K too (there it reads the row's last values, with a scale of 0): the waits before a load's use
// are counted in the loads made since, and a load that may not have been made does not count.
template <int WAVES, int R, int WK, bool EXPERTS, bool FINE, bool ZEROS>
__device__ __forceinline__ void multiply_item(const Launch& l, const RowTile& t, int column0, const Shared& s,
                                              float4v (&sum)[(R + 15) / 16]) {
  const ggk_w4_args& a = l.a;
  constexpr int M = (R + 15) / 16, kTurns = kChunk<R, WK, EXPERTS>, kLength = kRowLength<R, WK, EXPERTS>;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wk = wave % WK;
  const int column = lane % 16, row = lane / 16;        // of the lane in an instruction's operands; lane row
  const int my_column = lane / 4, my_piece = lane % 4;  // of the lane in a load
  const int steps = (a.k + kStep - 1) / kStep;
  const int turns = (steps + WK - 1) / WK;  // steps of a wave, at most
  const int units = (turns + kDepth - 1) / kDepth;
  // The turns are made in units of kDepth.  In step, the workgroups would all read the same lines of x at the same time,
  // and rows a power of two apart lie in a few channels of the L2: where it costs nothing else, each begins with
  // another unit and goes on around the end (64 rows of 8192 values, groups of 128: 25.2 us in step, 22.9 us so;
  // groups of 64: 26.6 and 27.2, and experts' items begin at their own times as it is).
  constexpr bool kTurned = !EXPERTS && !FINE;
  // The wait for the next step's weights also waits for what was loaded before their last kDepth - 1 loads; ahead of the
  // chunk's loads it waits for fewer of those (64 rows of 8192, groups of 64: 24.1 instead of 25.1 us).  With fewer rows
  // it gains nothing, and experts lose 1%.
  constexpr bool kWriteFirst = WAVES > kWaves;
  int unit = kTurned ? (int)((blockIdx.x / kXcds % (kCus / kXcds)) * units / (kCus / kXcds)) : 0;
  auto after = [&](int u) { return kTurned && u + 1 == units ? 0 : u + 1; };

  // A chunk of x into half `half` of s.x, 512 values of a row an instruction; zeros past K by the resource's range
  // check.  chunk: from the first turn on.
  auto stage = [&](int chunk, int half) {
    constexpr int kLoads = kTurns * WK / 4;  // of a row
    static_assert(kTurns * WK % 4 == 0, "whole instructions a row");
    const int k0 = chunk * kTurns * WK * kStep;
#pragma unroll
    for (int i = 0; i < (R * kLoads + WAVES - 1) / WAVES; ++i) {
      const int at = wave + i * WAVES, r = at / kLoads, k = k0 + at % kLoads * 512;
      const int place = 2 * ((half * R + r) * kLength + at % kLoads * 512);  // in bytes
      if (r < t.rows && k < a.k) {
        const _Float16* x = static_cast<const _Float16*>(a.x) +
                            (EXPERTS ? __builtin_amdgcn_readfirstlane(s.x_row[r]) : t.first + r) * a.ldx + k;
        gg::load_to_lds16(x, 2 * (a.k - k < 512 ? a.k - k : 512), gg::lds_address(s.x) + place, 16 * lane, 0);
      } else if (r < t.rows) {  // a chunk that K does not reach the end of
        *reinterpret_cast<uint4v*>(s.x + place + 16 * lane) = uint4v{0, 0, 0, 0};
      }
    }
  };
  constexpr int kChunks = kDepth / kTurns;  // of a unit
  stage(unit * kChunks, 0);

  const long long j = min(column0 + my_column, a.n - 1);
  const unsigned char* q = a.q + t.expert * a.stride_q + j * a.ldq;
  const _Float16* scales = static_cast<const _Float16*>(a.scales) + t.expert * a.stride_s + j * a.lds;
  const unsigned char* zeros = ZEROS ? a.zeros + t.expert * a.stride_z + j * a.ldz : nullptr;
  // Scale (low half) and zero point of the group that holds the lane's k, which goes from load to load in equal
  // strides: the group goes on by the whole groups of a stride, and one more where the rest has come to one.
  constexpr int kStride = (FINE ? 1 : kDepth) * WK * kStep;
  const int first_k = FINE ? wk * kStep + 32 * my_piece : (my_piece * WK + wk) * kStep;  // below 2^12: the product is exact
  const int first_group = (int)__umulhi((uint32_t)first_k, l.group_inverse);
  int scale_k = first_k, group = first_group, rest = first_k - first_group * a.group;
  if (kTurned && unit > 0) {
    scale_k += unit * kStride;
    group = scale_k / a.group;
    rest = scale_k - group * a.group;
  }
  const int last_group = a.k / a.group - 1;
  auto from_start = [&]() {
    scale_k = first_k;
    group = first_group;
    rest = first_k - first_group * a.group;
  };
  auto next_scale = [&]() {
    const int g = min(group, last_group);
    uint32_t v = *reinterpret_cast<const uint16_t*>(scales + g);
    if constexpr (ZEROS) v |= (uint32_t)zeros[g] << 16;
    v = scale_k < a.k ? v : 0;
    scale_k += kStride;
    group += l.stride_groups;
    rest += l.stride_rest;
    if (rest >= a.group) {
      rest -= a.group;
      ++group;
    }
    return v;
  };
  uint4v w[kDepth];
  uint32_t sz[FINE ? kDepth : 1];  // FINE: of the lane's 32 values of each step; else: of the lane's step of the next four
  auto load = [&](int turn, int d) {
    const int k = min((turn * WK + wk) * kStep + 32 * my_piece, a.k - 32);
    w[d] = *reinterpret_cast<const uint4v*>(q + k / 2);
    if constexpr (FINE) sz[d] = next_scale();
  };
  auto write = [&](int d) {
    *reinterpret_cast<uint4v*>(&s.w[wave][piece(my_column, my_piece)]) = w[d];
    if constexpr (FINE) s.sz[wave][my_column][my_piece] = sz[d];
  };
  // The next step's weights go through LDS while a step is multiplied: a wave's LDS operations keep their order, so
  // that what is written after a read does not change it.
  auto read = [&](uint4v& v, uint4v& g) {
    if constexpr (FINE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint32_t*>(&s.w[wave][piece(column, i) + 4 * row]);
      g = *reinterpret_cast<const uint4v*>(s.sz[wave][column]);
    } else {
      v = *reinterpret_cast<const uint4v*>(&s.w[wave][piece(column, row)]);
    }
  };
  if constexpr (!FINE) sz[0] = next_scale();
#pragma unroll
  for (int d = 0; d < kDepth; ++d) load(unit * kDepth + d, d);
#pragma unroll
  for (int m = 0; m < M; ++m) sum[m] = float4v{};
  const unsigned char* x[M];  // the lane's rows in LDS
#pragma unroll
  for (int m = 0; m < M; ++m) {
    x[m] = s.x + 2 * (min(16 * m + column, R - 1) * kLength + wk * kStep + (FINE ? 8 : 32) * row);
  }
  uint4v v, g, four;
  int next = units > 1 ? after(unit) : units;  // units: past the end, where loads repeat the last values
  if (kTurned && next == 0) from_start();
  write(0);
  load(next * kDepth, 0);
  read(v, g);
  for (int done = 0; done < units; ++done) {
    const int second = done + 2 < units ? after(next) : units;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (units == 1 && d >= turns) break;
      if constexpr (kWriteFirst) write((d + 1) % kDepth);
      const int half = kTurns == kDepth ? done % 2 : d / kTurns % 2;
      if (d % kTurns == 0) {
        // This chunk's loads are older than the weights' of the last kTurns steps; behind the barrier every wave's have
        // landed, and every wave is done with the chunk before, whose place the next one takes.
        asm volatile("" ::: "memory");
        gg::wait_vmcnt<kTurns>();
        gg::stage_barrier();
        if (d / kTurns + 1 < kChunks) {
          stage(unit * kChunks + d / kTurns + 1, 1 - half);
        } else if (done + 1 < units) {
          stage(next * kChunks, 1 - half);
        }
        if constexpr (FINE) asm volatile("" ::: "memory");
      }
      if constexpr (!FINE) {
        if (d == 0) {
          s.sz[wave][my_column][my_piece] = sz[0];
          four = *reinterpret_cast<const uint4v*>(s.sz[wave][column]);
          sz[0] = next_scale();
          if (kTurned && second == 0) from_start();
        }
      }
      uint4v next_v, next_g;
      if constexpr (!kWriteFirst) write((d + 1) % kDepth);
      load(d + 1 < kDepth ? next * kDepth + d + 1 : second * kDepth, (d + 1) % kDepth);
      read(next_v, next_g);
      if constexpr (!FINE) g = uint4v{four[d], four[d], four[d], four[d]};
      half8v b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        half2v minus_zero = {(_Float16)(-8.0f * kWeightUnit), (_Float16)(-8.0f * kWeightUnit)};
        if constexpr (ZEROS) {  // the zero point's bits are that many times 2^-24
          const half2v down = {(_Float16)-32768.0f, (_Float16)-32768.0f};
          minus_zero = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(g[i], g[i], 0x03020302u)) * down;
        }
        b[i] = unpack(v[i], minus_zero);
      }
      const int at = 2 * (half * R * kLength + d % kTurns * WK * kStep);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float4v part = float4v{};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const half8v xs = *reinterpret_cast<const half8v*>(x[m] + at + (FINE ? 64 : 16) * i);
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs, b[i], part, 0, 0, 0);
          if (FINE || i == 3) {
            const float scale = (float)__builtin_bit_cast(_Float16, (uint16_t)g[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[m][e] = fmaf(scale, part[e], sum[m][e]);
            part = float4v{};
          }
        }
      }
      v = next_v;
      g = next_g;
    }
    unit = next;
    next = second;
  }
}

__device__ __forceinline__ void store_y(const ggk_w4_args& a, int slot, int j, float y) {
  const long long at = slot * a.ldy + j;
  if (a.y_type == GGK_TYPE_F16) {
    static_cast<_Float16*>(a.y)[at] = (_Float16)y;
  } else {
    static_cast<float*>(a.y)[at] = y;
  }
}

// One tile of rows by the workgroup's columns from block0 on: sums, their join over the waves that split K, y.
template <int WAVES, int R, int WK, bool EXPERTS, bool FINE, bool ZEROS>
__device__ __forceinline__ void run_item(const Launch& l, const RowTile& t, int block0, const Shared& s) {
  const ggk_w4_args& a = l.a;
  constexpr int M = (R + 15) / 16, kColumns = 16 * (WAVES / WK);
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int column = lane % 16, row = lane / 16, wn = wave / WK, wk = wave % WK;
  float4v sum[M];
  multiply_item<WAVES, R, WK, EXPERTS, FINE, ZEROS>(l, t, block0 + wn * 16, s, sum);
  float* s_sum = reinterpret_cast<float*>(s.x);  // [WK][16 M][kColumns]
  gg::stage_barrier();
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s_sum[(wk * 16 * M + 16 * m + 4 * row + i) * kColumns + 16 * wn + column] = sum[m][i];
  }
  gg::stage_barrier();
  for (int i = tid; i < t.rows * kColumns; i += WAVES * kWave) {
    const int r = i / kColumns, c = i % kColumns, j = block0 + c, slot = EXPERTS ? s.slot[r] : t.first + r;
    if (j < a.n && slot >= 0) {
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w) y += s_sum[(w * 16 * M + r) * kColumns + c];
      y *= 1.0f / kWeightUnit;
      if (a.row_weights != nullptr) y *= a.row_weights[slot];
      store_y(a, slot, j, y);
    }
  }
}

// R: rows of an item, at most.  Measured, in calls one behind the other (a dispatch in a trace takes up to 3 us more): one row of 4096 by 14336 columns, 30 MB, 8.8 us, of which the workgroups'
// start is 3.2 and the rest runs at the cache's rate; 64 experts' matrices of that size, 256 slots on 46 of them, 1.4 GB, 312 to
// 343 us from card to card (4.1 to 4.5 TB/s, where a sum over 4 GB reads 4.0).  64 rows of 8192 by 8192 with groups of 64
// take 24 us, of which 13 are the issue of vector instructions alone: 7.9 M, 120 a wave and step, of them 44 to unpack, some
// 36 for a scale every 32 values, the rest addresses and fetches of scales; each weight is unpacked for both row tiles.  By
// 8 waves it took 27, and 22 without the loads of x, 25 without unpacking, 26 without reading x from LDS.
// Groups that are not whole steps cost the experts' rows the same: 64 experts of that size, all with slots, with zero points
// 423 us in groups of 128, 652 of 64, 739 of 32 (555 of 64 without zero points).  The registers are at their bound there:
// experts' items of 32 rows in such groups spill 12 of them (4 without zero points), and of 16 rows with one wave along K
// and zero points 7, none of it inside the loops over K.
template <int WAVES, int R, int WK, bool EXPERTS, bool FINE, bool ZEROS>
__global__ __launch_bounds__(WAVES * kWave, 4) void w4_kernel(Launch l) {
  const ggk_w4_args& a = l.a;
  constexpr int kColumns = 16 * (WAVES / WK);
  __shared__ alignas(16) unsigned char s_x[kXBytes<WAVES, R, WK, EXPERTS>];
  __shared__ alignas(16) unsigned char s_w[WAVES][16 * 64];
  __shared__ alignas(16) uint32_t s_sz[WAVES][16][4];
  const int tid = threadIdx.x;
  if constexpr (!EXPERTS) {
    const Shared s{s_x, s_w, s_sz, nullptr, nullptr};
    const int tiles = (a.rows + R - 1) / R;
    for (int tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
      const RowTile t{0, tile * R, min(R, a.rows - tile * R)};
      run_item<WAVES, R, WK, false, FINE, ZEROS>(l, t, blockIdx.x * kColumns, s);
      gg::stage_barrier();
    }
  } else {
    __shared__ int s_slot[R], s_x_row[R];
    __shared__ Experts<kTable<R>> s_experts;
    const Shared s{s_x, s_w, s_sz, s_slot, s_x_row};
    const int fan = a.rows / a.x_rows;
    list_experts<WAVES * kWave, R>(a, s_experts);
    const int tiles = s_experts.tile[a.experts + 1];
    int tile = blockIdx.x / l.blocks, block = blockIdx.x % l.blocks;
    while (tile < tiles) {
      const RowTile t = expert_tile<R>(a, s_experts, tile);
      for (int i = tid; i < t.rows; i += WAVES * kWave) {
        int slot = a.order[t.first + i];
        if (slot >= a.rows) slot = -1;
        s.slot[i] = slot;
        s.x_row[i] = max(slot, 0) / fan;  // where a slot names no row, row 0: its sums are not used
      }
      gg::stage_barrier();
      if (t.expert == a.experts) {
        for (int i = tid; i < t.rows * kColumns; i += WAVES * kWave) {
          const int slot = s.slot[i / kColumns], j = block * kColumns + i % kColumns;
          if (j < a.n && slot >= 0) store_y(a, slot, j, 0.0f);
        }
      } else if (R > 4 && t.rows <= 4) {
        // The rows are a constant of the whole loop over K: the compiler leaves out the wait between a matrix
        // instruction and the use of its result when a branch on them lies between.
        run_item<WAVES, 4, WK, true, FINE, ZEROS>(l, t, block * kColumns, s);
      } else if (R > 16 && t.rows <= 16) {
        run_item<WAVES, 16, WK, true, FINE, ZEROS>(l, t, block * kColumns, s);
      } else {
        run_item<WAVES, R, WK, true, FINE, ZEROS>(l, t, block * kColumns, s);
      }
      gg::stage_barrier();
      tile += l.stride_tiles;
      block += l.stride_blocks;
      if (block >= l.blocks) {
        block -= l.blocks;
        ++tile;
      }
    }
  }
}

template <int R, int WK, bool EXPERTS, int WAVES = kWaves>
hipError_t launch(const ggk_w4_args& a, hipStream_t stream) {
  if (EXPERTS && a.experts > kTable<R>) return hipErrorInvalidValue;
  const bool fine = a.group % kStep != 0;
  auto with_zeros = fine ? w4_kernel<WAVES, R, WK, EXPERTS, true, true> : w4_kernel<WAVES, R, WK, EXPERTS, false, true>;
  auto without = fine ? w4_kernel<WAVES, R, WK, EXPERTS, true, false> : w4_kernel<WAVES, R, WK, EXPERTS, false, false>;
  auto kernel = a.zeros != nullptr ? with_zeros : without;
  constexpr int kColumns = 16 * (WAVES / WK);
  const int stride = (fine ? 1 : kDepth) * WK * kStep;
  Launch l{};
  l.a = a;
  l.stride_groups = stride / a.group;
  l.stride_rest = stride % a.group;
  l.group_inverse = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  l.blocks = (a.n + kColumns - 1) / kColumns;
  const long long tiles = (a.rows + R - 1) / R + (EXPERTS ? min(a.rows, a.experts + 1) : 0);
  dim3 grid(l.blocks, (unsigned)(tiles < 65535 ? tiles : 65535));
  if (EXPERTS) {
    const long long items = tiles * l.blocks;
    grid = dim3((unsigned)(items < kCus * 2 ? items : kCus * 2));
    l.stride_tiles = (int)grid.x / l.blocks;
    l.stride_blocks = (int)grid.x % l.blocks;
  }
  hipLaunchKernelGGL(kernel, grid, dim3(WAVES * kWave), 0, stream, l);
  return hipGetLastError();
}

}  // namespace

extern "C" hipError_t ggk_w4_check(const ggk_w4_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_w4_args& a = *args;
  if (a.rows < 0 || a.rows > GGK_ROUTE_MAX_TOTAL_SLOTS || a.x_rows < 0 || a.n < 0 || a.n > GGK_W4_MAX_EXTENT ||
      a.k < 1 || a.k > GGK_W4_MAX_EXTENT || a.experts < 0 || a.experts > GGK_MOE_MAX_EXPERTS ||
      a.group < 32 || a.group % 32 != 0 || a.k % a.group != 0 || (a.y_type != GGK_TYPE_F32 && a.y_type != GGK_TYPE_F16)) {
    return hipErrorInvalidValue;
  }
  if (a.experts == 0 ? a.rows != a.x_rows : (a.rows > 0 && (a.x_rows < 1 || a.rows % a.x_rows != 0))) {
    return hipErrorInvalidValue;
  }
  if ((a.x_rows > 1 && a.ldx < a.k) || (a.rows > 1 && a.ldy < a.n) ||
      (a.n > 1 && (a.ldq < a.k / 2 || a.lds < a.k / a.group || (a.zeros != nullptr && a.ldz < a.k / a.group))) ||
      a.stride_q < 0 || a.stride_s < 0 || a.stride_z < 0) {
    return hipErrorInvalidValue;
  }
  if (reinterpret_cast<uintptr_t>(a.q) % 16 != 0 || (a.n > 1 && a.ldq % 16 != 0) ||
      (a.experts > 1 && a.stride_q % 16 != 0)) {
    return hipErrorInvalidValue;
  }
  if (a.rows > 0 && a.n > 0) {
    if (a.y == nullptr || a.x == nullptr || a.q == nullptr || a.scales == nullptr) {
      return hipErrorInvalidDevicePointer;
    }
    if (a.experts > 0 && (a.counts == nullptr || a.order == nullptr)) return hipErrorInvalidDevicePointer;
  }
  return hipSuccess;
}

extern "C" hipError_t ggk_w4_multiply(const ggk_w4_args* args, hipStream_t stream) {
  const hipError_t st = ggk_w4_check(args);
  if (st != hipSuccess || args->rows == 0 || args->n == 0) return st;
  const ggk_w4_args& a = *args;
  const long long columns = (a.n + 15) / 16;
  if (a.experts > 0) {
    // Waves that split K, where there are few without.  us of the forms (rows, waves along K) (32, 1), (16, 1), (16, 2) and
    // (16, 4), groups of 128, two slots a token: 64 experts of 4096 by 14336, 128 tokens 410, 398, 430, 503; 8 tokens 94, 91,
    // 98, 109; one 15.7, 15.8, 15.9, 17.9; of 14336 by 4096, 8 tokens 95, 93, 88, 93, one 39, 39, 23, 15; 16 experts of 1024 by
    // 2048, 512 slots 13.6, 14.4, 16.9, 21.5, by 512 9.5, 7.8, 8.1, 8.4; 8 experts of 4096 by 2048, one token 14.0, 14.1, 9.0,
    // 6.7, by 8192 14.8, 14.8, 10.0, 9.6; 300 experts of 1024 by 1024, 1024 slots -, 42, 47, 70.  The rule is right for many
    // slots; it does not look at K, which costs one token up to 1.5 times the best form.
    const long long waves = columns * min(a.rows, a.experts);
    if (waves >= 1024 && a.experts <= kTable<32>) return launch<32, 1, true>(a, stream);
    if (waves >= 512) return waves >= 1024 ? launch<16, 1, true>(a, stream) : launch<16, 2, true>(a, stream);
    return launch<16, 4, true>(a, stream);
  }
  // The form by what the busiest CU gets: its workgroups, each with its columns and a fixed cost as of `fixed` columns.
  const long long tiles = a.rows > 16 ? (a.rows + 31) / 32 : 1;
  const int fixed = a.rows > 16 ? 32 : 8;
  auto cost = [&](int width) {
    const long long workgroups = (a.n + width - 1) / width * tiles;
    return (workgroups + kCus - 1) / kCus * (width + fixed);
  };
  if (a.rows > 16) {
    // us of the three, narrow to wide: 40 rows of 2048 by 2048 6.2, 7.4, 10.2; 64 of 8192 by 8192 28, 24, 38; 64 of 4096
    // by 14336 26, 24, 18; 90 of 4096 by 8192 21, 23, 18.
    const long long narrow = cost(32), wide = cost(64), widest = cost(128);
    if (widest <= wide && widest <= narrow) return launch<32, 2, false, kManyWaves>(a, stream);
    return wide <= narrow ? launch<32, 4, false, kManyWaves>(a, stream) : launch<32, 4, false>(a, stream);
  }
  // us: one row of 4096 by 8192 in workgroups of 32 and 64 columns 6.8, 8.8, by 14336 10.0, 9.4, by 20480 13.1, 13.4;
  // 13 rows of 4096 by 6400 in 16, 32 and 64 8.7, 7.7, 9.9, by 10240 12.3, 10.6, 10.0, by 28672 23.7, 19.4, 15.9.
  const bool few = a.rows <= 4;
  const long long narrow = cost(16), wide = cost(32), widest = cost(64);
  if (widest <= wide && widest <= narrow) return few ? launch<4, 2, false>(a, stream) : launch<16, 2, false>(a, stream);
  if (wide <= narrow) return few ? launch<4, 4, false>(a, stream) : launch<16, 4, false>(a, stream);
  return few ? launch<4, 8, false>(a, stream) : launch<16, 8, false>(a, stream);
}
