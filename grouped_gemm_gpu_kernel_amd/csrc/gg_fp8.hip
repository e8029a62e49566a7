// gg_fp8.hip -- products of few rows with matrices of 8-bit numbers, one matrix
// or one an expert, plain or gated:
//
//   p[i][j] = sum over blocks b of x_scales[i][b] w_scales[j / 128][b] * sum over k in b of x[i][k] w[j][k]
//
// With few rows the weights' bytes are what counts.  Every wave streams its own columns through a ring of steps of its
// own in LDS, loaded there directly, several steps ahead, with x's rows and the scales of the same step beside them: no
// wave waits for another until its sums are whole.  1 row of 4096 by 14336 takes 11.2 us where the 59 MB of weights are still in the
// cache behind the L2s and 12.7 where they are not (4.6 TB/s with the launch); 61 rows in float 17.2 and 19.7; 1 row gated 24.8 and
// 25.0, by two launches (below).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>
#include <cstdio>

#include "gg_experts.h"
#include "gg_fp8.h"
#include "gg_phased.h"  // wait_lgkmcnt

namespace {

using namespace gg::fp8;
using gg::Experts;
using gg::RowTile;
using gg::kWave;

constexpr int kCus = 256, kXcds = 8;

struct Launch {
  ggk_fp8_args a, second;  // a second product, of the same rows, after the first one's column blocks (no gate)
  int blocks;              // of columns
  int blocks_of_a;         // of those, the first product's
  int tiles;               // of rows (one matrix)
};

// R rows of x (8, 16, 32, 64) by WN waves of NT tiles of 16 columns (with a gate: half of them gate, half up), WK waves
// along K, DEPTH steps in a wave's ring.
template <int R_, int NT_, int WN_, int WK_, int DEPTH_, bool GATED_, bool EXACT_>
struct Form {
  static constexpr int R = R_, NT = NT_, WN = WN_, WK = WK_, DEPTH = DEPTH_;
  static constexpr bool GATED = GATED_, EXACT = EXACT_;
  static constexpr int MT = (R + 15) / 16, WAVES = WN * WK, THREADS = WAVES * kWave;
  static constexpr int WL = 2 * NT, XL = R / 8, SL = R == 64 ? 2 : 1;  // load instructions of a step
  static constexpr int LOADS = WL + XL + SL;
  static constexpr int X = 1024 * WL, S = X + 1024 * XL, STEP = S + 256 * SL;  // offsets in a step, and its bytes
  static constexpr int WS = R == 64 ? 64 : 32;                                 // place of the weights' scales among the step's
  static constexpr int COLUMNS = WN * 16 * NT / (GATED ? 2 : 1);               // of y a workgroup computes
  static constexpr int SUM_LD = WN * 16 * NT + 4;
  static constexpr int RING = WAVES * DEPTH * STEP, SUMS = 4 * WK * MT * 16 * SUM_LD;
  static constexpr int BYTES = RING > SUMS ? RING : SUMS;
  static_assert(DEPTH >= 2 && LOADS * DEPTH < 64, "outstanding loads are counted in 6 bits");
  static_assert(!GATED || COLUMNS == 128, "a block of an 8-bit row");
};

// A step's products of 16 rows of x, times their scales.
template <class F, class Operand>
__device__ __forceinline__ void add_step(const Operand (&w)[F::NT], const Operand& x, float x_scale, float w_scale, float u_scale,
                                         float4v (&sum)[F::NT]) {
  const float scale = x_scale * w_scale, scale_u = x_scale * u_scale;
#pragma unroll
  for (int n = 0; n < F::NT; ++n) {
    const float4v part = multiply(w[n], x);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[n][e] = fmaf(F::GATED && n >= F::NT / 2 ? scale_u : scale, part[e], sum[n][e]);
  }
}

// The wave's sums over its steps of K of one tile of rows by its columns.
template <class F>
__device__ __forceinline__ void multiply_item(const ggk_fp8_args& a, const RowTile& t, const int* x_row, int column0, int turn,
                                              unsigned char* ring, float4v (&sum)[F::MT][F::NT]) {
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wk = wave % F::WK;
  const int steps = (a.k + kStep - 1) / kStep, mine = (steps - wk + F::WK - 1) / F::WK;
  const uint32_t ring_at = gg::lds_address(ring);
  constexpr int kTilesOfW = F::GATED ? F::NT / 2 : F::NT;

  // The lane's part of a load of 8 rows: row lane / 8, piece by the row's swizzle, which the instruction's parity flips.
  const int part = lane / 8, piece = (lane & 7) ^ (lane >> 4);
  uint32_t w_off[F::WL];
  const int base_column = min(column0, a.n - 1);
#pragma unroll
  for (int q = 0; q < F::WL; ++q) {
    const int tile = q / 2 % kTilesOfW, column = min(column0 + 16 * tile + 8 * (q & 1) + part, a.n - 1);
    const long long ld = F::GATED && q / 2 >= kTilesOfW ? a.ldu : a.ldw;
    w_off[q] = (uint32_t)((column - base_column) * ld) + 16 * (piece ^ (4 * (q & 1)));
  }
  const unsigned char* w0 = a.w + t.expert * a.stride_w + base_column * a.ldw;
  const unsigned char* u0 = F::GATED ? a.up + t.expert * a.stride_u + base_column * a.ldu : nullptr;
  const unsigned char* xp[F::XL];
#pragma unroll
  for (int q = 0; q < F::XL; ++q) {
    const int r = min(8 * q + part, t.rows - 1);
    xp[q] = a.x + (x_row != nullptr ? x_row[r] : t.first + r) * a.ldx + 16 * (piece ^ (4 * (q & 1)));
  }
  const int scale_row = min(F::R == 64 ? lane : lane % 32, t.rows - 1);
  const float* xs = a.x_scales + (x_row != nullptr ? x_row[scale_row] : t.first + scale_row) * a.ldxs;
  const float* ws = a.w_scales + t.expert * a.stride_ws + base_column / kStep * a.ldws;
  if (F::GATED && lane % 32 == 1) ws = a.up_scales + t.expert * a.stride_us + base_column / kStep * a.ldus;
  if (F::SL == 1 && lane >= 32) xs = ws;

  // In step, the waves would all read the same columns at a time, and rows a power of two apart lie in a few channels of
  // the L2: every wave begins with another of its steps and goes on around the end, and so do neighbouring workgroups of an XCD
  // and XCDs.
  const int first = (turn + wave / F::WK * max(mine / F::WN, 1)) % max(mine, 1);
  auto issue = [&](int i) {  // the wave's step i into its place of the ring
    const int turned = i + first < mine ? i + first : i + first - mine, step = turned * F::WK + wk, k0 = step * kStep;
    const uint32_t at = ring_at + (i % F::DEPTH) * F::STEP;
    const bool whole = k0 + kStep <= a.k;
#pragma unroll
    for (int q = 0; q < F::WL; ++q) {
      const bool in = whole || k0 + 16 * (piece ^ (4 * (q & 1))) < a.k;
      gg::load_to_lds16((F::GATED && q / 2 >= kTilesOfW ? u0 : w0) + k0, kOutOfRange, at + 1024 * q, in ? w_off[q] : kOutOfRange, 0);
    }
#pragma unroll
    for (int q = 0; q < F::XL; ++q) {
      const bool in = whole || k0 + 16 * (piece ^ (4 * (q & 1))) < a.k;
      load_to_lds16_at(in ? (const void*)(xp[q] + k0) : (const void*)&kZeros, at + F::X + 1024 * q);
    }
    load_to_lds4_at(xs + step, at + F::S);
    if constexpr (F::SL == 2) load_to_lds4_at(ws + step, at + F::S + 256);
  };

#pragma unroll
  for (int m = 0; m < F::MT; ++m) {
#pragma unroll
    for (int n = 0; n < F::NT; ++n) sum[m][n] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll
  for (int i = 0; i < F::DEPTH; ++i) {
    if (i < mine) issue(i);
  }
  const int j = lane % 16, g = lane / 16, x_j = F::R < 16 ? j % 8 : j;
  const uint32_t w_at = j * 128 + ((g ^ (j >> 1)) & 7) * 16, x_at = x_j * 128 + ((g ^ (x_j >> 1)) & 7) * 16;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    // Step i has landed when at most the loads of the DEPTH - 1 steps after it are on their way.
    if (i + F::DEPTH <= mine) {
      gg::wait_vmcnt<F::LOADS * (F::DEPTH - 1)>();
    } else {
      gg::wait_vmcnt<0>();
    }
    asm volatile("" ::: "memory");
    const uint32_t at = ring_at + (i % F::DEPTH) * F::STEP;
    int8v w[F::NT], x[F::MT];
    float x_scale[F::MT];
#pragma unroll
    for (int n = 0; n < F::NT; ++n) w[n] = read_fragment(at + w_at, at + (w_at ^ 64), 2048 * n);
#pragma unroll
    for (int m = 0; m < F::MT; ++m) {
      x[m] = read_fragment(at + x_at, at + (x_at ^ 64), F::X + 2048 * m);
      x_scale[m] = *(const GG_LDS float*)(uintptr_t)(at + F::S + 4 * (16 * m + x_j));
    }
    const float w_scale = *(const GG_LDS float*)(uintptr_t)(at + F::S + 4 * F::WS);
    const float u_scale = F::GATED ? *(const GG_LDS float*)(uintptr_t)(at + F::S + 4 * F::WS + 4) : 0.0f;
    // All of the step is in registers: its place takes another.
    asm volatile("" ::: "memory");
    gg::wait_lgkmcnt<0>();
    if (i + F::DEPTH < mine) issue(i + F::DEPTH);
    if constexpr (F::EXACT) {
      Halves h[F::NT];
#pragma unroll
      for (int n = 0; n < F::NT; ++n) h[n] = to_halves(w[n]);
#pragma unroll
      for (int m = 0; m < F::MT; ++m) add_step<F>(h, to_halves(x[m]), x_scale[m], w_scale, u_scale, sum[m]);
    } else {
#pragma unroll
      for (int m = 0; m < F::MT; ++m) add_step<F>(w, x[m], x_scale[m], w_scale, u_scale, sum[m]);
    }
  }
}

// One tile of rows by the workgroup's columns from block0 on: sums, their join over the waves along K, y.
template <class F, bool EXPERTS>
__device__ __forceinline__ void run_item(const ggk_fp8_args& a, const RowTile& t, const int* slots, const int* x_row,
                                         int block, unsigned char* s_bytes) {
  const int block0 = block * F::COLUMNS;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int j = lane % 16, g = lane / 16, wn = wave / F::WK, wk = wave % F::WK;
  float4v sum[F::MT][F::NT];
  multiply_item<F>(a, t, x_row, block0 + wn * (F::COLUMNS / F::WN), block + (int)(blockIdx.x % kXcds), s_bytes + wave * F::DEPTH * F::STEP, sum);
  float* s_sum = reinterpret_cast<float*>(s_bytes);  // [WK][16 MT][SUM_LD]
  gg::stage_barrier();
#pragma unroll
  for (int m = 0; m < F::MT; ++m) {
#pragma unroll
    for (int n = 0; n < F::NT; ++n) {
      *reinterpret_cast<float4v*>(&s_sum[(wk * 16 * F::MT + 16 * m + j) * F::SUM_LD + (wn * F::NT + n) * 16 + 4 * g]) = sum[m][n];
    }
  }
  gg::stage_barrier();
  auto total = [&](int r, int c) {
    float4v v = *reinterpret_cast<const float4v*>(&s_sum[r * F::SUM_LD + c]);
#pragma unroll
    for (int w = 1; w < F::WK; ++w) v += *reinterpret_cast<const float4v*>(&s_sum[(w * 16 * F::MT + r) * F::SUM_LD + c]);
    return v;
  };
  if constexpr (!F::GATED) {
    constexpr int kFours = F::COLUMNS / 4;
    for (int i = tid; i < t.rows * kFours; i += F::THREADS) {
      const int r = i / kFours, c = i % kFours * 4, column = block0 + c, slot = EXPERTS ? slots[r] : t.first + r;
      if (column < a.n && slot >= 0) {
        float4v v = total(r, c);
        if (a.row_weights != nullptr) v *= a.row_weights[slot];
        store4(a.y, a.y_type, slot * a.ldy + column, a.n - column, v);
      }
    }
  } else {
    // Sums stand as [wave][gate or up][columns]; 16 lanes take the block of a row, 8 columns each.
    constexpr int kHalf = F::NT / 2 * 16;
    for (int i = tid; i < (t.rows * 16 + F::THREADS - 1) / F::THREADS * F::THREADS; i += F::THREADS) {
      const int r = min(i / 16, t.rows - 1), c = i % 16 * 8, at = c / kHalf * 2 * kHalf + c % kHalf;
      float v[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float4v p = total(r, at + 4 * half), u = total(r, at + 4 * half + kHalf);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[4 * half + e] = a.gate == GGK_GATE_GELU ? gated<true>(p[e], u[e]) : gated<false>(p[e], u[e]);
        }
      }
      const int slot = EXPERTS ? slots[r] : t.first + r;
      store_numbers(a, slot, block0 + c, v, i / 16 < t.rows && slot >= 0);
    }
  }
}

// Rows without an expert.
template <class F>
__device__ __forceinline__ void clear_item(const ggk_fp8_args& a, const RowTile& t, const int* slots, int block0) {
  for (int i = threadIdx.x; i < t.rows * F::COLUMNS; i += F::THREADS) {
    const int slot = slots[i / F::COLUMNS], column = block0 + i % F::COLUMNS;
    if (column >= a.n || slot < 0) continue;
    if constexpr (F::GATED) {
      static_cast<unsigned char*>(a.y)[slot * a.ldy + column] = 0;
      if (column % kStep == 0) a.y_scales[slot * a.ldys + column / kStep] = gg::kFp8SmallestScale;
    } else {
      store_value(a.y, a.y_type, slot * a.ldy + column, 0.0f);
    }
  }
}

// PAIR: with a second product (with the arguments chosen at run time every call of experts took 2 us longer).
template <class F, bool EXPERTS, bool PAIR>
__global__ __launch_bounds__(F::THREADS, F::BYTES <= 40 * 1024 ? F::WAVES : F::BYTES <= 80 * 1024 ? F::WAVES / 2 : F::WAVES / 4) void fp8_stream_kernel(Launch l) {
  const ggk_fp8_args& a = l.a;
  __shared__ alignas(128) unsigned char s_bytes[F::BYTES];  // each wave's ring, then the sums
  if constexpr (!EXPERTS) {
    // Neighbouring workgroups go to different XCDs: each takes an eighth of the items in the order of column blocks, so that the
    // row tiles of a block follow each other and its L2 has the weights for all of them.
    const int items = l.blocks * l.tiles, share = (items + kXcds - 1) / kXcds, first_item = (int)(blockIdx.x % kXcds) * share;
    const int end = min(first_item + share, items);
    for (int item = first_item + (int)(blockIdx.x / kXcds); item < end; item += (int)(gridDim.x / kXcds)) {
      const int block = item / l.tiles, tile = item % l.tiles;
      const RowTile t{0, tile * F::R, min(F::R, a.rows - tile * F::R)};
      const bool first = !PAIR || block < l.blocks_of_a;
      run_item<F, false>(first ? l.a : l.second, t, nullptr, nullptr, first ? block : block - l.blocks_of_a, s_bytes);
      gg::stage_barrier();
    }
  } else {
    __shared__ int s_slot[F::R], s_x_row[F::R];
    __shared__ Experts<GGK_MOE_MAX_EXPERTS> s_experts;
    const int fan = a.rows / a.x_rows;
    gg::list_experts<F::THREADS, F::R>(a, s_experts);
    const long long items = (long long)s_experts.tile[a.experts + 1] * l.blocks;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
      const int tile = (int)(item / l.blocks), of = (int)(item % l.blocks);
      const bool first = !PAIR || of < l.blocks_of_a;
      const ggk_fp8_args& b = first ? l.a : l.second;
      const int block = first ? of : of - l.blocks_of_a;
      const RowTile t = gg::expert_tile<F::R>(a, s_experts, tile);
      for (int i = threadIdx.x; i < t.rows; i += F::THREADS) {
        int slot = a.order[t.first + i];
        if (slot >= a.rows) slot = -1;
        s_slot[i] = slot;
        s_x_row[i] = max(slot, 0) / fan;  // where a slot names no row, row 0: its sums are not used
      }
      gg::stage_barrier();
      if (t.expert == a.experts) {
        clear_item<F>(b, t, s_slot, block * F::COLUMNS);
      } else {
        run_item<F, true>(b, t, s_slot, s_x_row, block, s_bytes);
      }
      gg::stage_barrier();
    }
  }
}

// The 8-bit rows of gated products in a workspace, [2][rows][ld]: 16 lanes a block of a row.  Experts' slots in their order, so
// that those which it does not name stay as they are.
__global__ __launch_bounds__(256) void fp8_gate_kernel(ggk_fp8_args a, long long ld) {
  const long long blocks = (a.n + kStep - 1) / kStep, all = a.rows * blocks;
  const long long at = (long long)blockIdx.x * 16 + threadIdx.x / 16, of = at < all ? at : all - 1;
  const int j = (int)(of % blocks) * kStep + threadIdx.x % 16 * 8;
  long long row = of / blocks;
  if (a.experts > 0) row = a.order[row];
  const bool named = at < all && row >= 0 && row < a.rows;
  if (!named) row = 0;
  const float* gate = a.workspace + row * ld + j;
  const float* up = gate + a.rows * ld;
  float v[8];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float4v p = {0.0f, 0.0f, 0.0f, 0.0f}, u = p;
    if (j + 4 * half < ld) {
      p = reinterpret_cast<const float4v*>(gate)[half];
      u = reinterpret_cast<const float4v*>(up)[half];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * half + e] = a.gate == GGK_GATE_GELU ? gated<true>(p[e], u[e]) : gated<false>(p[e], u[e]);
  }
  store_numbers(a, row, j, v, named);
}

template <class F, bool EXPERTS>
hipError_t launch(const ggk_fp8_args& a, hipStream_t stream, const ggk_fp8_args* second = nullptr) {
  const int blocks = (a.n + F::COLUMNS - 1) / F::COLUMNS;
  Launch l{a, second != nullptr ? *second : a, second != nullptr ? 2 * blocks : blocks, blocks, 0};
  const long long tiles = (a.rows + F::R - 1) / F::R + (EXPERTS ? (a.rows < a.experts + 1 ? a.rows : a.experts + 1) : 0);
  long long grid;
  if (EXPERTS) {
    const long long items = tiles * l.blocks, most = kCus * (F::BYTES > 64 * 1024 ? 1 : 2);
    grid = items < most ? items : most;
  } else {
    // A launch has less than 2^32 threads; workgroups take further items in turn.  (2^30 items are 2^38 values of y at least.)
    const long long items = tiles * l.blocks, most = (1ll << 31) / F::THREADS;
    if (items > 1 << 30) return hipErrorInvalidValue;
    l.tiles = (int)tiles;
    grid = items < most ? (items + kXcds - 1) / kXcds * kXcds : most;
  }
  if constexpr (F::EXACT && !F::GATED) {
    if (second != nullptr) {
      hipLaunchKernelGGL((fp8_stream_kernel<F, EXPERTS, true>), dim3((unsigned)grid), dim3(F::THREADS), 0, stream, l);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((fp8_stream_kernel<F, EXPERTS, false>), dim3((unsigned)grid), dim3(F::THREADS), 0, stream, l);
  return hipGetLastError();
}

// What the rules below do with the form that they chose for a call: launch it, or say which it is.
struct Launches {
  hipStream_t stream;
  template <class F, bool EXPERTS>
  hipError_t take(const ggk_fp8_args& a, const ggk_fp8_args* second = nullptr) const {
    return launch<F, EXPERTS>(a, stream, second);
  }
  hipError_t take_tiles(const ggk_fp8_args& a) const { return multiply_tiles(a, stream); }
};
struct Names {
  char* text;
  int size;
  template <class F, bool EXPERTS>
  hipError_t take(const ggk_fp8_args&, const ggk_fp8_args* second = nullptr) const {
    snprintf(text, size, "stream rows=%d columns=%d k=%d %s %s %s", F::R, F::COLUMNS, F::WK, F::EXACT ? "float" : "8-bit",
             F::GATED ? "gated" : second != nullptr ? "pair" : "plain", EXPERTS ? "experts" : "one");
    return hipSuccess;
  }
  hipError_t take_tiles(const ggk_fp8_args& a) const {
    const bool gate = a.gate != GGK_GATE_NONE;
    snprintf(text, size, "tiles rows=%d columns=%d %s %s %s", tile_rows(a), gate ? 128 : 256, is_exact(a) ? "float" : "8-bit",
             gate ? "gated" : "plain", a.experts > 0 ? "experts" : "one");
    return hipSuccess;
  }
};

// What a plain call with n columns takes, in us: what the busiest CU gets, workgroups of 8 or 16 rows by 16 columns, or of 32 by 32,
// two on a CU; of 32 by 16 where one is enough.  Where x is larger than an XCD's L2, its rows come from beyond it for every column
// block: a step of 4 MB of x takes 0.19 us in binary16 (0.15 by the 8-bit instructions), of 6 MB 0.22, of 8 MB and more 0.27.
double estimate_rows(const ggk_fp8_args& a, double n) {
  const double steps = a.k / 128.0;
  if (a.rows <= 16) return 4 + ceil(ceil(n / 16) / (2 * kCus)) * (1 + 0.08 * steps);
  if (row_tiles(a, 32) * ceil(n / 16) <= kCus) return 5 + 0.075 * steps;
  const double in_l2 = (double)a.rows * a.k / 4e6, memory = 0.15 * (in_l2 > 1.8 ? 1.8 : in_l2), unit = is_exact(a) ? 0.19 : 0.15;
  const double step = memory > unit ? memory : unit;
  return 4 + ceil(row_tiles(a, 32) * ceil(n / 32) / (2 * kCus)) * (1.3 + step * steps);
}

// Gated products of 16 rows at once where every CU can get its own tile, else of 32.  us of the two: 32 rows of 4096 by 14336
// 36, 48, 128 of 4096 by 4096 25.5, 30; 64 rows of 4096 by 14336 62, 45, 32 of 8192 by 28672 133, 108.
bool has_own_tiles(const ggk_fp8_args& a) { return row_tiles(a, 16) * ceil(a.n / 128.0) <= kCus; }

// What a call takes here, in us; gated workgroups are alone on a CU.
double estimate_few(const ggk_fp8_args& a) {
  const double items = row_tiles(a, 32) * ceil(a.n / 128.0), rounds = ceil(items / kCus), steps = a.k / 128.0;
  if (a.gate == GGK_GATE_NONE) return a.experts > 0 ? 5 + rounds * 0.6 * steps : estimate_rows(a, a.n);
  if (a.experts > 0) return 5 + (rounds > 1 ? rounds * (2.5 + 1.15 * steps) : 1.5 + 0.95 * steps);
  const double cus = has_own_tiles(a) ? 0.62 * steps : rounds > 1 ? rounds * (2 + 1.05 * steps) : 1 + 0.85 * steps,
               memory = 2.0 * a.n * a.k / 4.5e6;
  return 4.5 + (cus > memory ? cus : memory);
}

// One matrix, or two of one shape: y and second's from the same rows.
template <class Run>
hipError_t multiply_rows(const ggk_fp8_args& a, const Run& run, const ggk_fp8_args* second = nullptr) {
  const bool exact = is_exact(a);
  const long long n = second != nullptr ? 2ll * a.n : a.n;
  // us by 8 rows at once, by 16, by 16 and 32 columns: 8 rows of 4096 by 4096 5.7, 6.0, 6.7, by 14336 11.5, 12.4, 11.3; 16 rows
  // 6.2, 5.7, 6.8 and 13.8, 12.4, 11.5, of 8192 by 8192 14.6, 12.3, 12.3.
  if (a.rows <= 8) return run.template take<Form<8, 1, 1, 8, 2, false, true>, false>(a, second);
  if (a.rows <= 16) {
    return n >= 8192 ? run.template take<Form<16, 1, 2, 4, 2, false, true>, false>(a, second)
                     : run.template take<Form<16, 1, 1, 8, 2, false, true>, false>(a, second);
  }
  // 32 rows twice where no CU gets a fourth of those workgroups (two are at work at once), else 64 at once.  us of the two: 64 rows of
  // 4096 by 12288 15.4, 16.7, by 12544 18.7, 16.8, 33 rows 14.9, 16.1 and 18.0, 16.2; of 8192 by 8192 17, 24, by 12800 42, 32; by
  // the 8-bit instructions 64 rows of 4096 by 12288 13.2, 15.4, by 12544 16.0, 15.5, 33 rows 12.5, 14.8 and 15.0, 14.8.
  if (a.rows > 32 && a.rows <= 64 && 2 * ((n + 31) / 32) > 3 * kCus) {
    return exact ? run.template take<Form<64, 4, 1, 4, 2, false, true>, false>(a, second)
                 : run.template take<Form<64, 4, 1, 4, 2, false, false>, false>(a, second);
  }
  // 16 columns with K shared by 8 waves where every CU can get its own, else 32 by 4.  us of the two: 128 rows of 8192 by 1024
  // 8.9, 10, 32 rows 7.2, 9.7, in float 8.3, 12; 32 of 14336 by 4096 14.2, 15.5; 64 of 4096 by 4096 9.9, 7.0.
  if (row_tiles(a, 32) * ceil(n / 16.0) <= kCus) {
    return exact ? run.template take<Form<32, 1, 1, 8, 2, false, true>, false>(a, second)
                 : run.template take<Form<32, 1, 1, 8, 2, false, false>, false>(a, second);
  }
  if (exact) return run.template take<Form<32, 2, 1, 4, 2, false, true>, false>(a, second);
  return run.template take<Form<32, 2, 1, 4, 2, false, false>, false>(a, second);
}

// The same for experts' slots: 8 rows by 32 columns, 16 by 256 or 32 by 128 (those share K by 4 waves, none and 2).  us of the three:
// 2 slots of 8 experts of 4096 by 14336 25, 25, 22, by 3584 9 by the first, 17.5 by the last.  Of the last two, by K: 256 slots of 128
// experts of 512 by 1408 twice 31, 34, 1200 slots of 1024 by 2048 59, 64; 64 slots of 64 experts of 2048 by 2048 21, 23.5, 700
// slots 59, 63; 256 slots of 32 experts of 4096 by 1408 twice 86, 80, 128 slots of 7168 125, 115, of 16 of 8192 by 512 51, 36;
// by slots an expert: 512 slots of 16 experts of 1024 by 2048 18, 16, 180 slots 11, 16.
bool is_narrow(const ggk_fp8_args& a, double n) { return a.rows <= 32 && row_tiles(a, 32) * ceil(n / 128) <= kCus / 4 * 3; }
bool is_sparse(const ggk_fp8_args& a) { return a.rows > 32 && a.rows <= 12ll * a.experts && a.k <= 2048; }
template <class Run>
hipError_t multiply_slots(const ggk_fp8_args& a, const Run& run, const ggk_fp8_args* second = nullptr) {
  if (is_narrow(a, second != nullptr ? 2.0 * a.n : a.n)) return run.template take<Form<8, 1, 2, 4, 2, false, true>, true>(a, second);
  if (is_sparse(a)) return run.template take<Form<16, 2, 8, 1, 3, false, true>, true>(a, second);
  if (is_exact(a)) return run.template take<Form<32, 2, 4, 2, 2, false, true>, true>(a, second);
  return run.template take<Form<32, 2, 4, 2, 2, false, false>, true>(a, second);
}
double estimate_slots(const ggk_fp8_args& a, double n) {
  const double steps = a.k / 128.0;
  if (is_narrow(a, n)) return 5 + ceil(row_tiles(a, 8) * ceil(n / 32) / (2 * kCus)) * (1 + 0.19 * steps);
  if (is_sparse(a)) return 5 + ceil(row_tiles(a, 16) * ceil(n / 256) / kCus) * 0.8 * steps;
  return 5 + ceil(row_tiles(a, 32) * ceil(n / 128) / kCus) * 0.6 * steps;
}

template <bool EXPERTS, class Run>
hipError_t multiply_few(const ggk_fp8_args& a, const Run& run) {
  if constexpr (EXPERTS) {
    // us with 32 rows at once, 16, 8: 16 experts of 1024 by 2048, 64 slots 16, 16, 18, 512 slots 25, 29, 41; 64 experts of 4096
    // by 14336, 16 slots 223, 218, 216, 256 slots 1011, 1022, 1095.
    if (a.gate != GGK_GATE_NONE) return run.template take<Form<32, 2, 8, 1, 2, true, true>, true>(a);
    return multiply_slots(a, run);
  } else if (a.gate != GGK_GATE_NONE) {
    if (a.rows <= 8) return run.template take<Form<8, 4, 4, 1, 4, true, true>, false>(a);
    if (has_own_tiles(a)) return run.template take<Form<16, 2, 8, 1, 3, true, true>, false>(a);
    return run.template take<Form<32, 2, 8, 1, 2, true, true>, false>(a);
  } else {
    return multiply_rows(a, run);
  }
}

// Gated products as both plain products, whose workgroups take 16 or 32 columns and share K, and their rows in a second launch:
// a block of an 8-bit row needs the largest of 128 columns, and so few workgroups cannot bring in the weights as fast.  us by one
// launch and by two: 1 row of 4096 by 14336 28.6, 25.3, by 2048 24.7, 9.3; 42 of 13280 by 1666 86, 22; 256 of 4096 by 1792 25.6,
// 22.3; 1 of 512 by 512 6.3, 9.4; 512 of 4096 by 1792 31, 34.6; 7267 of 480 by 246 15.7, 27; 2 slots of 8 experts of 4096 by 1792
// 31, 13, by 14336 45.8, 47.5; 512 slots of 16 experts of 1024 by 2048 25, 32.
constexpr long long kMostOfPair = 1 << 24;  // values of either product: 128 MB of workspace at most
long long pair_ld(const ggk_fp8_args& a) { return (a.n + 3) / 4 * 4; }
bool as_pair(const ggk_fp8_args& a) {
  if (a.gate == GGK_GATE_NONE || a.rows == 0 || a.n == 0 || a.rows * pair_ld(a) > kMostOfPair) return false;
  const double matrices = a.experts == 0 ? 1 : a.rows < a.experts ? a.rows : a.experts;
  const double memory = matrices * 2.0 * a.n * a.k / 5.5e6;
  const double cus = a.experts > 0 ? estimate_slots(a, 2.0 * a.n) - 2 : estimate_rows(a, 2.0 * a.n) - 4;
  const double two = 6 + (cus > memory ? cus : memory) + 16.0 * a.rows * a.n / 4e6, pair = two > 9.5 ? two : 9.5;
  return pair < (a.experts > 0 ? 0.9 : 1) * estimate_few(a) && !(tiles_take(a) && estimate_tiles(a) <= pair);
}
template <class Run>
hipError_t multiply_both(const ggk_fp8_args& a, const Run& run) {
  const long long ld = pair_ld(a);
  ggk_fp8_args gate = a;
  gate.gate = GGK_GATE_NONE;
  gate.y = a.workspace;
  gate.ldy = ld;
  gate.y_type = GGK_TYPE_F32;
  ggk_fp8_args up = gate;
  up.w = a.up;
  up.ldw = a.ldu;
  up.w_scales = a.up_scales;
  up.ldws = a.ldus;
  up.stride_w = a.stride_u;
  up.stride_ws = a.stride_us;
  up.y = a.workspace + a.rows * ld;
  return a.experts > 0 ? multiply_slots(gate, run, &up) : multiply_rows(gate, run, &up);
}
hipError_t multiply_pair(const ggk_fp8_args& a, hipStream_t stream) {
  const long long ld = pair_ld(a), blocks = (a.n + kStep - 1) / kStep;
  const hipError_t st = multiply_both(a, Launches{stream});
  if (st != hipSuccess) return st;
  hipLaunchKernelGGL(fp8_gate_kernel, dim3((unsigned)((a.rows * blocks + 15) / 16)), dim3(256), 0, stream, a, ld);
  return hipGetLastError();
}

long long pair_floats(const ggk_fp8_args& a) { return 2ll * a.rows * pair_ld(a); }
// As two launches: where the workspace is there for it.
bool with_workspace(const ggk_fp8_args& a) { return a.workspace != nullptr && a.workspace_floats > 0 && as_pair(a); }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Everything but the workspace's size.
hipError_t check(const ggk_fp8_args& a) {
  const bool gate = a.gate != GGK_GATE_NONE;
  if (a.rows < 0 || a.rows > GGK_ROUTE_MAX_TOTAL_SLOTS || a.x_rows < 0 || a.n < 0 || a.n > GGK_FP8_MAX_N || a.k < 16 ||
      a.k > GGK_FP8_MAX_K || a.k % 16 != 0 || a.experts < 0 || a.experts > GGK_MOE_MAX_EXPERTS ||
      a.gate < GGK_GATE_NONE || a.gate > GGK_GATE_GELU ||
      (!gate && a.y_type != GGK_TYPE_F32 && a.y_type != GGK_TYPE_F16 && a.y_type != GGK_TYPE_BF16) ||
      (gate && a.row_weights != nullptr) || a.fast < 0 || a.fast > 1 || (a.fast != 0 && (gate || a.y_type == GGK_TYPE_F32))) {
    return hipErrorInvalidValue;
  }
  if (a.experts == 0 ? a.rows != a.x_rows : (a.rows > 0 && (a.x_rows < 1 || a.rows % a.x_rows != 0))) {
    return hipErrorInvalidValue;
  }
  const long long blocks_k = (a.k + kStep - 1) / kStep, blocks_n = (a.n + kStep - 1) / kStep;
  const auto matrix = [&](const void* w, long long ld, long long stride, long long lds, long long stride_s) {
    if (a.n > 1 && (ld < a.k || ld > GGK_FP8_MAX_LD || ld % 16 != 0)) return false;
    if (blocks_n > 1 && lds < blocks_k) return false;
    return aligned16(w) && stride >= 0 && stride_s >= 0 && (a.experts <= 1 || stride % 16 == 0);
  };
  if (!matrix(a.w, a.ldw, a.stride_w, a.ldws, a.stride_ws) ||
      (gate && !matrix(a.up, a.ldu, a.stride_u, a.ldus, a.stride_us))) {
    return hipErrorInvalidValue;
  }
  if (!aligned16(a.x) || (a.x_rows > 1 && (a.ldx < a.k || a.ldx % 16 != 0 || a.ldxs < blocks_k)) ||
      (a.rows > 1 && (a.ldy < a.n || (gate && a.ldys < blocks_n)))) {
    return hipErrorInvalidValue;
  }
  if (!aligned16(a.workspace)) return hipErrorInvalidValue;
  if (a.rows > 0 && a.n > 0) {
    if (a.x == nullptr || a.x_scales == nullptr || a.w == nullptr || a.w_scales == nullptr || a.y == nullptr ||
        (gate && (a.up == nullptr || a.up_scales == nullptr || a.y_scales == nullptr)) ||
        (a.experts > 0 && (a.counts == nullptr || a.order == nullptr))) {
      return hipErrorInvalidDevicePointer;
    }
  }
  return hipSuccess;
}

// One launch.
template <class Run>
hipError_t multiply_one(const ggk_fp8_args& a, const Run& run) {
  // Few rows stream, many go on tiles, by what either is expected to take.  us of the two: 1536 rows of 2048 by 2048 30, 33, 2048
  // 39, 33; 512 of 4096 by 4096 33, 58, 1024 64, 59; 1024 of 8192 by 2048 73, 110, 1536 114, 111; 16 experts of 1024 by 2048, 512
  // slots 16, 24, 2048 slots 33, 25, gated 25, 46 and 53, 50; 64 experts of 4096 by 14336, 1024 slots 764, 882, 4096 slots 1366,
  // 1099.  By the 8-bit instructions 768 rows of 2048 by 2048 14, 16, 1536 25, 17; 384 of 4096 by 4096 22, 26, 768 40, 27; 64 experts
  // of 4096 by 14336, 512 slots 588, 574 (256 slots, 456 and 470, are missed: their counts are not known here).
  if (tiles_take(a) && estimate_tiles(a) < estimate_few(a)) return run.take_tiles(a);
  return a.experts > 0 ? multiply_few<true>(a, run) : multiply_few<false>(a, run);
}

// used: with_workspace(a).
hipError_t check_workspace(const ggk_fp8_args& a, bool used) {
  return a.workspace_floats < 0 || (used && a.workspace_floats < pair_floats(a)) ? hipErrorInvalidValue : hipSuccess;
}

}  // namespace

extern "C" hipError_t ggk_fp8_check(const ggk_fp8_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const hipError_t st = check(*args);
  return st != hipSuccess ? st : check_workspace(*args, with_workspace(*args));
}

extern "C" hipError_t ggk_fp8_workspace(const ggk_fp8_args* args, long long* floats) {
  const hipError_t st = floats == nullptr || args == nullptr ? hipErrorInvalidValue : check(*args);
  if (st == hipSuccess) *floats = as_pair(*args) ? pair_floats(*args) : 0;
  return st;
}

extern "C" hipError_t ggk_fp8_multiply(const ggk_fp8_args* args, hipStream_t stream) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_fp8_args& a = *args;
  hipError_t st = check(a);
  if (st != hipSuccess) return st;
  const bool pair = with_workspace(a);
  st = check_workspace(a, pair);
  if (st != hipSuccess || a.rows == 0 || a.n == 0) return st;
  if (pair) return multiply_pair(a, stream);
  return multiply_one(a, Launches{stream});
}

extern "C" hipError_t ggk_fp8_form(const ggk_fp8_args* args, char* text, int size) {
  hipError_t st = text == nullptr || size < 1 ? hipErrorInvalidValue : ggk_fp8_check(args);
  if (st != hipSuccess) return st;
  text[0] = 0;
  if (args->rows == 0 || args->n == 0) return st;
  const Names names{text, size};
  return with_workspace(*args) ? multiply_both(*args, names) : multiply_one(*args, names);
}
