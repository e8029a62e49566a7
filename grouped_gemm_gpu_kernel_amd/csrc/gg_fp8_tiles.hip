// gg_fp8_tiles.hip -- products of many rows with matrices of 8-bit numbers, one
// matrix or one an expert, plain or gated, on tiles of 256 or 128 rows by 256 columns.
//
// A workgroup of 8 waves (2 x 4) computes 256 rows of x by 256 columns.  A stage is one block of K, 128 bytes of each row, in
// four units of 16 KB in the order the loop reads them:
//   B0, B1  half of each wave's columns (with a gate: gate, up)
//   A0, A1  rows 0 .. 127 and 128 .. 255 of the tile, 64 of each a wave
// LDS holds two stages; loads go straight into it, five units ahead.  A phase multiplies one pair of units, 64 x 32 a
// wave: 8 instructions of 16 x 16 x 128.  Their results are one block's sums, which a multiply-add brings into the sums in
// float with the block's scales: that runs on the vector unit beside the matrix unit, two instructions behind it.
//   phase 0  A0 B0, reads B1            phase 2  A1 B0, reads B0 of the next stage
//   phase 1  A0 B1, reads A1            phase 3  A1 B1, reads A0 of the next stage
// Fragments are read into registers as their last use frees them, so that A and B take 64 registers beside 128 of sums.
// Phase f reads unit f + 2, issues the loads of unit f + 8 into the place whose fragments phase f - 2 read, and waits at
// its end for this wave's loads of unit f + 3 and its reads of the phases before; one barrier tells every wave both.
//
// Tiles of 128 rows (A0 alone) hold three stages in LDS and the next stage's fragments in a second set of registers, with one
// barrier a stage.  Products are made in binary16, on tiles of 128 rows, unless the caller asks for the 8-bit instructions; with a
// gate a tile has 128 columns of both matrices.  8192^3 takes 915 to 975 us by card (1.1 to 1.2 PFLOP/s), by the 8-bit instructions
// 428 to 508 (2.2 to 2.6), at the clock that its power allows; on zeros those take 331.  64 experts of 4096 by 14336, 16384 slots: 2235
// to 2340 us, and 1265 to 1370, the latter by HBM where experts have few rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>
#include <type_traits>

#include "gg_experts.h"
#include "gg_fp8.h"
#include "gg_phased.h"  // wait_lgkmcnt, phase_barrier

namespace {

using namespace gg::fp8;
using gg::RowTile;
using gg::kWave;

constexpr int kCus = 256, kXcds = 8;
constexpr int kRows = 256, kWaves = 8, kThreads = kWaves * kWave;
constexpr int kUnit = 128 * kStep;  // bytes
constexpr int kB0 = 0, kA0 = kUnit, kB1 = 2 * kUnit, kA1 = 3 * kUnit, kParity = 4 * kUnit, kPlaces = 9;
constexpr int kLoads = 2;           // load instructions of a unit and wave
constexpr int kScaleSteps = 4;      // stages of scales loaded at once, 16 bytes a row
constexpr int kScales = 4096 + 128; // bytes of those: 256 rows, and a row of each unit's weights
constexpr int kMost = 512;          // experts that the table has room for
constexpr int kGroup = 4;           // row tiles that go along the columns together

template <bool GATED>
constexpr int kColumns = GATED ? 128 : 256;

struct Launch {
  ggk_fp8_args a;
  int blocks;            // of columns
  int height;            // rows of a tile, 256 or 128
  int fan;               // slots of a row of x
  uint32_t scale_bytes;  // of all of x's scales (experts)
};

struct Shared {
  unsigned char* stages;  // places of units, then two sets of scales
  int* slot;              // of the tile's rows, -1 for none
};

// Sums of one tile: [rows half][16 rows][unit of columns][16 columns].
template <int HALVES>
using Sums = float4v[HALVES][4][2][2];

template <bool EXPERTS, bool GATED>
struct Loader {
  const ggk_fp8_args& a;
  uint32_t a_off[2][2];  // [half][load]
  const unsigned char* x0;
  const unsigned char* b0[2];  // by unit; the same matrix without a gate
  uint32_t b_off[2], b_records[2], b_step[2];
  uint32_t s_off, s_records;
  const float* s0;
  int piece16, wave;

  __device__ __forceinline__ Loader(const Launch& l, const RowTile& t, const int* slot, int n0, int wave_)
      : a(l.a), wave(wave_) {
    const int tid = gg::opaque_tid(wave), row = tid / 8;
    const int piece = (tid & 7) ^ (row >> 1 & 7);
    piece16 = 16 * piece;
    x0 = EXPERTS ? a.x : a.x + t.first * a.ldx;
    // Where a slot names no row, row 0: its sums are not used.
    auto x_row = [&](int r) { return (unsigned)max(slot[r], 0) / (unsigned)l.fan; };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // Rows past the tile's are zeros: nothing is read for them, and their products take less power.
        const int r = 128 * half + 64 * i + row;
        a_off[half][i] = r < t.rows ? (uint32_t)((EXPERTS ? x_row(r) : r) * a.ldx) + piece16 : 0xffffffffu;
      }
    }
    const int column = GATED ? row : 64 * (row / 32) + row % 32;
#pragma unroll
    for (int unit = 0; unit < 2; ++unit) {
      const bool up = GATED && unit == 1;
      const long long ld = up ? a.ldu : a.ldw;
      b0[unit] = (up ? a.up + t.expert * a.stride_u : a.w + t.expert * a.stride_w) + n0 * ld;
      b_off[unit] = (uint32_t)(column * ld) + piece16;
      // Rows past the matrix lie past the records and read as zero.
      const long long records = (long long)(min(a.n - n0, 256) - 1) * ld + a.k;
      b_records[unit] = (uint32_t)records;
      b_step[unit] = (uint32_t)((GATED ? 64 : 128) * ld);
    }
    // Scales of four stages, 16 bytes a row: waves 0 to 3 x's, 4 and 5 the units' of the weights.
    const int blocks_k = (a.k + kStep - 1) / kStep;
    if (wave < 4) {
      const int r = min(tid, t.rows - 1);
      s0 = EXPERTS ? a.x_scales : a.x_scales + t.first * a.ldxs;
      s_off = (uint32_t)((EXPERTS ? x_row(r) : r) * a.ldxs * 4);
      s_records = EXPERTS ? l.scale_bytes : (uint32_t)(((t.rows - 1) * a.ldxs + blocks_k) * 4);
    } else {
      const int block = n0 / kStep, unit = wave & 1;
      if (GATED && unit == 1) {
        s0 = a.up_scales + t.expert * a.stride_us + block * a.ldus;
      } else {
        const int at = min(block + (GATED ? 0 : unit), (a.n - 1) / kStep);
        s0 = a.w_scales + t.expert * a.stride_ws + at * a.ldws;
      }
      s_off = 0;
      s_records = (uint32_t)(blocks_k * 4);
    }
  }

  __device__ __forceinline__ void issue_a(int kt, int half, uint32_t unit, int i) const {
    const uint32_t off = kt * kStep + piece16 < a.k ? a_off[half][i] : 0xffffffffu;
    gg::load_to_lds16(x0 + kt * kStep, 0xfffffff0u, unit + 1024u * (uint32_t)(i * kWaves + wave), off, 0);
  }
  __device__ __forceinline__ void issue_b(int kt, int which, uint32_t unit, int i) const {
    const uint32_t off = kt * kStep + piece16 < a.k ? b_off[which] : kOutOfRange;
    const uint32_t records = kt * kStep < a.k ? b_records[which] - kt * kStep : 0;
    gg::load_to_lds16(b0[which] + kt * kStep, records, unit + 1024u * (uint32_t)(i * kWaves + wave), off,
                      i * b_step[which] + (GATED ? 0 : which * (b_step[which] / 4)));
  }
  __device__ __forceinline__ void issue_scales(int chunk, uint32_t scales) const {
    const uint32_t skip = 4 * kScaleSteps * chunk;
    if (wave < 4) {
      gg::load_to_lds16(s0 + kScaleSteps * chunk, s_records - skip, scales + 1024u * (uint32_t)wave, s_off, 0);
    } else if (wave < 6 && gg::opaque_lane() == 0) {  // the other lanes' places are not theirs
      gg::load_to_lds16(s0 + kScaleSteps * chunk, s_records - skip, scales + 4096u + 16u * (uint32_t)(wave - 4), s_off, 0);
    }
  }
};

// Of a lane in the operands of the instructions: LDS byte addresses of its fragments in the first unit, in the two pieces that
// a fragment is read as, and of its scales.
template <bool GATED>
struct Lane {
  uint32_t a_lo, a_hi, b_lo, b_hi, x_scale, w_scale;
  __device__ __forceinline__ Lane(uint32_t lds, int wave) {
    const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
    const int wm = wave >> 2, wn = wave & 3;
    const uint32_t at = (uint32_t)(j * 128 + ((g ^ (j >> 1)) & 7) * 16);
    a_lo = lds + at + wm * 64 * 128;
    a_hi = lds + (at ^ 64) + wm * 64 * 128;
    b_lo = lds + at + wn * 32 * 128;
    b_hi = lds + (at ^ 64) + wn * 32 * 128;
    x_scale = lds + kPlaces * kUnit + (wm * 64 + j) * 16;
    w_scale = lds + kPlaces * kUnit + 4096 + (GATED ? 0 : (wn >> 1) * 16);
  }
};

// A lane's address in a fragment's unit, held in a register (the empty asm): reads add the rest as the instructions' own
// offsets.  With an addition for every read the vector unit was short of slots beside the matrix instructions (8192^3: 460 us
// instead of 444).
__device__ __forceinline__ uint32_t held(uint32_t at) {
  asm volatile("" : "+v"(at));
  return at;
}

__device__ __forceinline__ void add_scaled(float4v& sum, const float4v& v, float scale) {
#pragma unroll
  for (int e = 0; e < 4; ++e) sum[e] = fmaf(scale, v[e], sum[e]);
}

// Scales of stage kt lie in set (kt / 4) % 2.
__device__ __forceinline__ uint32_t scales_of(int kt) { return ((kt >> 2) & 1) * kScales + (kt & 3) * 4; }

template <int HALVES>
__device__ __forceinline__ void clear(Sums<HALVES>& acc) {
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[h][i][u][n] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
  }
}

// The sums of the tile of at most 128 rows at rows t, columns n0 on.
template <bool EXPERTS>
__device__ __forceinline__ void multiply_tile(const Launch& l, const RowTile& t, const Shared& s, int n0, int wave,
                                              Sums<1>& acc) {
  const ggk_fp8_args& p = l.a;
  const int nk = (p.k + kStep - 1) / kStep;
  const Loader<EXPERTS, false> loader(l, t, s.slot, n0, wave);
  const uint32_t lds = gg::lds_address(s.stages), scales_at = lds + kPlaces * kUnit;
  const Lane<false> lane(lds, wave);

  // Two sets of operands: one is multiplied while the next stage's is read into the other.
  int8v a[2][4], b[2][4];  // [set][16 rows], [set][2 unit + 16 columns]
  float x_scale[2][4], w_scale[2];
  float4v part[16];  // results of this stage's instructions, three of them alive
  float4v left[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};  // of the stage before, its last two
  float left_scale = 0.0f;
  clear<1>(acc);

  uint32_t lo, hi;
  auto read = [&](uint32_t place, int set, int f) {  // fragment f (0..7): the stage's columns, then its rows
    if (f == 0) {
      lo = held(lane.b_lo + place);
      hi = held(lane.b_hi + place);
    }
    if (f == 4) {
      lo = held(lane.a_lo + place);
      hi = held(lane.a_hi + place);
    }
    if (f < 4) {
      b[set][f] = read_fragment(lo, hi, (f / 2) * 2 * kUnit + (f % 2) * 2048u);
    } else {
      a[set][f - 4] = read_fragment(lo, hi, kUnit + (f - 4) * 2048u);
    }
  };
  auto read_scales = [&](int kt, int set) {
    const uint32_t at = scales_of(kt);
#pragma unroll
    for (int i = 0; i < 4; ++i) x_scale[set][i] = *(const GG_LDS float*)(uintptr_t)(lane.x_scale + at + 256u * i);
    w_scale[set] = *(const GG_LDS float*)(uintptr_t)(lane.w_scale + at);
  };
  auto issue = [&](int kt, uint32_t place, int i) {  // load i (0..5) of a stage; past K zeros, and memory is not touched
    if (i / 2 == 1) {
      loader.issue_a(kt, 0, lds + place + kUnit, i % 2);
    } else {
      loader.issue_b(kt, i / 4, lds + place + i / 2 * kUnit, i % 2);
    }
  };

  loader.issue_scales(0, scales_at);
#pragma unroll
  for (int kt = 0; kt < 3; ++kt) {
#pragma unroll
    for (int i = 0; i < 6; ++i) issue(kt, kt * 3 * kUnit, i);
  }
  gg::wait_vmcnt<12>();
  gg::phase_barrier();
#pragma unroll
  for (int f = 0; f < 8; ++f) read(0, 0, f);
  read_scales(0, 0);
  gg::wait_vmcnt<6>();
  gg::wait_lgkmcnt<0>();
  gg::phase_barrier();

  // Stage kt, whose operands are in set `set` and whose three places, at `here`, are free.
  uint32_t here = 0;
  auto stage = [&](int kt, auto set_tag) {
    constexpr int set = decltype(set_tag)::value, other = 1 - set;
    const uint32_t next = here == 6 * kUnit ? 0 : here + 3 * kUnit;
    if ((kt & 3) == 0 && kt + kScaleSteps < nk) loader.issue_scales(kt / 4 + 1, scales_at + ((kt / 4 + 1) & 1) * kScales);
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = x_scale[set][i] * w_scale[set];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = r / 4, n = (i & 1) != 0 ? 3 - r % 4 : r % 4;
      part[r] = multiply(b[set][n], a[set][i]);
      __builtin_amdgcn_sched_barrier(0);
      if (r < 2) {
        add_scaled(acc[0][3][0][1 - r], left[r], left_scale);
      } else {
        const int q = r - 2, qi = q / 4, qn = (qi & 1) != 0 ? 3 - q % 4 : q % 4;
        add_scaled(acc[0][qi][qn / 2][qn % 2], part[q], scale[qi]);
      }
      if (r < 12 && r % 3 != 2) read(next, other, r / 3 * 2 + r % 3);
      if (r == 12) read_scales(kt + 1, other);
      if (r % 3 == 2) issue(kt + 3, here, r / 3);
      if (r == 15) issue(kt + 3, here, 5);
      __builtin_amdgcn_sched_barrier(0);
    }
    left[0] = part[14];
    left[1] = part[15];
    left_scale = scale[3];
    // The next stage's operands are in every wave's registers, and the one after it has landed.
    gg::wait_lgkmcnt<0>();
    gg::wait_vmcnt<6>();
    gg::phase_barrier();
    here = next;
  };
  int kt = 0;
#pragma unroll 1
  for (; kt + 1 < nk; kt += 2) {
    stage(kt, std::integral_constant<int, 0>{});
    stage(kt + 1, std::integral_constant<int, 1>{});
  }
  if (kt < nk) stage(kt, std::integral_constant<int, 0>{});
  add_scaled(acc[0][3][0][1], left[0], left_scale);
  add_scaled(acc[0][3][0][0], left[1], left_scale);
  gg::wait_vmcnt<0>();
}

// The same in binary16, which holds the numbers exactly.  A wave turns its fragments into binary16 once a stage, 128
// instructions beside 64 products that take the matrix unit four times as long each: while a quarter of x's or w's is multiplied
// for the last time, the next one takes its registers.  Turned into binary16 in front of the stage's products, 8192^3 in float
// took 1026 us, so 970 on the same card; leaving out products of rows past the tile's, in tiles of 64 or 32 rows or by a branch
// around them, gained nothing: zeros take little power.
template <bool EXPERTS, bool GATED>
__device__ __forceinline__ void multiply_tile_exact(const Launch& l, const RowTile& t, const Shared& s, int n0, int wave,
                                                    Sums<1>& acc) {
  const ggk_fp8_args& p = l.a;
  const int nk = (p.k + kStep - 1) / kStep;
  const Loader<EXPERTS, GATED> loader(l, t, s.slot, n0, wave);
  const uint32_t lds = gg::lds_address(s.stages), scales_at = lds + kPlaces * kUnit;
  const Lane<GATED> lane(lds, wave);
  uint4v a[4][2], b[2][4];  // pieces of 16 numbers
  float x_scale[4], w_scale[2];
  clear<1>(acc);

  auto read_a = [&](uint32_t place, int i) {
    a[i][0] = read_piece(lane.a_lo + place, kUnit + i * 2048u);
    a[i][1] = read_piece(lane.a_hi + place, kUnit + i * 2048u);
  };
  auto read_b = [&](uint32_t place, int half) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      b[half][n] = read_piece((half == 0 ? lane.b_lo : lane.b_hi) + place, (n / 2) * 2 * kUnit + (n % 2) * 2048u);
    }
  };
  auto quarter = [](const uint4v& piece, int q) { return q % 2 == 0 ? to_halves(piece.x, piece.y) : to_halves(piece.z, piece.w); };
  auto read_scales = [&](int kt) {
    const uint32_t at = scales_of(kt);
#pragma unroll
    for (int i = 0; i < 4; ++i) x_scale[i] = *(const GG_LDS float*)(uintptr_t)(lane.x_scale + at + 256u * i);
    w_scale[0] = *(const GG_LDS float*)(uintptr_t)(lane.w_scale + at);
    if constexpr (GATED) w_scale[1] = *(const GG_LDS float*)(uintptr_t)(lane.w_scale + at + 16u);
  };
  auto issue = [&](int kt, uint32_t place, int i) {  // load i (0..5) of a stage; past K zeros, and memory is not touched
    if (i / 2 == 1) {
      loader.issue_a(kt, 0, lds + place + kUnit, i % 2);
    } else {
      loader.issue_b(kt, i / 4, lds + place + i / 2 * kUnit, i % 2);
    }
  };

  loader.issue_scales(0, scales_at);
#pragma unroll
  for (int kt = 0; kt < 3; ++kt) {
#pragma unroll
    for (int i = 0; i < 6; ++i) issue(kt, kt * 3 * kUnit, i);
  }
  gg::wait_vmcnt<12>();
  gg::phase_barrier();
  read_b(0, 0);
  read_b(0, 1);
#pragma unroll
  for (int i = 0; i < 4; ++i) read_a(0, i);
  gg::wait_vmcnt<6>();
  gg::wait_lgkmcnt<0>();
  gg::phase_barrier();

  half8v w[4][4], x[4];  // [16 columns][quarter], [quarter]
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    x[q] = quarter(a[0][q / 2], q);
#pragma unroll
    for (int n = 0; n < 4; ++n) w[n][q] = quarter(b[q / 2][n], q);
  }

  // Stage kt, whose operands are in registers and whose three places, at `here`, are free.  As the last products with a
  // quarter of x or w are on their way, the next ones' numbers take its registers.
  uint32_t here = 0;
#pragma unroll 1
  for (int kt = 0; kt < nk; ++kt) {
    const uint32_t next = here == 6 * kUnit ? 0 : here + 3 * kUnit;
    if ((kt & 3) == 0 && kt + kScaleSteps < nk) loader.issue_scales(kt / 4 + 1, scales_at + ((kt / 4 + 1) & 1) * kScales);
    read_scales(kt);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // The loads of stage kt + 3.
#pragma unroll
      for (int load = 6 * i / 4; load < 6 * (i + 1) / 4; ++load) issue(kt + 3, here, load);
      read_a(next, i);
      float4v part[4] = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (i == 3 && q % 2 == 0) read_b(next, q / 2);
#pragma unroll
        for (int n = 0; n < 4; ++n) part[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[n][q], x[q], part[n], 0, 0, 0);
        x[q] = quarter(a[(i + 1) % 4][q / 2], q);
        if (i == 3 && q % 2 == 1) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            w[n][q - 1] = quarter(b[q / 2][n], q - 1);
            w[n][q] = quarter(b[q / 2][n], q);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) add_scaled(acc[0][i][n / 2][n % 2], part[n], x_scale[i] * w_scale[GATED ? n / 2 : 0]);
    }
    // The next stage's operands are in every wave's registers, and the one after it has landed.
    gg::wait_lgkmcnt<0>();
    gg::wait_vmcnt<6>();
    gg::phase_barrier();
    here = next;
  }
  gg::wait_vmcnt<0>();
}

// The sums of the tile of more rows at rows t, columns n0 on.
template <bool EXPERTS>
__device__ __forceinline__ void multiply_tile(const Launch& l, const RowTile& t, const Shared& s, int n0, int wave,
                                              Sums<2>& acc) {
  const ggk_fp8_args& p = l.a;
  const int nk = (p.k + kStep - 1) / kStep;
  const Loader<EXPERTS, false> loader(l, t, s.slot, n0, wave);
  const uint32_t lds = gg::lds_address(s.stages), scales_at = lds + kPlaces * kUnit;
  const Lane<false> lane(lds, wave);

  int8v a[4], b[2][2];
  float x_scale[2][4], w_scale, w_next;  // x's by half of the rows; of the next stage while this one's are used
  float4v part[8];      // results of this phase's instructions, three of them alive
  float4v left[2];      // of the phase before, its last two
  float left_scale;
  clear<2>(acc);
  left[0] = left[1] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  left_scale = 0.0f;

  uint32_t lo, hi;
  auto read_a = [&](uint32_t parity, uint32_t unit, int i) {
    if (i == 0) {
      lo = held(lane.a_lo + parity);
      hi = held(lane.a_hi + parity);
    }
    a[i] = read_fragment(lo, hi, unit + 2048u * i);
  };
  auto read_b = [&](uint32_t parity, uint32_t unit, int which, int n, bool begin) {
    if (begin) {
      lo = held(lane.b_lo + parity);
      hi = held(lane.b_hi + parity);
    }
    b[which][n] = read_fragment(lo, hi, unit + 2048u * n);
  };
  // Scales of stage kt: rows of A half `half` (into set `set`), and the units' weights.  Read two phases ahead, so that their
  // wait is none for the fragments read since.
  auto read_x_scales = [&](int kt, int half, int set) {
    const uint32_t at = lane.x_scale + scales_of(kt) + half * 2048;
#pragma unroll
    for (int i = 0; i < 4; ++i) x_scale[set][i] = *(const GG_LDS float*)(uintptr_t)(at + 256u * i);
  };
  auto read_w_scales = [&](int kt) {
    const uint32_t at = lane.w_scale + scales_of(kt);
    w_next = *(const GG_LDS float*)(uintptr_t)at;
  };
  auto next_w_scales = [&]() {
    w_scale = w_next;
  };
  // The 8 instructions of (A half, B unit), rows first, columns back and forth; the sums of the two before last are brought
  // in behind each.  last_half, last_unit: of the phase before.
  auto phase = [&](int half, int unit, int last_half, int last_unit, auto&& issue, auto&& read) {
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = x_scale[half][i] * w_scale;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int i = r >> 1, n = (i & 1) != 0 ? 1 - (r & 1) : r & 1;
      part[r] = multiply(b[unit][n], a[i]);
      __builtin_amdgcn_sched_barrier(0);
      if (r < 2) {
        add_scaled(acc[last_half][3][last_unit][1 - r], left[r], left_scale);
      } else {
        const int q = r - 2, qi = q >> 1, qn = (qi & 1) != 0 ? 1 - (q & 1) : q & 1;
        add_scaled(acc[half][qi][unit][qn], part[q], scale[qi]);
      }
      read(r);
      issue(r);
      __builtin_amdgcn_sched_barrier(0);
    }
    left[0] = part[6];
    left[1] = part[7];
    left_scale = scale[3];
  };

  loader.issue_scales(0, scales_at);
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const uint32_t st = lds + kt * kParity;
#pragma unroll
    for (int i = 0; i < 2; ++i) loader.issue_b(kt, 0, st + kB0, i);
#pragma unroll
    for (int i = 0; i < 2; ++i) loader.issue_a(kt, 0, st + kA0, i);
#pragma unroll
    for (int i = 0; i < 2; ++i) loader.issue_b(kt, 1, st + kB1, i);
#pragma unroll
    for (int i = 0; i < 2; ++i) loader.issue_a(kt, 1, st + kA1, i);
  }
  gg::wait_vmcnt<6 * kLoads>();
  gg::phase_barrier();
#pragma unroll
  for (int n = 0; n < 2; ++n) read_b(0, kB0, 0, n, n == 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) read_a(0, kA0, i);
  read_x_scales(0, 0, 0);
  read_w_scales(0);
  next_w_scales();
  gg::wait_vmcnt<5 * kLoads>();
  gg::wait_lgkmcnt<0>();
  gg::phase_barrier();

  // One stage.  ISSUE: the loads of stage kt + 2 are issued; else everything has been and the waits count down.  LAST:
  // nothing more is read.
  auto stage = [&](int kt, auto issue_tag, auto last_tag) {
    constexpr bool ISSUE = decltype(issue_tag)::value, LAST = decltype(last_tag)::value;
    constexpr int N = kLoads;
    const uint32_t here = (uint32_t)(kt & 1) * kParity, next = kParity - here;
    const uint32_t st = lds + here;
    // Scales of the next four stages, behind the last use of the set before theirs.
    if ((kt & 3) == 0 && kt + kScaleSteps < nk) loader.issue_scales(kt / 4 + 1, scales_at + ((kt / 4 + 1) & 1) * kScales);
    phase(0, 0, 1, 1, [&](int r) { if (ISSUE && (r == 4 || r == 6)) loader.issue_b(kt + 2, 0, st + kB0, r / 2 - 2); },
          [&](int r) {
            if (r == 1 || r == 3) read_b(here, kB1, 1, r / 2, r == 1);
            if (r == 5) read_x_scales(kt, 1, 1);
          });
    gg::wait_vmcnt<ISSUE ? 5 * N : LAST ? 0 : 4 * N>();
    gg::phase_barrier();
    phase(0, 1, 0, 0, [&](int r) { if (ISSUE && (r == 4 || r == 6)) loader.issue_a(kt + 2, 0, st + kA0, r / 2 - 2); },
          [&](int r) { if (r & 1) read_a(here, kA1, r / 2); });
    if constexpr (!LAST) {
      gg::wait_vmcnt<ISSUE ? 5 * N : 3 * N>();
      gg::phase_barrier();
    }
    phase(1, 0, 0, 1, [&](int r) { if (ISSUE && (r == 4 || r == 6)) loader.issue_b(kt + 2, 1, st + kB1, r / 2 - 2); },
          [&](int r) {
            if constexpr (!LAST) {
              if (r == 1) {
                read_x_scales(kt + 1, 0, 0);
                read_w_scales(kt + 1);
              }
              if (r >= 6) read_b(next, kB0, 0, 7 - r, r == 6);
            }
          });
    if constexpr (!LAST) {
      gg::wait_vmcnt<ISSUE ? 5 * N : 2 * N>();
      gg::phase_barrier();
    }
    phase(1, 1, 1, 0, [&](int r) { if (ISSUE && (r == 4 || r == 6)) loader.issue_a(kt + 2, 1, st + kA1, r / 2 - 2); },
          [&](int r) { if constexpr (!LAST) { if (r & 1) read_a(next, kA0, r / 2); } });
    if constexpr (!LAST) {
      gg::wait_lgkmcnt<8>();  // phase 2's reads, which nothing has used yet; this phase's eight may be on their way
      next_w_scales();
      gg::wait_vmcnt<ISSUE ? 5 * N : N>();
      gg::phase_barrier();
    }
  };
  int kt = 0;
#pragma unroll 1
  for (; kt < nk - 2; ++kt) stage(kt, std::true_type{}, std::false_type{});
  if (nk >= 2) stage(kt++, std::false_type{}, std::false_type{});
  stage(kt, std::false_type{}, std::true_type{});  // a single stage also waits for the (empty) loads past K
  add_scaled(acc[1][3][1][1], left[0], left_scale);
  add_scaled(acc[1][3][1][0], left[1], left_scale);
  gg::wait_vmcnt<0>();
}

// Of a lane's four columns of two neighbouring 16s, what 16 bytes hold of one: lanes 16 apart trade (a row of y then gets 64
// bytes of an instruction, not 32).
template <class T>
struct Sixteen {
  typedef T Four __attribute__((ext_vector_type(4)));
  static constexpr bool kTrade = sizeof(T) == 2;
  uint4v v[kTrade ? 1 : 2];
  __device__ __forceinline__ Sixteen(const Four& a, const Four& b) {
    if constexpr (kTrade) {
      const uint2v p = __builtin_bit_cast(uint2v, a), q = __builtin_bit_cast(uint2v, b);
      const auto lo = __builtin_amdgcn_permlane16_swap(p.x, q.x, false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(p.y, q.y, false, false);
      v[0] = uint4v{lo[0], hi[0], lo[1], hi[1]};
    } else {
      v[0] = __builtin_bit_cast(uint4v, a);
      v[1] = __builtin_bit_cast(uint4v, b);
    }
  }
  // First column of v[i] for lanes g of a row.
  static __device__ __forceinline__ int column(int g, int i) { return kTrade ? 16 * (g & 1) + 8 * (g >> 1) : 16 * i + 4 * g; }
};

// y of a tile: 16 bytes a lane and store, wherever rows begin; the 16 bytes of a row that n cuts by way of LDS, value by value.
// (With all of a tile's rows by way of LDS where they do not begin on multiples of 16 bytes, 5076 slots of 16 experts of 288 by
// 2082 took 56 us, so 28.)
template <bool EXPERTS, class T, int HALVES>
__device__ __forceinline__ void store_tile(const ggk_fp8_args& a, const RowTile& t, const Shared& s, int n0, int wm, int wn,
                                           const Sums<HALVES>& acc) {
  using Four = typename Sixteen<T>::Four;
  constexpr int kEach = 16 / sizeof(T);
  const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
  const int columns = min(a.n - n0, 256), whole = columns / kEach * kEach;
  if (whole < columns) gg::stage_barrier();
#pragma unroll
  for (int half = 0; half < HALVES; ++half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 128 * half + 64 * wm + 16 * i + j;
      const int slot = r < t.rows ? (EXPERTS ? s.slot[r] : t.first + r) : -1;
      const float weight = EXPERTS && a.row_weights != nullptr && slot >= 0 ? a.row_weights[slot] : 1.0f;
      T* y = static_cast<T*>(a.y) + slot * a.ldy + n0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        Four four[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) four[n][e] = (T)(acc[half][i][u][n][e] * weight);
        }
        const Sixteen<T> part(four[0], four[1]);
#pragma unroll
        for (int n = 0; n < (int)(sizeof(part.v) / 16); ++n) {
          const int column = 64 * wn + 32 * u + Sixteen<T>::column(g, n);
          if (slot >= 0 && column < whole) *reinterpret_cast<gg::Any16*>(y + column) = part.v[n];
          if (whole < columns && column == whole) *reinterpret_cast<uint4v*>(s.stages + 16 * r) = part.v[n];
        }
      }
    }
  }
  if (whole < columns) {
    gg::stage_barrier();
    for (int i = threadIdx.x; i < t.rows * kEach; i += kThreads) {
      const int r = i / kEach, c = whole + i % kEach, slot = EXPERTS ? s.slot[r] : t.first + r;
      if (slot >= 0 && c < columns) {
        static_cast<T*>(a.y)[slot * a.ldy + n0 + c] = *reinterpret_cast<const T*>(s.stages + sizeof(T) * i);
      }
    }
  }
}

// The 8-bit rows of a gated tile, of 128 rows.
template <bool EXPERTS, bool GELU>
__device__ __forceinline__ void store_rows(const ggk_fp8_args& a, const RowTile& t, const Shared& s, int n0, int wm, int wn,
                                           Sums<1>& acc) {
  const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
  // Values stay in the registers of gate's sums; a row's 128 columns lie in 4 lanes of 4 waves.
  constexpr int kLd = 128 + 16;
  uint32_t* s_most = reinterpret_cast<uint32_t*>(s.stages + 128 * kLd);  // [128][4]
  gg::stage_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t most = 0;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = gated<GELU>(acc[0][i][0][n][e], acc[0][i][1][n][e]);
        if (n0 + 32 * wn + 16 * n + 4 * g + e >= a.n) v = 0.0f;
        acc[0][i][0][n][e] = v;
        most = max(most, gg::magnitude_bits(v));
      }
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
    if (g == 0) s_most[(64 * wm + 16 * i + j) * 4 + wn] = most;
  }
  gg::stage_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 64 * wm + 16 * i + j;
    const uint4v most = *reinterpret_cast<const uint4v*>(&s_most[r * 4]);
    const uint32_t largest = max(max(most.x, most.y), max(most.z, most.w));
    const float scale = gg::fp8_scale(largest);
    const gg::Fp8Divisor by(scale, __builtin_bit_cast(float, largest));
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float4v v = acc[0][i][0][n];
      *reinterpret_cast<uint32_t*>(s.stages + r * kLd + 32 * wn + 16 * n + 4 * g) =
          gg::fp8_numbers(v[0], v[1], v[2], v[3], by);
    }
    if (wn == 0 && g == 0 && r < t.rows) {
      const int slot = EXPERTS ? s.slot[r] : t.first + r;
      if (slot >= 0) a.y_scales[slot * a.ldys + n0 / kStep] = scale;
    }
  }
  gg::stage_barrier();
  const int tid = threadIdx.x;
  for (int i = tid; i < t.rows * 8; i += kThreads) {
    const int r = i / 8, column = n0 + i % 8 * 16, slot = EXPERTS ? s.slot[r] : t.first + r;
    if (slot < 0 || column >= a.n) continue;
    const unsigned char* from = s.stages + r * kLd + i % 8 * 16;
    unsigned char* y = static_cast<unsigned char*>(a.y) + slot * a.ldy + column;
    if (column + 16 <= a.n) {
      *reinterpret_cast<gg::Any16*>(y) = *reinterpret_cast<const uint4v*>(from);
    } else {
      for (int c = 0; c < 16 && column + c < a.n; ++c) y[c] = from[c];
    }
  }
}

template <bool EXPERTS, bool GATED, bool EXACT, int HALVES>
__device__ __forceinline__ void run_tile(const Launch& l, const RowTile& t, const Shared& s, int n0) {
  const ggk_fp8_args& a = l.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave >> 2, wn = wave & 3;
  Sums<HALVES> acc;
  if constexpr (EXACT) {
    multiply_tile_exact<EXPERTS, GATED>(l, t, s, n0, wave, acc);
  } else {
    multiply_tile<EXPERTS>(l, t, s, n0, wave, acc);
  }
  if constexpr (GATED) {
    if (a.gate == GGK_GATE_GELU) {
      store_rows<EXPERTS, true>(a, t, s, n0, wm, wn, acc);
    } else {
      store_rows<EXPERTS, false>(a, t, s, n0, wm, wn, acc);
    }
  } else if (EXACT && a.y_type == GGK_TYPE_F32) {
    store_tile<EXPERTS, float, HALVES>(a, t, s, n0, wm, wn, acc);
  } else if (a.y_type == GGK_TYPE_BF16) {
    store_tile<EXPERTS, __bf16, HALVES>(a, t, s, n0, wm, wn, acc);
  } else {
    store_tile<EXPERTS, _Float16, HALVES>(a, t, s, n0, wm, wn, acc);
  }
}

template <bool EXPERTS, bool GATED, bool EXACT>
__device__ __forceinline__ void run_either(const Launch& l, const RowTile& t, const Shared& s, int n0) {
  if constexpr (EXACT) {
    run_tile<EXPERTS, GATED, true, 1>(l, t, s, n0);
  } else if (t.rows <= kRows / 2) {
    run_tile<EXPERTS, GATED, false, 1>(l, t, s, n0);
  } else {
    run_tile<EXPERTS, GATED, false, 2>(l, t, s, n0);
  }
}

// Rows without an expert.
template <bool GATED>
__device__ __forceinline__ void clear_row(const ggk_fp8_args& a, int slot) {
  if (slot < 0 || slot >= a.rows) return;
  for (int column = threadIdx.x; column < a.n; column += kThreads) {
    if constexpr (GATED) {
      static_cast<unsigned char*>(a.y)[slot * a.ldy + column] = 0;
      if (column % kStep == 0) a.y_scales[slot * a.ldys + column / kStep] = gg::kFp8SmallestScale;
    } else {
      store_value(a.y, a.y_type, slot * a.ldy + column, 0.0f);
    }
  }
}

// Row tile and column block of place p in an order that goes along the columns kGroup row tiles at a time, so that the
// workgroups of an XCD share both; each column block begins with another of them, so that a workgroup meets all.
__device__ __forceinline__ void place(long long p, int tiles, int blocks, int* tile, int* block) {
  const long long group = p / ((long long)kGroup * blocks);
  const int in = (int)(p - group * kGroup * blocks), height = min(kGroup, tiles - (int)group * kGroup);
  *block = in / height;
  *tile = (int)group * kGroup + (in % height + *block) % height;
}

// Experts' rows as tiles: whole ones of more than 128 rows, and a rest of at most 128 where there is one.
constexpr int kWhole = 20, kRest = 11;  // what a tile costs: a stage of each, measured on a full chip

template <int MOST>
struct Tiles {
  int first[MOST + 2];  // places in the order, as in Experts; rows without an expert last
  int tile[MOST + 1];   // tiles of the experts before, and of all
  int cost[MOST + 1];   // and what they cost
  int waves[32];
};

__device__ __forceinline__ int whole_tiles(const Launch& l, int rows) {
  return l.height == kRows ? (rows + kRows / 2 - 1) / kRows : 0;
}
__device__ __forceinline__ int tiles_of(const Launch& l, int rows) { return (rows + l.height - 1) / l.height; }

template <class Table>
__device__ __forceinline__ void list_tiles(const Launch& l, Table& s) {
  const ggk_fp8_args& a = l.a;
  int placed = 0, tiles = 0, cost = 0;
  for (int e0 = 0; e0 < a.experts; e0 += kThreads) {
    const int e = e0 + threadIdx.x;
    const int count = e < a.experts ? min(max(a.counts[e], 0), a.rows) : 0;
    int all, all_tiles, all_cost;
    const int first = gg::add_up_to(gg::block_before<kThreads>(count, a.rows, s.waves, &all), placed, a.rows);
    const int rows = min(count, a.rows - first), mine = tiles_of(l, rows), whole = whole_tiles(l, rows);
    const int at_tile = gg::block_before<kThreads>(mine, 0x3fffffff, s.waves, &all_tiles) + tiles;
    const int at_cost = gg::block_before<kThreads>(kWhole * whole + kRest * (mine - whole), 0x3fffffff, s.waves, &all_cost) + cost;
    if (e < a.experts) {
      s.first[e] = first;
      s.tile[e] = at_tile;
      s.cost[e] = at_cost;
    }
    placed = gg::add_up_to(placed, all, a.rows);
    tiles += all_tiles;
    cost += all_cost;
  }
  if (threadIdx.x == 0) {
    s.first[a.experts] = placed;
    s.first[a.experts + 1] = a.rows;
    s.tile[a.experts] = tiles;
    s.cost[a.experts] = cost;
  }
  __syncthreads();
}

// Last of a rising table's a.experts entries (times `by`) that is at most v; the first is 0.
__device__ __forceinline__ int find_expert(const ggk_fp8_args& a, const int* table, long long by, long long v) {
  const int lane = threadIdx.x % kWave;
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += kWave) {
    before += __popcll(__ballot(e0 + lane < a.experts && table[min(e0 + lane, a.experts)] * by <= v));
  }
  return before - 1;
}

// First item, of those that begin a column block of a group, at cost `at` of all or after it.
template <class Table>
__device__ __forceinline__ long long item_at(const Launch& l, const Table& s, long long at) {
  const ggk_fp8_args& a = l.a;
  const int blocks = l.blocks;
  const int e = find_expert(a, s.cost, blocks, at), rows = s.first[e + 1] - s.first[e];
  const int each = l.height == kRows ? kWhole : kRest;  // of the tiles of every group but the last
  const int tiles = tiles_of(l, rows), groups = (tiles + kGroup - 1) / kGroup;
  long long left = at - (long long)s.cost[e] * blocks, item = (long long)s.tile[e] * blocks;
  const int group = (int)min(left / (kGroup * each * (long long)blocks), (long long)groups - 1);
  left -= (long long)group * kGroup * each * blocks;
  item += (long long)group * kGroup * blocks;
  const int cost = group < groups - 1 ? kGroup * each : s.cost[e + 1] - s.cost[e] - group * kGroup * each;
  return item + (left + cost - 1) / cost * min(kGroup, tiles - group * kGroup);
}

template <bool EXPERTS, bool GATED, bool EXACT>
__global__ __launch_bounds__(kThreads, 2) void fp8_tile_kernel(Launch l) {
  const ggk_fp8_args& a = l.a;
  __shared__ alignas(128) unsigned char s_stages[kPlaces * kUnit + 2 * kScales];
  __shared__ int s_slot[EXPERTS ? kRows : 1];
  const Shared s{s_stages, s_slot};
  // Neighbouring workgroups go to different XCDs, each with an L2 of its own: an XCD takes a run of the order, an eighth of
  // the items or of what they cost.
  const int xcd = blockIdx.x % kXcds, in_xcd = blockIdx.x / kXcds;
  if constexpr (!EXPERTS) {
    const int tiles = (a.rows + l.height - 1) / l.height;
    const long long items = (long long)tiles * l.blocks, share = (items + kXcds - 1) / kXcds;
    const long long end = min((xcd + 1) * share, items);
    for (long long item = xcd * share + in_xcd; item < end; item += kCus / kXcds) {
      int tile, block;
      place(item, tiles, l.blocks, &tile, &block);
      const RowTile t{0, tile * l.height, min(l.height, a.rows - tile * l.height)};
      run_either<false, GATED, EXACT>(l, t, s, block * kColumns<GATED>);
      gg::stage_barrier();
    }
  } else {
    __shared__ Tiles<kMost> s_tiles;
    list_tiles(l, s_tiles);
    const long long cost = (long long)s_tiles.cost[a.experts] * l.blocks, items = (long long)s_tiles.tile[a.experts] * l.blocks;
    const long long end = xcd + 1 < kXcds && cost > 0 ? item_at(l, s_tiles, cost * (xcd + 1) / kXcds) : items;
    const long long begin = xcd > 0 && cost > 0 ? item_at(l, s_tiles, cost * xcd / kXcds) : 0;
    for (long long item = begin + in_xcd; item < end; item += kCus / kXcds) {
      const int e = find_expert(a, s_tiles.tile, l.blocks, item), rows = s_tiles.first[e + 1] - s_tiles.first[e];
      int tile, block;
      place(item - (long long)s_tiles.tile[e] * l.blocks, tiles_of(l, rows), l.blocks, &tile, &block);
      const RowTile t{e, s_tiles.first[e] + tile * l.height, min(l.height, rows - tile * l.height)};
      for (int r = threadIdx.x; r < t.rows; r += kThreads) {
        const int slot = a.order[t.first + r];
        s_slot[r] = slot < a.rows ? slot : -1;
      }
      gg::stage_barrier();
      run_either<true, GATED, EXACT>(l, t, s, block * kColumns<GATED>);
      gg::stage_barrier();
    }
    // Rows without an expert.
    for (int at = s_tiles.first[a.experts] + blockIdx.x; at < a.rows; at += kCus) clear_row<GATED>(a, a.order[at]);
  }
}

template <bool EXPERTS, bool GATED, bool EXACT>
hipError_t launch(const ggk_fp8_args& a, int height, hipStream_t stream) {
  Launch l{a, (a.n + kColumns<GATED> - 1) / kColumns<GATED>, height, a.rows / a.x_rows, 0};
  if (EXPERTS) l.scale_bytes = (uint32_t)(((a.x_rows - 1) * a.ldxs + (a.k + kStep - 1) / kStep) * 4);
  hipLaunchKernelGGL((fp8_tile_kernel<EXPERTS, GATED, EXACT>), dim3(kCus), dim3(kThreads), 0, stream, l);
  return hipGetLastError();
}

template <bool EXPERTS>
hipError_t launch(const ggk_fp8_args& a, int height, hipStream_t stream) {
  if (a.gate != GGK_GATE_NONE) return launch<EXPERTS, true, true>(a, height, stream);
  return is_exact(a) ? launch<EXPERTS, false, true>(a, height, stream) : launch<EXPERTS, false, false>(a, height, stream);
}

// What a call takes on tiles of `height` rows, in us: what the busiest CU gets; of experts' tiles, whose counts the host does
// not know, a tenth more.  A stage of a tile of 256 rows takes 1.2 us where half of the CUs work and 1.7 where all do, one of 128
// rows 0.7 and 0.95 (0.62 where few work), in binary16 1.6 and 1.75, gated 1.75.
double estimate(const ggk_fp8_args& a, int height) {
  const bool gate = a.gate != GGK_GATE_NONE;
  const double columns = gate ? 128 : 256, stages = (a.k + kStep - 1) / kStep;
  const double of_a_cu = row_tiles(a, height) * ceil(a.n / columns) * (a.experts > 0 ? 1.1 : 1) / kCus, rounds = ceil(of_a_cu);
  const double at_work = of_a_cu / rounds;
  const double of_128 = at_work < 0.34 ? 0.62 : 0.45 + 0.5 * at_work;
  const double of_exact = gate ? 1.75 : 1.55 + 0.2 * at_work;
  const double stage = is_exact(a) ? of_exact : height == kRows ? 0.9 + 0.8 * at_work : of_128;
  return (a.experts > 0 ? 10 : 8) + rounds * (stage * stages + (gate ? 4 : 2));
}

// Tiles of 256 rows or of 128.  us of the two, by the 8-bit instructions: 1024 rows of 8192 by 8192 86, 65, 1280 90, 107, 8192 453, 522; 1500 of 4096 by
// 4096 46, 30.  Experts' tiles of 256 rows, with a rest of 128 and less each, where those of 128 would not fit the CUs at once:
// 64 experts of 4096 by 14336, 16384 slots 1338, 1438, 16 of 1024 by 2048, 2048 slots 20, 18.  In binary16 the registers hold 128.
int height_of(const ggk_fp8_args& a) {
  if (is_exact(a)) return kRows / 2;
  const bool small = a.experts > 0 ? row_tiles(a, kRows / 2) * ceil(a.n / 256.0) <= kCus : estimate(a, kRows / 2) < estimate(a, kRows);
  return small ? kRows / 2 : kRows;
}

}  // namespace

namespace gg {
namespace fp8 {

bool tiles_take(const ggk_fp8_args& a) {
  // Offsets from the tile's first row (experts: from x) are 32 bits.
  const long long rows = a.experts > 0 ? a.x_rows : kRows;
  return a.experts <= kMost && rows * a.ldx < 0xfffffff0ll - kStep && rows * a.ldxs * 4 < 0x7fffffffll;
}

double estimate_tiles(const ggk_fp8_args& a) { return estimate(a, a.experts > 0 ? kRows / 2 : height_of(a)); }

int tile_rows(const ggk_fp8_args& a) { return height_of(a); }

hipError_t multiply_tiles(const ggk_fp8_args& a, hipStream_t stream) {
  return a.experts > 0 ? launch<true>(a, height_of(a), stream) : launch<false>(a, height_of(a), stream);
}

}  // namespace fp8
}  // namespace gg
