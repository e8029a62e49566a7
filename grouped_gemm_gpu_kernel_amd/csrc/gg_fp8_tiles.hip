// gg_fp8_tiles.hip -- products of many rows with matrices of 8-bit numbers, one
// matrix or one an expert, plain or gated, on 256 x 256 tiles.
//
// A workgroup of 8 waves (2 x 4) computes 256 rows of x by 256 columns (with a gate: 128 of gate and the same 128 of up).
// A stage is one block of K, 128 bytes of each row, in four units of 16 KB in the order the loop reads them:
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
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gg_experts.h"
#include "gg_fp8.h"
#include "gg_phased.h"  // wait_lgkmcnt, phase_barrier

namespace {

using namespace gg::fp8;
using gg::Experts;
using gg::RowTile;
using gg::kWave;

constexpr int kCus = 256, kXcds = 8;
constexpr int kRows = 256, kWaves = 8, kThreads = kWaves * kWave;
constexpr int kUnit = 128 * kStep;  // bytes
constexpr int kB0 = 0, kA0 = kUnit, kB1 = 2 * kUnit, kA1 = 3 * kUnit, kParity = 4 * kUnit;
constexpr int kLoads = 2;           // load instructions of a unit and wave
constexpr int kScaleSteps = 4;      // stages of scales loaded at once, 16 bytes a row
constexpr int kScales = 6 * 1024;   // bytes of those: 256 rows, and a row of each unit's weights in 1 KB each
constexpr int kGroup = 4;           // row tiles that go along the columns together

template <bool GATED>
constexpr int kColumns = GATED ? 128 : 256;

struct Launch {
  ggk_fp8_args a;
  int blocks;            // of columns
  uint32_t scale_bytes;  // of all of x's scales (experts)
};

struct Shared {
  unsigned char* stages;  // two stages, then two sets of scales
  int* slot;              // of the tile's rows, -1 for none
  int* x_row;
};

// Sums of one tile: [rows half][16 rows][unit of columns][16 columns].
typedef float4v Sums[2][4][2][2];

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

  __device__ __forceinline__ Loader(const Launch& l, const RowTile& t, const int* x_row, int n0, int wave_)
      : a(l.a), wave(wave_) {
    const int tid = gg::opaque_tid(wave), row = tid / 8;
    const int piece = (tid & 7) ^ (row >> 1 & 7);
    piece16 = 16 * piece;
    x0 = EXPERTS ? a.x : a.x + t.first * a.ldx;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = min(128 * half + 64 * i + row, t.rows - 1);
        a_off[half][i] = (uint32_t)((EXPERTS ? x_row[r] : r) * a.ldx) + piece16;
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
    const int lane = tid % kWave;
    const int blocks_k = (a.k + kStep - 1) / kStep;
    if (wave < 4) {
      const int r = min(tid, t.rows - 1);
      s0 = EXPERTS ? a.x_scales : a.x_scales + t.first * a.ldxs;
      s_off = (uint32_t)((EXPERTS ? x_row[r] : r) * a.ldxs * 4);
      s_records = EXPERTS ? l.scale_bytes : (uint32_t)(((t.rows - 1) * a.ldxs + blocks_k) * 4);
    } else {
      const int block = n0 / kStep, unit = wave & 1;
      if (GATED && unit == 1) {
        s0 = a.up_scales + t.expert * a.stride_us + block * a.ldus;
      } else {
        const int at = min(block + (GATED ? 0 : unit), (a.n - 1) / kStep);
        s0 = a.w_scales + t.expert * a.stride_ws + at * a.ldws;
      }
      s_off = lane == 0 ? 0 : kOutOfRange;
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
    if (wave >= 6) return;
    const uint32_t skip = 4 * kScaleSteps * chunk;
    gg::load_to_lds16(s0 + kScaleSteps * chunk, s_records - skip, scales + 1024u * (uint32_t)wave, s_off, 0);
  }
};

// The sums of the tile at rows t, columns n0 on.
template <bool EXPERTS, bool GATED>
__device__ __forceinline__ void multiply_tile(const Launch& l, const RowTile& t, const Shared& s, int n0, int wave, Sums& acc) {
  const ggk_fp8_args& p = l.a;
  const int nk = (p.k + kStep - 1) / kStep;
  const Loader<EXPERTS, GATED> loader(l, t, s.x_row, n0, wave);
  const uint32_t lds = gg::lds_address(s.stages), scales_at = lds + 2 * kParity;
  const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
  const int wm = wave >> 2, wn = wave & 3;
  const uint32_t lane_at = (uint32_t)(j * 128 + ((g ^ (j >> 1)) & 7) * 16);
  const uint32_t a_lane = lds + lane_at + wm * 64 * 128, b_lane = lds + lane_at + wn * 32 * 128;
  const uint32_t x_scale_lane = scales_at + (wm * 64 + j) * 16;
  const uint32_t w_scale_lane = scales_at + 4096 + (GATED ? 0 : (wn >> 1) * 1024);

  int8v a[4], b[2][2];
  float x_scale[4], w_scale[2];
  float4v part[8];      // results of this phase's instructions, three of them alive
  float4v left[2];      // of the phase before, its last two
  float left_scale;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[h][i][u][n] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
  }
  left[0] = left[1] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  left_scale = 0.0f;

  auto read_a = [&](uint32_t unit, int i) { a[i] = read_fragment(a_lane + unit + 2048u * i); };
  auto read_b = [&](uint32_t unit, int which, int n) { b[which][n] = read_fragment(b_lane + unit + 2048u * n); };
  // Scales of stage kt: rows of A half `half`, and the units' weights.
  auto read_x_scales = [&](int kt, int half) {
    const uint32_t at = x_scale_lane + ((kt >> 2) & 1) * kScales + (kt & 3) * 4 + half * 2048;
#pragma unroll
    for (int i = 0; i < 4; ++i) x_scale[i] = *(const GG_LDS float*)(uintptr_t)(at + 256u * i);
  };
  auto read_w_scales = [&](int kt) {
    const uint32_t at = w_scale_lane + ((kt >> 2) & 1) * kScales + (kt & 3) * 4;
    w_scale[0] = *(const GG_LDS float*)(uintptr_t)at;
    if constexpr (GATED) w_scale[1] = *(const GG_LDS float*)(uintptr_t)(at + 1024u);
  };
  auto add = [&](float4v& sum, const float4v& v, float scale) {
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = fmaf(scale, v[e], sum[e]);
  };
  // The 8 instructions of (A half, B unit), rows first, columns back and forth; the sums of the two before last are brought
  // in behind each.  last_half, last_unit: of the phase before.
  auto phase = [&](int half, int unit, int last_half, int last_unit, auto&& issue, auto&& read) {
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = x_scale[i] * w_scale[GATED ? unit : 0];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int i = r >> 1, n = (i & 1) != 0 ? 1 - (r & 1) : r & 1;
      part[r] = multiply(b[unit][n], a[i]);
      __builtin_amdgcn_sched_barrier(0);
      if (r < 2) {
        add(acc[last_half][3][last_unit][1 - r], left[r], left_scale);
      } else {
        const int q = r - 2, qi = q >> 1, qn = (qi & 1) != 0 ? 1 - (q & 1) : q & 1;
        add(acc[half][qi][unit][qn], part[q], scale[qi]);
      }
      read(r);
      if (r == 4) issue(0);
      if (r == 6) issue(1);
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
  for (int n = 0; n < 2; ++n) read_b(kB0, 0, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) read_a(kA0, i);
  read_x_scales(0, 0);
  read_w_scales(0);
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
    phase(0, 0, 1, 1, [&](int i) { if constexpr (ISSUE) loader.issue_b(kt + 2, 0, st + kB0, i); },
          [&](int r) { if (r == 1 || r == 3) read_b(here + kB1, 1, r / 2); });
    gg::wait_lgkmcnt<0>();
    gg::wait_vmcnt<ISSUE ? 5 * N : LAST ? 0 : 4 * N>();
    gg::phase_barrier();
    phase(0, 1, 0, 0, [&](int i) { if constexpr (ISSUE) loader.issue_a(kt + 2, 0, st + kA0, i); },
          [&](int r) { if (r & 1) read_a(here + kA1, r / 2); });
    read_x_scales(kt, 1);
    if constexpr (!LAST) {
      gg::wait_vmcnt<ISSUE ? 5 * N : 3 * N>();
      gg::phase_barrier();
    }
    phase(1, 0, 0, 1, [&](int i) { if constexpr (ISSUE) loader.issue_b(kt + 2, 1, st + kB1, i); },
          [&](int r) { if constexpr (!LAST) { if (r >= 6) read_b(next + kB0, 0, 7 - r); } });
    if constexpr (!LAST) {
      gg::wait_vmcnt<ISSUE ? 5 * N : 2 * N>();
      gg::phase_barrier();
    }
    phase(1, 1, 1, 0, [&](int i) { if constexpr (ISSUE) loader.issue_a(kt + 2, 1, st + kA1, i); },
          [&](int r) { if constexpr (!LAST) { if (r & 1) read_a(next + kA0, r / 2); } });
    if constexpr (!LAST) {
      gg::wait_lgkmcnt<8>();  // phase 2's reads, which nothing has used yet; this phase's eight may be on their way
      read_x_scales(kt + 1, 0);
      read_w_scales(kt + 1);
      gg::wait_vmcnt<ISSUE ? 5 * N : N>();
      gg::phase_barrier();
    }
  };
  int kt = 0;
#pragma unroll 1
  for (; kt < nk - 2; ++kt) stage(kt, std::true_type{}, std::false_type{});
  if (nk >= 2) stage(kt++, std::false_type{}, std::false_type{});
  stage(kt, std::false_type{}, std::true_type{});  // a single stage also waits for the (empty) loads past K
  add(acc[1][3][1][1], left[0], left_scale);
  add(acc[1][3][1][0], left[1], left_scale);
  gg::wait_vmcnt<0>();
}

// y of a tile, in a 16-bit type.
template <bool EXPERTS, class T>
__device__ __forceinline__ void store_tile(const ggk_fp8_args& a, const RowTile& t, const Shared& s, int n0, int wm, int wn,
                                           const Sums& acc) {
  const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
  const bool vec = a.n % 4 == 0 && a.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % 8 == 0;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 128 * half + 64 * wm + 16 * i + j;
      const int slot = r < t.rows ? (EXPERTS ? s.slot[r] : t.first + r) : -1;
      const float weight = EXPERTS && a.row_weights != nullptr && slot >= 0 ? a.row_weights[slot] : 1.0f;
      T* y = static_cast<T*>(a.y) + slot * a.ldy;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int column = n0 + 64 * wn + 32 * u + 16 * n + 4 * g;
          uint16_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = __builtin_bit_cast(uint16_t, (T)(acc[half][i][u][n][e] * weight));
          if (slot < 0) continue;
          if (vec) {
            if (column < a.n) {
              *reinterpret_cast<uint2v*>(y + column) = uint2v{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (column + e < a.n) reinterpret_cast<uint16_t*>(y)[column + e] = h[e];
            }
          }
        }
      }
    }
  }
}

// The 8-bit rows of a gated tile.
template <bool EXPERTS, bool GELU>
__device__ __forceinline__ void store_rows(const ggk_fp8_args& a, const RowTile& t, const Shared& s, int n0, int wm, int wn,
                                           Sums& acc) {
  const int lane = gg::opaque_lane(), g = lane >> 4, j = lane & 15;
      // Values stay in the registers of gate's sums; a row's 128 columns lie in 4 lanes of 4 waves.
      constexpr int kLd = 128 + 16;
      uint32_t* s_most = reinterpret_cast<uint32_t*>(s.stages + kRows * kLd);  // [256][4]
      gg::stage_barrier();
  #pragma unroll
      for (int half = 0; half < 2; ++half) {
  #pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t most = 0;
  #pragma unroll
          for (int n = 0; n < 2; ++n) {
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = gated<GELU>(acc[half][i][0][n][e], acc[half][i][1][n][e]);
              if (n0 + 32 * wn + 16 * n + 4 * g + e >= a.n) v = 0.0f;
              acc[half][i][0][n][e] = v;
              most = max(most, gg::magnitude_bits(v));
            }
          }
          most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
          most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
          if (g == 0) s_most[(128 * half + 64 * wm + 16 * i + j) * 4 + wn] = most;
        }
      }
      gg::stage_barrier();
  #pragma unroll
      for (int half = 0; half < 2; ++half) {
  #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 128 * half + 64 * wm + 16 * i + j;
          const uint4v most = *reinterpret_cast<const uint4v*>(&s_most[r * 4]);
          const float scale = gg::fp8_scale(max(max(most.x, most.y), max(most.z, most.w)));
          const gg::Fp8Divisor by(scale);
  #pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float4v v = acc[half][i][0][n];
            *reinterpret_cast<uint32_t*>(s.stages + r * kLd + 32 * wn + 16 * n + 4 * g) =
                gg::fp8_numbers(v[0], v[1], v[2], v[3], by);
          }
          if (wn == 0 && g == 0 && r < t.rows) {
            const int slot = EXPERTS ? s.slot[r] : t.first + r;
            if (slot >= 0) a.y_scales[slot * a.ldys + n0 / kStep] = scale;
          }
        }
      }
      gg::stage_barrier();
      const int tid = threadIdx.x;
      for (int i = tid; i < t.rows * 8; i += kThreads) {
        const int r = i / 8, column = n0 + i % 8 * 16, slot = EXPERTS ? s.slot[r] : t.first + r;
        if (slot < 0 || column >= a.n) continue;
        const unsigned char* from = s.stages + r * kLd + i % 8 * 16;
        unsigned char* y = static_cast<unsigned char*>(a.y) + slot * a.ldy + column;
        if (column + 16 <= a.n && reinterpret_cast<uintptr_t>(y) % 16 == 0) {
          *reinterpret_cast<uint4v*>(y) = *reinterpret_cast<const uint4v*>(from);
        } else {
          for (int c = 0; c < 16 && column + c < a.n; ++c) y[c] = from[c];
        }
      }
}

template <bool EXPERTS, bool GATED>
__device__ __forceinline__ void run_tile(const Launch& l, const RowTile& t, const Shared& s, int n0) {
  const ggk_fp8_args& a = l.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave >> 2, wn = wave & 3;
  Sums acc;
  multiply_tile<EXPERTS, GATED>(l, t, s, n0, wave, acc);
  if constexpr (!GATED) {
    if (a.y_type == GGK_TYPE_BF16) {
      store_tile<EXPERTS, __bf16>(a, t, s, n0, wm, wn, acc);
    } else {
      store_tile<EXPERTS, _Float16>(a, t, s, n0, wm, wn, acc);
    }
  } else {
    if (a.gate == GGK_GATE_GELU) {
      store_rows<EXPERTS, true>(a, t, s, n0, wm, wn, acc);
    } else {
      store_rows<EXPERTS, false>(a, t, s, n0, wm, wn, acc);
    }
  }
}

// Rows without an expert.
template <bool GATED>
__device__ __forceinline__ void clear_tile(const ggk_fp8_args& a, const RowTile& t, const int* slots, int n0) {
  for (int i = threadIdx.x; i < t.rows * kColumns<GATED>; i += kThreads) {
    const int slot = slots[i / kColumns<GATED>], column = n0 + i % kColumns<GATED>;
    if (column >= a.n || slot < 0) continue;
    if constexpr (GATED) {
      static_cast<unsigned char*>(a.y)[slot * a.ldy + column] = 0;
      if (column % kStep == 0) a.y_scales[slot * a.ldys + column / kStep] = gg::kFp8SmallestScale;
    } else {
      store_value(a.y, a.y_type, slot * a.ldy + column, 0.0f);
    }
  }
}

// Tile and column block of place p in an order that goes along the columns kGroup row tiles at a time.
__device__ __forceinline__ void place(long long p, int tiles, int blocks, int* tile, int* block) {
  const long long group = p / ((long long)kGroup * blocks);
  const int in = (int)(p - group * kGroup * blocks), height = min(kGroup, tiles - (int)group * kGroup);
  *tile = (int)group * kGroup + in % height;
  *block = in / height;
}

template <bool EXPERTS, bool GATED>
__global__ __launch_bounds__(kThreads, 2) void fp8_tile_kernel(Launch l) {
  const ggk_fp8_args& a = l.a;
  __shared__ alignas(128) unsigned char s_stages[2 * kParity + 2 * kScales];
  __shared__ int s_slot[EXPERTS ? kRows : 1], s_x_row[EXPERTS ? kRows : 1];
  __shared__ Experts<EXPERTS ? GGK_MOE_MAX_EXPERTS : 1> s_experts;
  const Shared s{s_stages, s_slot, s_x_row};
  int tiles = (a.rows + kRows - 1) / kRows;
  if constexpr (EXPERTS) {
    gg::list_experts<kThreads, kRows>(a, s_experts);
    tiles = s_experts.tile[a.experts + 1];
  }
  // Neighbouring workgroups go to different XCDs, each with an L2 of its own: an XCD takes a run of the order.
  const long long items = (long long)tiles * l.blocks, share = (items + kXcds - 1) / kXcds;
  const long long first = blockIdx.x % kXcds * share, end = min(first + share, items);
  const int fan = EXPERTS ? a.rows / a.x_rows : 1;
  for (long long item = first + blockIdx.x / kXcds; item < end; item += gridDim.x / kXcds) {
    int tile, block;
    place(item, tiles, l.blocks, &tile, &block);
    const int n0 = block * kColumns<GATED>;
    if constexpr (!EXPERTS) {
      const RowTile t{0, tile * kRows, min(kRows, a.rows - tile * kRows)};
      run_tile<false, GATED>(l, t, s, n0);
    } else {
      const RowTile t = gg::expert_tile<kRows>(a, s_experts, tile);
      for (int i = threadIdx.x; i < t.rows; i += kThreads) {
        int slot = a.order[t.first + i];
        if (slot >= a.rows) slot = -1;
        s_slot[i] = slot;
        s_x_row[i] = max(slot, 0) / fan;  // where a slot names no row, row 0: its sums are not used
      }
      gg::stage_barrier();
      if (t.expert == a.experts) {
        clear_tile<GATED>(a, t, s_slot, n0);
      } else {
        run_tile<true, GATED>(l, t, s, n0);
      }
    }
    gg::stage_barrier();
  }
}

template <bool EXPERTS, bool GATED>
hipError_t launch(const ggk_fp8_args& a, hipStream_t stream) {
  Launch l{a, (a.n + kColumns<GATED> - 1) / kColumns<GATED>, 0};
  if (EXPERTS) l.scale_bytes = (uint32_t)(((a.x_rows - 1) * a.ldxs + (a.k + kStep - 1) / kStep) * 4);
  hipLaunchKernelGGL((fp8_tile_kernel<EXPERTS, GATED>), dim3(kCus), dim3(kThreads), 0, stream, l);
  return hipGetLastError();
}

}  // namespace

namespace gg {
namespace fp8 {

bool tiles_take(const ggk_fp8_args& a) {
  // Offsets from the tile's first row (experts: from x) are 32 bits.
  const long long rows = a.experts > 0 ? a.x_rows : kRows;
  return rows * a.ldx < 0xfffffff0ll - kStep && rows * a.ldxs * 4 < 0x7fffffffll;
}

hipError_t multiply_tiles(const ggk_fp8_args& a, hipStream_t stream) {
  if (a.experts > 0) return a.gate != GGK_GATE_NONE ? launch<true, true>(a, stream) : launch<true, false>(a, stream);
  return a.gate != GGK_GATE_NONE ? launch<false, true>(a, stream) : launch<false, false>(a, stream);
}

}  // namespace fp8
}  // namespace gg
