// gg_w4.hip -- products of a few rows with 4-bit weights, one matrix or one an
// expert:
//
//   y[i][j] = sum_g scales[j][g] * sum_{k in g} x[i][k] * (q[j][k] - zeros[j][g])
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grouped_gemm_amd_kernels.h"

namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kRowTile = 8;  // rows of y a wave computes at once

__device__ __forceinline__ float wave_sum(float v) {
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
  return v;
}

// The row tiles of a launch: tile index -> expert (a.experts: the slots past the counts, which are set to 0),
// first place in the order and rows.  Every wave finds its own.
struct RowTile {
  int expert, first, rows;
};

__device__ RowTile find_tile(const ggk_w4_args& a, long long tile, long long* tiles) {
  const int lane = threadIdx.x % kWave;
  RowTile found{-1, 0, 0};
  long long tiles_before = 0;
  long long places_before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += kWave) {
    const int e = e0 + lane;
    const int count = e < a.experts ? max(a.counts[e], 0) : 0;
    long long places = count;
    for (int d = 1; d < kWave; d *= 2) {
      const long long other = __shfl_up(places, d, kWave);
      if (lane >= d) places += other;
    }
    const long long begin = min((long long)a.rows, places_before + places - count);
    const long long end = min((long long)a.rows, places_before + places);
    const int rows = (int)(end - begin);
    const long long mine = (rows + kRowTile - 1) / kRowTile;
    long long sum = mine;
    for (int d = 1; d < kWave; d *= 2) {
      const long long other = __shfl_up(sum, d, kWave);
      if (lane >= d) sum += other;
    }
    const long long at = tile - (tiles_before + sum - mine);
    const unsigned long long here = __ballot(at >= 0 && at < mine);
    if (here != 0) {
      const int src = __builtin_ctzll(here);
      const int first = (int)(begin + at * kRowTile);
      found.expert = __shfl(e, src, kWave);
      found.first = __shfl(first, src, kWave);
      found.rows = __shfl(min(kRowTile, (int)end - first), src, kWave);
    }
    places_before += __shfl(places, kWave - 1, kWave);
    tiles_before += __shfl(sum, kWave - 1, kWave);
  }
  const int placed = (int)min((long long)a.rows, places_before);
  const long long rest = (a.rows - placed + kRowTile - 1) / kRowTile;
  const long long at = tile - tiles_before;
  if (at >= 0 && at < rest) {
    found.expert = a.experts;
    found.first = (int)(placed + at * kRowTile);
    found.rows = min(kRowTile, a.rows - found.first);
  }
  *tiles = tiles_before + rest;
  return found;
}

// One wave an output column j and row tile; lane holds every 64th byte of q's row.
__global__ __launch_bounds__(kThreads) void w4_kernel(ggk_w4_args a) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int columns = (a.n + kWaves - 1) / kWaves;
  const int fan = a.x_rows > 0 ? a.rows / a.x_rows : 1;
  long long tiles = (a.rows + kRowTile - 1) / kRowTile;
  if (a.experts > 0) (void)find_tile(a, 0, &tiles);
  for (long long w = blockIdx.x; w < tiles * columns; w += gridDim.x) {
    RowTile t{0, (int)(w / columns) * kRowTile, 0};
    t.rows = min(kRowTile, a.rows - t.first);
    if (a.experts > 0) t = find_tile(a, w / columns, &tiles);
    const int j = (int)(w % columns) * kWaves + wave;
    if (j >= a.n) continue;
    int slot[kRowTile];
    const _Float16* x[kRowTile];
#pragma unroll
    for (int i = 0; i < kRowTile; ++i) {
      int s = i < t.rows ? t.first + i : -1;
      if (s >= 0 && a.experts > 0) {
        s = a.order[s];
        if (s >= a.rows) s = -1;
      }
      slot[i] = s;
      x[i] = static_cast<const _Float16*>(a.x) + (s < 0 ? 0 : s / fan) * a.ldx;
    }
    float acc[kRowTile] = {};
    if (t.expert < a.experts || a.experts == 0) {
      const unsigned char* q = a.q + t.expert * a.stride_q + (long long)j * a.ldq;
      const _Float16* scales = static_cast<const _Float16*>(a.scales) + t.expert * a.stride_s + (long long)j * a.lds;
      const unsigned char* zeros = a.zeros == nullptr ? nullptr : a.zeros + t.expert * a.stride_z + (long long)j * a.ldz;
      for (int b = lane; b < a.k / 2; b += kWave) {
        const int g = 2 * b / a.group;
        const float zero = zeros == nullptr ? 8.0f : (float)zeros[g];
        const float s = (float)scales[g];
        const float lo = (float)(q[b] & 15) - zero, hi = (float)(q[b] >> 4) - zero;
#pragma unroll
        for (int i = 0; i < kRowTile; ++i) {
          if (slot[i] >= 0) acc[i] += s * ((float)x[i][2 * b] * lo + (float)x[i][2 * b + 1] * hi);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRowTile; ++i) {
      const float sum = wave_sum(acc[i]);
      if (lane == 0 && slot[i] >= 0) {
        const bool zero = a.experts > 0 && t.expert == a.experts;
        const float y = zero ? 0.0f : (a.row_weights != nullptr ? sum * a.row_weights[slot[i]] : sum);
        const long long at = slot[i] * a.ldy + j;
        if (a.y_type == GGK_TYPE_F16) {
          static_cast<_Float16*>(a.y)[at] = (_Float16)y;
        } else {
          static_cast<float*>(a.y)[at] = y;
        }
      }
    }
  }
}

}  // namespace

extern "C" hipError_t ggk_w4_check(const ggk_w4_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_w4_args& a = *args;
  if (a.rows < 0 || a.rows > GGK_ROUTE_MAX_TOTAL_SLOTS || a.x_rows < 0 || a.n < 0 || a.k < 0 || a.experts < 0 || a.experts > GGK_MOE_MAX_EXPERTS ||
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
    if (a.y == nullptr || (a.k > 0 && (a.x == nullptr || a.q == nullptr || a.scales == nullptr))) {
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
  const long long tiles = (a.rows + kRowTile - 1) / kRowTile + (a.experts > 0 ? min(a.rows, a.experts + 1) : 0);
  const long long blocks = tiles * ((a.n + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(w4_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}
