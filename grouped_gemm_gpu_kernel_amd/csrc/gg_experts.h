// gg_experts.h -- the rows of every expert as tiles, listed in LDS from the
// counts that routing left on the device.  Args: a call's arguments with
// experts, rows and counts (device memory, not trusted).
#pragma once

#include <hip/hip_runtime.h>

#include "gg_common.h"

namespace gg {

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

template <int THREADS, int ROWS, class Args, class Table>
__device__ void list_experts(const Args& a, Table& s) {
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

template <int ROWS, class Args, class Table>
__device__ RowTile expert_tile(const Args& a, const Table& s, int tile) {
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

}  // namespace gg
