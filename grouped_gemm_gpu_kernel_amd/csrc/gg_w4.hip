// gg_w4.hip -- products of a few rows with 4-bit weights, one matrix or one an
// expert:
//
//   y[i][j] = sum_g scales[j][g] * sum_{k in g} x[i][k] * (q[j][k] - zeros[j][g])
//
// With few rows the weights' bytes are what counts: they are read once, 16
// bytes a lane, straight into registers, and turned into binary16 there.
// q - zero is an integer of at most 9 bits, so binary16 holds it exactly, the
// matrix instructions (v_mfma_f32_16x16x32_f16: 16 rows of x by 16 columns j)
// sum exact products in float, and a group's scale multiplies its sum: no weight
// is ever rounded.
//
// A workgroup of 8 waves computes 16 NT (8 / WK) columns of up to 16 MAXT rows: WK waves split K among them, step
// by step, so that a narrow matrix still gives every CU loads to wait for, and their sums are joined in LDS in the
// waves' order.  x goes through LDS, a chunk of K at a time (all of it if the rows are few): read by every wave
// from memory it would take the vector memory path for longer than the weights do (four 16-byte loads a lane
// for each 16 bytes of weights).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grouped_gemm_amd_kernels.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
// A row of x may start on any element.
typedef half8v half8_any __attribute__((aligned(2)));

constexpr int kWave = 64;
constexpr int kCus = 256;
constexpr int kStep = 128;  // values of k a wave takes at once: 16 bytes of each of 16 rows of q in 4 lanes
constexpr int kMaxExperts = GGK_MOE_MAX_EXPERTS;

// The 8 weights of a dword less `zero`, in the order k0 k4 k1 k5 k2 k6 k3 k7.  1024 + q and 1024 + 16 q are
// what the nibbles are as the low mantissa bits of 0x6400; both differences are exact.
__device__ __forceinline__ half8v unpack(uint32_t w, half2v low, half2v high) {
  const half2v sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const uint32_t v = w >> 8;
  const half2v a = __builtin_bit_cast(half2v, (w & 0x000f000fu) | 0x64006400u) - low;
  const half2v b = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w & 0x00f000f0u) | 0x64006400u), sixteenth, -high);
  const half2v c = __builtin_bit_cast(half2v, (v & 0x000f000fu) | 0x64006400u) - low;
  const half2v d = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (v & 0x00f000f0u) | 0x64006400u), sixteenth, -high);
  return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x in the same order.
__device__ __forceinline__ half8v like_weights(half8v x) { return __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7); }

// Register j of lane row r to register r of lane row j (rows of 16 lanes).
__device__ __forceinline__ void transpose_rows(uint4v& w) {
  uint2v r = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  const uint32_t a0 = r[0], a2 = r[1];
  r = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const uint32_t a1 = r[0], a3 = r[1];
  r = __builtin_amdgcn_permlane16_swap(a0, a1, false, false);
  w[0] = r[0];
  w[1] = r[1];
  r = __builtin_amdgcn_permlane16_swap(a2, a3, false, false);
  w[2] = r[0];
  w[3] = r[1];
}

// The values of all four lane rows, in every lane.
__device__ __forceinline__ void gather_rows(uint32_t v, uint32_t (&out)[4]) {
  const uint2v even_odd = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  const uint2v e = __builtin_amdgcn_permlane32_swap(even_odd[0], even_odd[0], false, false);
  const uint2v o = __builtin_amdgcn_permlane32_swap(even_odd[1], even_odd[1], false, false);
  out[0] = e[0];
  out[1] = o[0];
  out[2] = e[1];
  out[3] = o[1];
}

// The rows of one tile: the expert, its first place in the order, how many.
struct RowTile {
  int expert, first, rows;
};

// Places and row tiles of every expert, made once a workgroup: expert e has places [first[e], first[e + 1]) and tiles
// [tile[e], tile[e + 1]); "expert" a.experts has the places that the counts leave.  Counts are clamped to >= 0 and
// their sums to the rows there are.
struct Experts {
  int first[kMaxExperts + 2];
  int tile[kMaxExperts + 2];
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

template <int THREADS, int ROWS>
__device__ void list_experts(const ggk_w4_args& a, Experts& s) {
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

template <int ROWS>
__device__ RowTile expert_tile(const ggk_w4_args& a, const Experts& s, int tile) {
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

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kDepth = 4;  // steps a wave has in flight

template <int MAXT>
struct Shared {
  // Rows of x, each 16 bytes longer than its chunk so that the 16 rows of an instruction's operand lie in
  // distinct banks; at the end the waves' sums.
  static constexpr int kXBytes = MAXT == 1 ? 32 * 1024 + 16 * 16 : 64 * 1024 + 64 * 16;
  alignas(16) unsigned char x[kXBytes];
  int slot[16 * MAXT];
  Experts experts;
};

// One item's rows and columns: sums over the wave's steps of K.  M row tiles of 16.
// FINE: groups that are not whole steps; each instruction's 32 values then lie in one group, for which a step's
// dwords are exchanged between the lanes of a column.
template <int M, int NT, int WK, int MAXT, bool FINE, bool ZEROS>
__device__ __forceinline__ void multiply_item(const ggk_w4_args& a, const RowTile& t, int column0, Shared<MAXT>& s,
                                              float4v (&sum)[M][NT]) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int column = lane % 16, row = lane / 16;  // of the lane in an instruction's operands; lane row
  const int wk = wave % WK;
  const int steps = (a.k + kStep - 1) / kStep;
  const int turns = (steps + WK - 1) / WK;  // steps of a wave, at most
  // Turns that a chunk of x holds, and its row length in values.
  const int rows = max(1, t.rows);
  const int chunk_turns = min(turns, (Shared<MAXT>::kXBytes / rows - 16) / (2 * kStep * WK));
  const int chunk_k = chunk_turns * WK * kStep;
  const int ld = chunk_k + 8;

  const unsigned char* q[NT];
  const _Float16* scales[NT];
  const unsigned char* zeros[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    const long long j = min(column0 + 16 * c + column, a.n - 1);
    q[c] = a.q + t.expert * a.stride_q + j * a.ldq;
    scales[c] = static_cast<const _Float16*>(a.scales) + t.expert * a.stride_s + j * a.lds;
    zeros[c] = ZEROS ? a.zeros + t.expert * a.stride_z + j * a.ldz : nullptr;
  }
  auto scale_of = [&](int c, int k) {  // scale and zero point of the group of k
    const int g = k / a.group;
    uint32_t v = *reinterpret_cast<const uint16_t*>(scales[c] + g);
    if constexpr (ZEROS) v |= (uint32_t)zeros[c][g] << 16;
    return v;
  };
  uint4v w[kDepth][NT];
  uint32_t sz[FINE ? kDepth : 1][NT];  // FINE: the lane row's 32 values of a step; else: the lane row's step of the next four
  auto load = [&](int turn, int d) {
    const int mine = (turn * WK + wk) * kStep + 32 * row;  // the lane's 32 values of k
    const bool in = mine < a.k;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      w[d][c] = uint4v{0, 0, 0, 0};
      if (in) w[d][c] = *reinterpret_cast<const uint4v*>(q[c] + mine / 2);
      if constexpr (FINE) sz[d][c] = in ? scale_of(c, mine) : 0;
    }
  };
  auto load_scales = [&](int turn) {
#pragma unroll
    for (int c = 0; c < NT; ++c) sz[0][c] = scale_of(c, min(((turn + row) * WK + wk) * kStep, a.k - kStep));
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) load(d, d);
  if constexpr (!FINE) load_scales(0);
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int c = 0; c < NT; ++c) sum[m][c] = float4v{};
  }

  // x of one chunk, in the order of the weights' halves, zeros past K and for slots that name no row.
  const int fan = a.rows / a.x_rows;
  auto stage = [&](int chunk) {
    const int pieces = chunk_k / 8;
    for (int i = tid; i < t.rows * pieces; i += kThreads) {
      const int r = i / pieces, p = i % pieces, k = chunk * chunk_k + 8 * p;
      const int slot = s.slot[r];
      half8v x = half8v{};
      if (slot >= 0 && k < a.k) x = *reinterpret_cast<const half8_any*>(static_cast<const _Float16*>(a.x) + slot / fan * a.ldx + k);
      *reinterpret_cast<half8v*>(s.x + 2 * (r * ld + 8 * p)) = like_weights(x);
    }
  };
  // The lane's rows of x in LDS; rows past the tile's are read as its last (their sums are not used).
  const unsigned char* x[M];
#pragma unroll
  for (int m = 0; m < M; ++m) x[m] = s.x + 2 * (min(16 * m + column, rows - 1) * ld + (FINE ? 8 : 32) * row);

  uint32_t four[NT][4];
  int in_chunk = chunk_turns;
  for (int turn0 = 0; turn0 < turns; turn0 += kDepth) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int turn = turn0 + d;
      if (turn >= turns) break;
      if (in_chunk == chunk_turns) {
        if (turn > 0) __syncthreads();
        stage(turn / chunk_turns);
        __syncthreads();
        in_chunk = 0;
      }
      if constexpr (!FINE) {
        if (d == 0) {
#pragma unroll
          for (int c = 0; c < NT; ++c) gather_rows(sz[0][c], four[c]);
          load_scales(turn + kDepth);
        }
      }
      const int at = 2 * (in_chunk * WK + wk) * kStep;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        uint32_t g[4];
        if constexpr (FINE) {
          transpose_rows(w[d][c]);
          gather_rows(sz[d][c], g);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) g[j] = turn * WK + wk < steps ? four[c][d] : 0;  // no step: zero times zero
        }
        half8v v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const _Float16 zero = ZEROS ? (_Float16)(float)(g[j] >> 16) : (_Float16)8.0f;
          const _Float16 low = (_Float16)1024.0f + zero, high = (_Float16)64.0f + zero;
          v[j] = unpack(w[d][c][j], half2v{low, low}, half2v{high, high});
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          float4v part = float4v{};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const half8v xs = *reinterpret_cast<const half8v*>(x[m] + at + (FINE ? 64 : 16) * j);
            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs, v[j], part, 0, 0, 0);
            if (FINE || j == 3) {
              const float scale = (float)__builtin_bit_cast(_Float16, (uint16_t)g[j]);
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[m][c][i] = fmaf(scale, part[i], sum[m][c][i]);
              part = float4v{};
            }
          }
        }
      }
      load(turn + kDepth, d);
      ++in_chunk;
    }
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

// Joins the waves' sums and writes y.
template <int M, int NT, int WK, int MAXT>
__device__ __forceinline__ void finish_item(const ggk_w4_args& a, const RowTile& t, int block0, Shared<MAXT>& s,
                                            const float4v (&sum)[M][NT]) {
  constexpr int kColumns = 16 * NT * (kWaves / WK);  // of the workgroup
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int column = lane % 16, row = lane / 16, wn = wave / WK, wk = wave % WK;
  float* s_sum = reinterpret_cast<float*>(s.x);  // [WK][16 M][kColumns]
  static_assert(WK * 16 * MAXT * kColumns * 4 <= Shared<MAXT>::kXBytes, "the sums fit x's place");
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int c = 0; c < NT; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s_sum[(wk * 16 * M + 16 * m + 4 * row + i) * kColumns + 16 * (wn * NT + c) + column] = sum[m][c][i];
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < t.rows * kColumns; i += kThreads) {
    const int r = i / kColumns, c = i % kColumns, j = block0 + c, slot = s.slot[r];
    if (j < a.n && slot >= 0) {
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w) y += s_sum[(w * 16 * M + r) * kColumns + c];
      if (a.row_weights != nullptr) y *= a.row_weights[slot];
      store_y(a, slot, j, y);
    }
  }
}

template <int M, int NT, int WK, int MAXT, bool FINE, bool ZEROS>
__device__ __forceinline__ void run_item(const ggk_w4_args& a, const RowTile& t, int block0, Shared<MAXT>& s) {
  float4v sum[M][NT];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  multiply_item<M, NT, WK, MAXT, FINE, ZEROS>(a, t, block0 + wave / WK * 16 * NT, s, sum);
  finish_item<M, NT, WK, MAXT>(a, t, block0, s, sum);
}

template <int NT, int WK, int MAXT, bool FINE, bool ZEROS>
__global__ __launch_bounds__(kThreads, 4) void w4_kernel(ggk_w4_args a) {
  constexpr int kRows = 16 * MAXT, kColumns = 16 * NT * (kWaves / WK);
  __shared__ Shared<MAXT> s;
  const int tid = threadIdx.x;
  const int blocks = (a.n + kColumns - 1) / kColumns;
  int tiles = (a.rows + kRows - 1) / kRows;
  if (a.experts > 0) {
    list_experts<kThreads, kRows>(a, s.experts);
    tiles = s.experts.tile[a.experts + 1];
  }
  for (long long item = blockIdx.x; item < (long long)tiles * blocks; item += gridDim.x) {
    const int tile = (int)(item / blocks), block0 = (int)(item % blocks) * kColumns;
    RowTile t{0, tile * kRows, 0};
    t.rows = min(kRows, a.rows - t.first);
    if (a.experts > 0) t = expert_tile<kRows>(a, s.experts, tile);
    for (int i = tid; i < t.rows; i += kThreads) {
      int slot = t.first + i;
      if (a.experts > 0) {
        slot = a.order[slot];
        if (slot >= a.rows) slot = -1;
      }
      s.slot[i] = slot;
    }
    __syncthreads();
    if (a.experts > 0 && t.expert == a.experts) {
      for (int i = tid; i < t.rows * kColumns; i += kThreads) {
        const int slot = s.slot[i / kColumns], j = block0 + i % kColumns;
        if (j < a.n && slot >= 0) store_y(a, slot, j, 0.0f);
      }
    } else if (MAXT == 1 || t.rows <= 16) {
      // Row tiles are a constant of the whole loop over K: the compiler leaves out the wait between a matrix
      // instruction and the use of its result when a branch on them lies between.
      run_item<1, NT, WK, MAXT, FINE, ZEROS>(a, t, block0, s);
    } else if (t.rows <= 32) {
      run_item<2, NT, WK, MAXT, FINE, ZEROS>(a, t, block0, s);
    } else {
      run_item<MAXT, NT, WK, MAXT, FINE, ZEROS>(a, t, block0, s);
    }
    __syncthreads();
  }
}

template <int NT, int WK, int MAXT>
hipError_t launch(const ggk_w4_args& a, hipStream_t stream) {
  const bool fine = a.group % kStep != 0;
  auto kernel = fine ? (a.zeros != nullptr ? w4_kernel<NT, WK, MAXT, true, true> : w4_kernel<NT, WK, MAXT, true, false>)
                     : (a.zeros != nullptr ? w4_kernel<NT, WK, MAXT, false, true> : w4_kernel<NT, WK, MAXT, false, false>);
  const int columns = 16 * NT * (kWaves / WK), rows = 16 * MAXT;
  const long long tiles = (a.rows + rows - 1) / rows + (a.experts > 0 ? min(a.rows, a.experts + 1) : 0);
  const long long items = tiles * ((a.n + columns - 1) / columns);
  const long long most = a.experts > 0 ? kCus * 2 : 0x7fffffff;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(items < most ? items : most)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

extern "C" hipError_t ggk_w4_check(const ggk_w4_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_w4_args& a = *args;
  if (a.rows < 0 || a.rows > GGK_ROUTE_MAX_TOTAL_SLOTS || a.x_rows < 0 || a.n < 0 || a.k < 1 || a.experts < 0 || a.experts > GGK_MOE_MAX_EXPERTS ||
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
  // Waves that split K: as many as it takes for 4096 waves in all, half of what the GPU holds.
  const int row_tiles = a.experts > 0 ? min(a.rows, a.experts) : (a.rows + 63) / 64;
  const long long waves = (long long)((a.n + 15) / 16) * row_tiles;
  if (a.experts > 0 || a.rows > 16) {
    return waves >= 4096 ? launch<1, 1, 4>(a, stream) : waves >= 2048 ? launch<1, 2, 4>(a, stream) : launch<1, 4, 4>(a, stream);
  }
  return waves >= 4096   ? launch<1, 1, 1>(a, stream)
         : waves >= 2048 ? launch<1, 2, 1>(a, stream)
         : waves >= 1024 ? launch<1, 4, 1>(a, stream)
                         : launch<1, 8, 1>(a, stream);
}
