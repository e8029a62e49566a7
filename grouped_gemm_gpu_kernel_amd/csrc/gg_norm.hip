// gg_norm.hip -- the root-mean-square norm of rows with the residual's addition,
// written as 8-bit rows:
//
//   h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight
//   scale of 128 columns = max(max |y| / 448, 2^-126), q = y / scale
//
// Bound by the bytes of x, the residual and the outputs: a row is read once and held in registers, 8 neighbouring
// columns a lane and chunk, so that a block of 128 columns is one DPP row of 16 lanes and its largest value is found
// without LDS.  A row takes a wave up to 2048 columns, else a workgroup of 4 waves (16 above 16384), with at most 64
// values a lane.  16384 rows of 8192 with residual and y take 214 us (5.65 TB/s), without them 83; one row 3.4 in a graph.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gg_common.h"
#include "gg_fp8_rows.h"
#include "grouped_gemm_amd_kernels.h"

namespace {

using gg::kWave;
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

template <int TYPE>
struct Type;
template <>
struct Type<GGK_TYPE_F32> {
  using T = float;
};
template <>
struct Type<GGK_TYPE_F16> {
  using T = _Float16;
};
template <>
struct Type<GGK_TYPE_BF16> {
  using T = __bf16;
};

// `count` (0 to 8) values from p on; the rest is 0.  Rows may begin anywhere: 8 values are moved by instructions of 16 bytes at
// their type's alignment.  WHOLE: all 8 or none are there (columns in multiples of 8; 8192 rows of 5120 float take 101 us so, 115
// with the other loop).
template <class T, bool WHOLE>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[8]) {
  T t[8] = {};
  if (WHOLE ? count > 0 : count == 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4v part = reinterpret_cast<const gg::Any16*>(p)[i];
      __builtin_memcpy(t + i * (16 / sizeof(T)), &part, 16);
    }
  } else if (!WHOLE && count > 0) {
#pragma unroll
    for (int i = 0; i < 7; ++i) {
      if (i < count) t[i] = p[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}

template <class T, bool WHOLE>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
  if (WHOLE ? count > 0 : count == 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      uint4v part;
      __builtin_memcpy(&part, t + i * (16 / sizeof(T)), 16);
      reinterpret_cast<gg::Any16*>(p)[i] = part;
    }
  } else if (!WHOLE && count > 0) {
#pragma unroll
    for (int i = 0; i < 7; ++i) {
      if (i < count) p[i] = t[i];
    }
  }
}

template <int TYPE, int WTYPE, int LANES, int CHUNKS, bool WHOLE>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_kernel(ggk_norm_fp8_args a) {
  using T = typename Type<TYPE>::T;
  using W = typename Type<WTYPE>::T;
  constexpr int kThreads = LANES < 256 ? 256 : LANES, kRows = kThreads / LANES, kWaves = LANES / kWave;
  const int lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * kRows + threadIdx.x / LANES;
  if (kRows > 1 && row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* residual = a.residual != nullptr ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  float h[CHUNKS][8];
  float squares = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int at = 8 * (c * LANES + lane), count = min(max(a.columns - at, 0), 8);
    load8<T, WHOLE>(x + at, count, h[c]);
  }
  if (residual != nullptr) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int at = 8 * (c * LANES + lane), count = min(max(a.columns - at, 0), 8);
      float r[8];
      load8<T, WHOLE>(residual + at, count, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[c][i] += r[i];
    }
  }
  T* sum = a.sum != nullptr ? static_cast<T*>(a.sum) + row * a.ldsum : nullptr;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int at = 8 * (c * LANES + lane), count = min(max(a.columns - at, 0), 8);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) part = fmaf(h[c][i], h[c][i], part);
    squares += part;
    if (sum != nullptr) store8<T, WHOLE>(sum + at, count, h[c]);
  }
#pragma unroll
  for (int d = kWave / 2; d > 0; d /= 2) squares += __shfl_xor(squares, d, kWave);
  if constexpr (kWaves > 1) {
    __shared__ float s_squares[kWaves];
    if (lane % kWave == 0) s_squares[lane / kWave] = squares;
    __syncthreads();
    squares = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) squares += s_squares[w];
  }
  // Numbers are quotients in which the factor cancels: values carry its power of two, which rounds nothing, and scales and y
  // the rest of it.
  const float factor = 1.0f / sqrtf(squares / (float)a.columns + a.eps);
  const bool splits = factor > 0.0f && factor < __builtin_inff();
  int exponent = 0;
  const float part_of_one = frexpf(factor, &exponent), rest = splits ? part_of_one : 1.0f;
  const float power = splits ? ldexpf(1.0f, exponent) : factor;
  const W* weight = static_cast<const W*>(a.weight);
  T* y = a.y != nullptr ? static_cast<T*>(a.y) + row * a.ldy : nullptr;
  unsigned char* q = a.q + row * a.ldq;
  float* scales = a.scales + row * a.lds;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int at = 8 * (c * LANES + lane), count = min(max(a.columns - at, 0), 8);
    float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    if (weight != nullptr) load8<W, WHOLE>(weight + at, count, w);
    uint32_t largest = 0;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = (WHOLE ? count > 0 : i < count) ? h[c][i] * power * w[i] : 0.0f;  // past the end 0 * power may be NaN
      largest = max(largest, gg::magnitude_bits(v[i]));
    }
    if (y != nullptr) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = v[i] * rest;
      store8<T, WHOLE>(y + at, count, out);
    }
    const float most = __builtin_bit_cast(float, gg::row_max16(largest));
    const float scale = gg::fp8_scale(gg::magnitude_bits(most * rest));
    const gg::Fp8Divisor by(scale == gg::kFp8SmallestScale ? scale / rest : most * (1.0f / gg::kFp8Largest), most);
    const uint2v numbers = {gg::fp8_numbers(v[0], v[1], v[2], v[3], by),
                            gg::fp8_numbers(v[4], v[5], v[6], v[7], by)};
    if (WHOLE ? count > 0 : count == 8) {
      *reinterpret_cast<gg::Any8*>(q + at) = numbers;
    } else if (!WHOLE && count > 0) {
#pragma unroll
      for (int i = 0; i < 7; ++i) {
        if (i < count) q[at + i] = (unsigned char)(numbers[i / 4] >> (8 * (i % 4)));
      }
    }
    if (lane % 16 == 0 && count > 0) scales[at / gg::kFp8Block] = scale;
  }
}

// The rows from `first` on, `rows` of them.
template <class T>
ggk_norm_fp8_args run_of(const ggk_norm_fp8_args& a, long long first, int rows) {
  ggk_norm_fp8_args b = a;
  b.rows = rows;
  b.x = static_cast<const T*>(a.x) + first * a.ldx;
  if (a.residual != nullptr) b.residual = static_cast<const T*>(a.residual) + first * a.ldr;
  b.q = a.q + first * a.ldq;
  b.scales = a.scales + first * a.lds;
  if (a.y != nullptr) b.y = static_cast<T*>(a.y) + first * a.ldy;
  if (a.sum != nullptr) b.sum = static_cast<T*>(a.sum) + first * a.ldsum;
  return b;
}

template <int TYPE, int WTYPE, bool WHOLE>
hipError_t launch_rows(const ggk_norm_fp8_args& a, hipStream_t stream) {
  // A launch has less than 2^32 threads: more rows (2^21 of the widest and up) go by several.
  const auto go = [&](auto kernel, int rows, int threads) {
    const int most = (int)((1ll << 31) / threads) * rows;
    for (int first = 0; first < a.rows; first += most) {
      const ggk_norm_fp8_args b = run_of<typename Type<TYPE>::T>(a, first, a.rows - first < most ? a.rows - first : most);
      hipLaunchKernelGGL(kernel, dim3((b.rows + rows - 1) / rows), dim3(threads), 0, stream, b);
      const hipError_t st = hipGetLastError();
      if (st != hipSuccess) return st;
    }
    return hipSuccess;
  };
  const int chunks = (a.columns + 7) / 8;
  if (chunks <= 64) return go(norm_kernel<TYPE, WTYPE, 64, 1, WHOLE>, 4, 256);
  if (chunks <= 256) return go(norm_kernel<TYPE, WTYPE, 64, 4, WHOLE>, 4, 256);
  if (chunks <= 512) return go(norm_kernel<TYPE, WTYPE, 256, 2, WHOLE>, 1, 256);
  if (chunks <= 1024) return go(norm_kernel<TYPE, WTYPE, 256, 4, WHOLE>, 1, 256);
  if (chunks <= 2048) return go(norm_kernel<TYPE, WTYPE, 256, 8, WHOLE>, 1, 256);
  return go(norm_kernel<TYPE, WTYPE, 1024, 4, WHOLE>, 1, 1024);
}

template <int TYPE, int WTYPE>
hipError_t launch(const ggk_norm_fp8_args& a, hipStream_t stream) {
  return a.columns % 8 == 0 ? launch_rows<TYPE, WTYPE, true>(a, stream) : launch_rows<TYPE, WTYPE, false>(a, stream);
}

bool is_type(int type) { return type == GGK_TYPE_F32 || type == GGK_TYPE_F16 || type == GGK_TYPE_BF16; }

}  // namespace

extern "C" hipError_t ggk_norm_fp8_check(const ggk_norm_fp8_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_norm_fp8_args& a = *args;
  if (a.rows < 0 || a.rows > GGK_ROUTE_MAX_TOTAL_SLOTS || a.columns < 1 || a.columns > GGK_NORM_MAX_COLUMNS ||
      !is_type(a.type) || (a.weight != nullptr && !is_type(a.weight_type)) ||
      (a.weight != nullptr && a.weight_type != a.type && a.weight_type != GGK_TYPE_F32)) {
    return hipErrorInvalidValue;
  }
  const int blocks = (a.columns + gg::kFp8Block - 1) / gg::kFp8Block;
  if (a.rows > 1 && (a.ldx < a.columns || a.ldq < a.columns || a.lds < blocks ||
                     (a.residual != nullptr && a.ldr < a.columns) || (a.y != nullptr && a.ldy < a.columns) ||
                     (a.sum != nullptr && a.ldsum < a.columns))) {
    return hipErrorInvalidValue;
  }
  if (a.rows > 0 && (a.x == nullptr || a.q == nullptr || a.scales == nullptr)) return hipErrorInvalidDevicePointer;
  return hipSuccess;
}

extern "C" hipError_t ggk_norm_fp8(const ggk_norm_fp8_args* args, hipStream_t stream) {
  const hipError_t st = ggk_norm_fp8_check(args);
  if (st != hipSuccess || args->rows == 0) return st;
  const ggk_norm_fp8_args& a = *args;
  const bool same = a.weight == nullptr || a.weight_type == a.type;
  switch (a.type) {
    case GGK_TYPE_F32: return launch<GGK_TYPE_F32, GGK_TYPE_F32>(a, stream);
    case GGK_TYPE_F16:
      return same ? launch<GGK_TYPE_F16, GGK_TYPE_F16>(a, stream) : launch<GGK_TYPE_F16, GGK_TYPE_F32>(a, stream);
    default:
      return same ? launch<GGK_TYPE_BF16, GGK_TYPE_BF16>(a, stream)
                  : launch<GGK_TYPE_BF16, GGK_TYPE_F32>(a, stream);
  }
}
