// gg_route.hip -- the routing of a mixture-of-experts layer: which experts each
// token takes and with what weights, how many slots each expert got, the order
// of the slots by expert, the balance loss, and the gradient with respect to
// the router's logits.
//
//   z_te   logits, -inf where an expert is closed to a token
//   ids    the `slots` largest z_t, ties to the lower expert, NaN above all
//   a_ts   exp(z_ts - max) / sum over the chosen (normalize) or over all experts
//   w_ts   scale * a_ts
//   L      experts * sum_e f_e P_e,  f_e = counts_e / sum counts,
//          P_e = mean over the routed tokens of p_te = softmax(z_t)_e
//
// A token is routed when one of its slots has an expert.  Logits are read
// once forward and once backward (with one write of the gradient); the softmax
// is computed again in the backward pass, which costs less than p's bytes.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <stdint.h>

#include "grouped_gemm_amd_kernels.h"

namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxExperts = GGK_MOE_MAX_EXPERTS;
constexpr int kMaxBlocks = 1024;  // blocks of tokens, each with one partial sum per expert

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float* out) { *out = v; }
__device__ __forceinline__ void from_float(float v, _Float16* out) { *out = (_Float16)v; }
__device__ __forceinline__ void from_float(float v, __hip_bfloat16* out) { *out = __float2bfloat16(v); }

// A logit as an unsigned key of the same order: NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kClosedKey = 0x007fffffu;  // order_key(-inf): no expert is chosen at or below it

__device__ __forceinline__ float wave_sum(float v) {
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  for (int d = 1; d < kWave; d *= 2) v = fmaxf(v, __shfl_xor(v, d, kWave));
  return v;
}

struct Plan {
  int blocks, rows_per_block;
};

Plan plan_blocks(int tokens) {
  int rows = (tokens + kMaxBlocks - 1) / kMaxBlocks;
  rows = rows < 16 ? 16 : rows;
  const int blocks = tokens > 0 ? (tokens + rows - 1) / rows : 1;
  return {blocks, rows};
}

// Workspace: partial sums of p [experts][blocks], then slot counts [experts + 1][blocks] (the last row: slots
// without an expert), then per expert the sum of p and the number of routed tokens.
struct Workspace {
  float* p;
  int* count;
  int* routed;
};

Workspace carve(void* base, int experts, int blocks) {
  char* b = static_cast<char*>(base);
  Workspace w;
  w.p = reinterpret_cast<float*>(b);
  w.count = reinterpret_cast<int*>(b + sizeof(float) * (size_t)experts * blocks);
  w.routed = w.count + (size_t)(experts + 1) * blocks;
  return w;
}

size_t workspace_bytes(int experts, int blocks) {
  return sizeof(int) * ((size_t)experts * blocks + (size_t)(experts + 1) * blocks + (size_t)blocks);
}

// One wave a token: lane holds experts lane + 64 j.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void route_rows_kernel(ggk_route_args a, Workspace ws, Plan plan) {
  __shared__ int s_count[kMaxExperts + 1];
  __shared__ float s_p[kWaves][kMaxExperts];
  __shared__ int s_routed;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  for (int e = tid; e <= a.experts; e += kThreads) s_count[e] = 0;
  if (tid == 0) s_routed = 0;
  __syncthreads();
  float sums[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sums[j] = 0.0f;
  const int first = blockIdx.x * plan.rows_per_block;
  const int last = min(a.tokens, first + plan.rows_per_block);
  for (int t = first + wave; t < last; t += kWaves) {
    const T* row = static_cast<const T*>(a.logits) + (long long)t * a.ld;
    const bool live = a.token_mask == nullptr || a.token_mask[t] != 0;
    float z[V];
    uint32_t key[V];
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + kWave * j;
      z[j] = live && e < a.experts ? to_float(row[e]) : -__builtin_inff();
      key[j] = order_key(z[j]);
      top = fmaxf(top, z[j]);
    }
    top = wave_max(top);
    float my_z = 0.0f;
    int my_id = -1;
    const long long slot0 = (long long)t * a.slots;
    if (a.given_ids != nullptr) {
      if (lane < a.slots && live) {
        const int id = a.given_ids[slot0 + lane];
        if (id >= 0 && id < a.experts) {
          my_z = to_float(row[id]);
          if (order_key(my_z) > kClosedKey) my_id = id;
        }
      }
    } else {
      for (int s = 0; s < a.slots; ++s) {
        uint32_t best = 0;
        int at = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (key[j] > best) {
            best = key[j];
            at = lane + kWave * j;
          }
        }
        for (int d = 1; d < kWave; d *= 2) {
          const uint32_t other = __shfl_xor(best, d, kWave);
          const int other_at = __shfl_xor(at, d, kWave);
          if (other > best || (other == best && other_at < at)) {
            best = other;
            at = other_at;
          }
        }
        if (best <= kClosedKey) break;
        float chosen_z = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (at == lane + kWave * j) {
            key[j] = 0;
            chosen_z = z[j];
          }
        }
        chosen_z = __shfl(chosen_z, at % kWave, kWave);
        if (lane == s) {
          my_id = at;
          my_z = chosen_z;
        }
      }
    }
    const bool routed = __ballot(my_id >= 0) != 0;
    const bool has = my_id >= 0;
    float total = 0.0f, p[V];
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = 0.0f;
    if (routed) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = expf(z[j] - top);
        total += p[j];
      }
      total = wave_sum(total);
      const float inv = 1.0f / total;
#pragma unroll
      for (int j = 0; j < V; ++j) sums[j] += p[j] * inv;
    }
    // A NaN logit is the largest of its row for the choice, and makes the row's weights NaN.
    float w = 0.0f;
    if (a.normalize) {
      const float peak = wave_max(has ? my_z : -__builtin_inff());
      const float e = has ? expf(my_z - peak) : 0.0f;
      const float sum = wave_sum(e);
      w = has ? a.scale * (e / sum) : 0.0f;
    } else if (has) {
      w = a.scale * (expf(my_z - top) / total);
    }
    if (lane < a.slots) {
      a.weights[slot0 + lane] = w;
      a.ids[slot0 + lane] = my_id;
      atomicAdd(&s_count[has ? my_id : a.experts], 1);
    }
    if (lane == 0 && routed) atomicAdd(&s_routed, 1);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (lane + kWave * j < a.experts) s_p[wave][lane + kWave * j] = sums[j];
  }
  __syncthreads();
  for (int e = tid; e <= a.experts; e += kThreads) {
    ws.count[(size_t)e * plan.blocks + blockIdx.x] = s_count[e];
    if (e < a.experts) {
      float p = 0.0f;
      for (int w = 0; w < kWaves; ++w) p += s_p[w][e];
      ws.p[(size_t)e * plan.blocks + blockIdx.x] = p;
    }
  }
  if (tid == 0) ws.routed[blockIdx.x] = s_routed;
}

// One block an expert (and one for the slots without any): its slot counts over the blocks of tokens become their
// exclusive prefix sums, its count the total; p's sum goes to the front of its row.
__global__ __launch_bounds__(kThreads) void route_columns_kernel(ggk_route_args a, Workspace ws, int blocks) {
  __shared__ int s_total[kWaves];
  __shared__ float s_sum[kWaves];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int* count = ws.count + (size_t)e * blocks;
  constexpr int kPer = kMaxBlocks / kThreads;
  int mine[kPer], sum = 0;
  float p = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    mine[i] = b < blocks ? count[b] : 0;
    sum += mine[i];
    if (b < blocks && e < a.experts) p += ws.p[(size_t)e * blocks + b];
  }
  int x = sum;
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  p = wave_sum(p);
  if (lane == kWave - 1) s_total[wave] = x;
  if (lane == 0) s_sum[wave] = p;
  __syncthreads();
  int before = x - sum, total = 0;
  p = 0.0f;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? s_total[w] : 0;
    total += s_total[w];
    p += s_sum[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    if (b < blocks) count[b] = before;
    before += mine[i];
  }
  if (tid == 0 && e < a.experts) {
    a.counts[e] = total;
    ws.p[(size_t)e * blocks] = p;
  }
}

// Places each slot at its expert's part of the order, slots of a block in their own order; block 0 also
// computes the loss.
__global__ __launch_bounds__(kThreads) void route_order_kernel(ggk_route_args a, Workspace ws, Plan plan) {
  __shared__ int s_at[kMaxExperts + 1];
  __shared__ int s_totals[kThreads];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  constexpr int kPer = (kMaxExperts + kThreads) / kThreads;
  int mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    mine[i] = e < a.experts ? a.counts[e] : 0;
    sum += mine[i];
  }
  s_totals[tid] = sum;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < tid; ++i) before += s_totals[i];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    if (e <= a.experts) s_at[e] = before + ws.count[(size_t)e * plan.blocks + blockIdx.x];
    before += mine[i];
  }
  __syncthreads();
  if (wave == 0) {
    const long long first = (long long)blockIdx.x * plan.rows_per_block * a.slots;
    long long last = first + (long long)plan.rows_per_block * a.slots;
    const long long all = (long long)a.tokens * a.slots;
    last = last < all ? last : all;
    for (long long i0 = first; i0 < last; i0 += kWave) {
      const bool in = i0 + lane < last;
      int id = in ? a.ids[i0 + lane] : -1;
      id = id < 0 ? a.experts : id;
      unsigned long long same = __ballot(in);
      for (int bit = 0; bit < 11; ++bit) {
        const unsigned long long set = __ballot((id >> bit) & 1);
        same &= ((id >> bit) & 1) ? set : ~set;
      }
      if (in) {
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int at = s_at[id];
        __builtin_amdgcn_wave_barrier();
        a.order[at + rank] = (int)(i0 + lane);
        if (rank == 0) s_at[id] = at + __popcll(same);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  } else if (wave == 1 && blockIdx.x == 0 && a.loss != nullptr) {
    int routed = 0;
    for (int b = lane; b < plan.blocks; b += kWave) routed += ws.routed[b];
    float used = 0.0f, part = 0.0f;
    for (int d = 1; d < kWave; d *= 2) routed += __shfl_xor(routed, d, kWave);
    for (int e = lane; e < a.experts; e += kWave) used += (float)a.counts[e];
    used = wave_sum(used);
    const float inv_used = used > 0.0f ? 1.0f / used : 0.0f;
    const float inv_routed = routed > 0 ? 1.0f / (float)routed : 0.0f;
    for (int e = lane; e < a.experts; e += kWave) {
      const float f = (float)a.counts[e] * inv_used;
      part += f * (ws.p[(size_t)e * plan.blocks] * inv_routed);
      a.slope[e] = (float)a.experts * f * inv_routed;
    }
    part = wave_sum(part);
    if (lane == 0) *a.loss = (float)a.experts * part;
  }
}

// dz of one token a wave.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void route_gradient_kernel(ggk_route_gradient_args a) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const float d_loss = a.d_loss != nullptr ? *a.d_loss : 0.0f;
  for (int t = blockIdx.x * kWaves + wave; t < a.tokens; t += gridDim.x * kWaves) {
    const T* row = static_cast<const T*>(a.logits) + (long long)t * a.ld;
    T* out = static_cast<T*>(a.d_logits) + (long long)t * a.experts;
    const long long slot0 = (long long)t * a.slots;
    const int my_id = lane < a.slots ? a.ids[slot0 + lane] : -1;
    const bool has = my_id >= 0 && my_id < a.experts;
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.0f;
    if (__ballot(has) != 0) {
      float z[V], top = -__builtin_inff(), total = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = lane + kWave * j;
        z[j] = e < a.experts ? to_float(row[e]) : -__builtin_inff();
        top = fmaxf(top, z[j]);
      }
      top = wave_max(top);
      float p[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = expf(z[j] - top);
        total += p[j];
      }
      total = wave_sum(total);
      const float my_z = has ? to_float(row[my_id]) : -__builtin_inff();
      float my_a = 0.0f;
      if (a.normalize) {
        const float peak = wave_max(my_z);
        const float e = has ? expf(my_z - peak) : 0.0f;
        my_a = e / wave_sum(e);
      } else {
        my_a = has ? expf(my_z - top) / total : 0.0f;
      }
      const float g = has && a.d_weights != nullptr ? a.scale * a.d_weights[slot0 + lane] : 0.0f;
      const float mean = wave_sum(has ? my_a * g : 0.0f);
      const float my_d = has ? (a.normalize ? my_a * (g - mean) : my_a * g) : 0.0f;
      float c[V], dot = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = lane + kWave * j;
        p[j] = p[j] / total;
        c[j] = e < a.experts && a.slope != nullptr ? d_loss * a.slope[e] : 0.0f;
        dot += p[j] * c[j];
      }
      dot = wave_sum(dot) + (a.normalize ? 0.0f : mean);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = p[j] * (c[j] - dot);
      for (int s = 0; s < a.slots; ++s) {
        const int id = __shfl(has ? my_id : -1, s, kWave);
        const float part = __shfl(my_d, s, kWave);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += id == lane + kWave * j ? part : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (lane + kWave * j < a.experts) from_float(d[j], &out[lane + kWave * j]);
    }
  }
}

template <class T>
hipError_t launch_rows(const ggk_route_args& a, const Workspace& ws, const Plan& plan, hipStream_t stream) {
  auto kernel = a.experts <= 64 ? route_rows_kernel<T, 1>
                : a.experts <= 128 ? route_rows_kernel<T, 2>
                : a.experts <= 256 ? route_rows_kernel<T, 4>
                : a.experts <= 512 ? route_rows_kernel<T, 8> : route_rows_kernel<T, 16>;
  hipLaunchKernelGGL(kernel, dim3(plan.blocks), dim3(kThreads), 0, stream, a, ws, plan);
  return hipGetLastError();
}

template <class T>
hipError_t launch_gradient(const ggk_route_gradient_args& a, hipStream_t stream) {
  auto kernel = a.experts <= 64 ? route_gradient_kernel<T, 1>
                : a.experts <= 128 ? route_gradient_kernel<T, 2>
                : a.experts <= 256 ? route_gradient_kernel<T, 4>
                : a.experts <= 512 ? route_gradient_kernel<T, 8> : route_gradient_kernel<T, 16>;
  const int blocks = min((a.tokens + kWaves - 1) / kWaves, 8192);
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

bool bad_sizes(int tokens, int experts, int slots, int type, long long ld) {
  return tokens < 0 || experts < 1 || experts > kMaxExperts || slots < 1 || slots > GGK_ROUTE_MAX_SLOTS ||
         (type != GGK_TYPE_F32 && type != GGK_TYPE_F16 && type != GGK_TYPE_BF16) || (tokens > 1 && ld < experts) ||
         (long long)tokens * slots > 0x7fffffffLL;
}

}  // namespace

extern "C" size_t ggk_route_workspace(int tokens, int experts) {
  if (tokens < 0 || experts < 1 || experts > kMaxExperts) return 0;
  return workspace_bytes(experts, plan_blocks(tokens).blocks);
}

extern "C" hipError_t ggk_route_check(const ggk_route_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_route_args& a = *args;
  if (bad_sizes(a.tokens, a.experts, a.slots, a.type, a.ld)) return hipErrorInvalidValue;
  if (a.given_ids == nullptr && a.slots > a.experts) return hipErrorInvalidValue;
  if (a.workspace_bytes < ggk_route_workspace(a.tokens, a.experts)) return hipErrorInvalidValue;
  if (a.counts == nullptr || a.workspace == nullptr || (a.loss == nullptr) != (a.slope == nullptr) ||
      (a.tokens > 0 && (a.logits == nullptr || a.weights == nullptr || a.ids == nullptr || a.order == nullptr))) {
    return hipErrorInvalidDevicePointer;
  }
  return hipSuccess;
}

extern "C" hipError_t ggk_route(const ggk_route_args* args, hipStream_t stream) {
  hipError_t st = ggk_route_check(args);
  if (st != hipSuccess) return st;
  const ggk_route_args& a = *args;
  const Plan plan = plan_blocks(a.tokens);
  const Workspace ws = carve(a.workspace, a.experts, plan.blocks);
  st = a.type == GGK_TYPE_F32 ? launch_rows<float>(a, ws, plan, stream)
       : a.type == GGK_TYPE_F16 ? launch_rows<_Float16>(a, ws, plan, stream)
                                : launch_rows<__hip_bfloat16>(a, ws, plan, stream);
  if (st != hipSuccess) return st;
  hipLaunchKernelGGL(route_columns_kernel, dim3(a.experts + 1), dim3(kThreads), 0, stream, a, ws, plan.blocks);
  st = hipGetLastError();
  if (st != hipSuccess) return st;
  hipLaunchKernelGGL(route_order_kernel, dim3(plan.blocks), dim3(kThreads), 0, stream, a, ws, plan);
  return hipGetLastError();
}

extern "C" hipError_t ggk_route_gradient_check(const ggk_route_gradient_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_route_gradient_args& a = *args;
  if (bad_sizes(a.tokens, a.experts, a.slots, a.type, a.ld)) return hipErrorInvalidValue;
  if (a.tokens > 0 && (a.logits == nullptr || a.ids == nullptr || a.d_logits == nullptr ||
                       (a.d_loss != nullptr && a.slope == nullptr))) {
    return hipErrorInvalidDevicePointer;
  }
  return hipSuccess;
}

extern "C" hipError_t ggk_route_gradient(const ggk_route_gradient_args* args, hipStream_t stream) {
  const hipError_t st = ggk_route_gradient_check(args);
  if (st != hipSuccess || args->tokens == 0) return st;
  return args->type == GGK_TYPE_F32 ? launch_gradient<float>(*args, stream)
         : args->type == GGK_TYPE_F16 ? launch_gradient<_Float16>(*args, stream)
                                      : launch_gradient<__hip_bfloat16>(*args, stream);
}
