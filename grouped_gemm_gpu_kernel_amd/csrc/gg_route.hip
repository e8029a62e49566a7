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

#include <type_traits>

#include "grouped_gemm_amd_kernels.h"

namespace {

constexpr int kWave = 64;
constexpr int kThreads = 512;
constexpr int kSmallThreads = 1024;  // of the workgroup that routes a few tokens by itself
constexpr int kMaxExperts = GGK_MOE_MAX_EXPERTS;

typedef unsigned int uint2v __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- logits

// A logit as an unsigned key of the same order: NaN above everything, -0 equal to 0.  A float's key has 32
// bits; a 16-bit type's leaves room for the expert below it, lower experts larger, which makes keys of a
// token distinct and their maximum the choice itself.
template <class T>
struct Logit;

template <>
struct Logit<float> {
  static constexpr bool kDistinct = false;
  static constexpr uint32_t kClosed = 0x007fffffu;  // key of -inf: no expert is chosen at or below it
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ uint32_t key(float v, int) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  }
  // The logit of a key (NaN of NaN's).
  static __device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
  }
  static __device__ __forceinline__ float store(float v) { return v; }
};

template <class T, uint32_t NAN_BITS, uint32_t INF_BITS>
struct Logit16 {
  static constexpr bool kDistinct = true;
  static constexpr uint32_t kClosed = ((~INF_BITS & 0x7fffu) << 16) | 0xffffu;
  static __device__ __forceinline__ uint32_t key(T v, int expert) {
    uint32_t b = __builtin_bit_cast(uint16_t, v);
    if ((b & 0x7fffu) > INF_BITS) {
      b = 0xffffu;
    } else {
      b = b == 0x8000u ? 0u : b;
      b = b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
    }
    return b << 16 | (0xffffu - (uint32_t)expert);
  }
  static __device__ __forceinline__ T bits_of_key(uint32_t k) {
    uint32_t b = k >> 16;
    b = b == 0xffffu ? NAN_BITS : (b & 0x8000u ? b & 0x7fffu : ~b & 0xffffu);
    return __builtin_bit_cast(T, (uint16_t)b);
  }
};

template <>
struct Logit<_Float16> : Logit16<_Float16, 0x7e00u, 0x7c00u> {
  static __device__ __forceinline__ float value(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ float of_key(uint32_t k) { return (float)bits_of_key(k); }
  static __device__ __forceinline__ _Float16 store(float v) { return (_Float16)v; }
};

template <>
struct Logit<__hip_bfloat16> : Logit16<__hip_bfloat16, 0x7fc0u, 0x7f80u> {
  static __device__ __forceinline__ float value(__hip_bfloat16 v) {
    return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
  }
  static __device__ __forceinline__ float of_key(uint32_t k) { return value(bits_of_key(k)); }
  static __device__ __forceinline__ __hip_bfloat16 store(float v) { return __float2bfloat16(v); }
};

// exp(x) for x <= 0 on the hardware's exp2: x is rounded once more by the product, which a softmax over
// logits of spread d bears as it bears the rounding of z - max (d half steps of float).
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// ---------------------------------------------------------------- groups of lanes

// A token's logits are held by L lanes: 16 (one DPP row, four tokens a wave) or the whole wave.  Reductions
// exchange within the row by DPP -- neighbours, pairs, halves mirrored, the row mirrored, so that every
// lane adds the same pairs and ends with the same bits -- and across rows by the lane swaps of gfx950.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);  // every lane reads a lane of its row
}

template <int L, class Op>
__device__ __forceinline__ uint32_t group_reduce(uint32_t x, Op op) {
  x = op(x, dpp<0xb1>(x));   // quad_perm [1, 0, 3, 2]
  x = op(x, dpp<0x4e>(x));   // quad_perm [2, 3, 0, 1]
  x = op(x, dpp<0x141>(x));  // row_half_mirror
  x = op(x, dpp<0x140>(x));  // row_mirror
  if constexpr (L == kWave) {
    uint2v r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = op(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = op(r[0], r[1]);
  }
  return x;
}

template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
  return group_reduce<L>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int L>
__device__ __forceinline__ uint32_t group_min(uint32_t x) {
  return group_reduce<L>(x, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
template <int L>
__device__ __forceinline__ float group_max(float x) {
  return __uint_as_float(group_reduce<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int L>
__device__ __forceinline__ float group_sum(float x) {
  return __uint_as_float(group_reduce<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// Does the predicate hold for any lane of this lane's group?
template <int L>
__device__ __forceinline__ bool group_any(bool v) {
  const unsigned long long b = __ballot(v);
  if constexpr (L == kWave) return b != 0;
  return ((b >> (threadIdx.x & 48)) & 0xffffu) != 0;
}

// Expert of value j of a lane: V values in vectors of W, so that a vector's load is 4 to 16 bytes.
template <int L, int V>
struct Columns {
  static constexpr int W = V < 4 ? V : 4;
  static __device__ __forceinline__ int expert(int lane, int j) { return (j / W * L + lane) * W + j % W; }
};

// The lane's values of a row, `fill` past the experts.  vectors: every row's start and length are whole vectors.
template <class T, int L, int V>
__device__ __forceinline__ void load_row(const T* row, int lane, int experts, bool vectors, T fill, T* out) {
  constexpr int W = Columns<L, V>::W;
  typedef struct alignas(sizeof(T) * W) {
    T v[W];
  } Vector;
#pragma unroll
  for (int j = 0; j < V; j += W) {
    const int e = Columns<L, V>::expert(lane, j);
    if (vectors) {
      if (e < experts) {
        const Vector x = *reinterpret_cast<const Vector*>(row + e);
#pragma unroll
        for (int i = 0; i < W; ++i) out[j + i] = x.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) out[j + i] = fill;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) out[j + i] = e + i < experts ? row[e + i] : fill;
    }
  }
}

template <class T, int V>
bool whole_vectors(const void* base, long long ld, int experts) {
  constexpr long long kBytes = sizeof(T) * (V < 4 ? V : 4);
  return reinterpret_cast<uintptr_t>(base) % kBytes == 0 && ld * (long long)sizeof(T) % kBytes == 0 &&
         experts * (long long)sizeof(T) % kBytes == 0;
}

// ---------------------------------------------------------------- forward

// Tokens are dealt to blocks in runs of `rows`.
struct Plan {
  int blocks, rows;
  bool columns;  // the columns kernel runs between the rows and the order
  bool vectors;
  int run;  // tokens of a group whose p are added up in its registers before they go to LDS; 0: all of them
};

// A float sum of n terms is off by up to n half steps, and terms that are alike make that much of it.  Sums of p over a
// group's tokens are made in runs of about the root of their number, but of 64 at least, and the runs added up in LDS:
// 2^25 tokens of two experts, 2048 a group, were off by 253 half steps in one sum.
int tokens_a_run(int tokens) {
  if (tokens <= 64) return 0;
  int run = 64;
  while ((long long)run * run < tokens) ++run;
  return run;
}

// Workspace, written by the rows kernel: per block and expert the slots taken (one more column: slots without an
// expert; rows padded to whole vectors of four) and the sum of p, then per block the routed tokens.  The columns
// kernel turns the counts into sums over the blocks before, and the first block's sums of p into those over all.
struct Workspace {
  int* count;   // [blocks][pitch]
  float* p;     // [blocks][experts]
  int* routed;  // [blocks]
};

__host__ __device__ inline int count_pitch(int experts) { return (experts + 4) / 4 * 4; }

// At most this many entries of `count` are summed by every block of the order kernel itself, and with 41 to 80 experts
// there are fewer blocks so that they stay below it: two launches instead of three.  us of 16384 tokens without and with
// the loss, so and with 512 blocks: 41 experts 10.4, 13.3 and 11.2, 15.5; 64 experts 9.8, 12.5 and 11.2, 15.4; 80 experts
// 10.9, 17.0 and 12.0, 16.8.  65536 tokens have more to do than fewer blocks do well: 64 experts 17.7, 22.9 and 15.4, 19.4.
// With 128 experts and 8192 tokens (32 K entries) the order kernel's own sums took 15.0, the columns kernel 12.9; limits of
// 10, 20, 40, 80 and 160 K: 65521 tokens of 256 experts with the loss 49.5, 50.5, 49.8, 69.7 and 65.1.
constexpr int kMaxOwnSums = 20 * 1024;
constexpr int kMaxBlocks = 512;

Plan plan_blocks(int tokens, int experts) {
  const int least = kThreads / 16;  // one token a group
  const int own = kMaxOwnSums / experts;
  const int most = own >= kMaxBlocks / 2 && own < kMaxBlocks ? own : kMaxBlocks;
  int rows = (tokens + most - 1) / most;
  rows = rows < least ? least : (rows + least - 1) / least * least;
  const int blocks = tokens > 0 ? (tokens + rows - 1) / rows : 1;
  return {blocks, rows, (long long)blocks * experts > kMaxOwnSums, false, 0};
}

// So many tokens are routed by one workgroup.  Up to 256 experts it takes 64 at a time, at 16 lanes each: with 64 experts
// 4.5 us for one token and 6.4 for 128, where two launches take 6.7 for 129 (256 experts: 8.1 and 16.5, two launches 10.8:
// the second round of 64 loses there).  Above, a wave a token, it takes 16 at a
// time: with 512 experts and 8 slots 8.3 us for 16, 12.6 for 32, 21.5 for 64 and 38.7 for 128, where two launches take 18.
// (More than 16 slots also take a wave each, 20 of 64 experts 12, 21, 38 and 72, two launches 28; but the workspace's
// size does not know the slots.)  The counts per wave have to fit 64 KB of LDS.
bool is_small(int tokens, int experts) { return tokens <= (experts <= 256 ? 128 : 32) && experts <= 768; }

size_t workspace_ints(int experts, int blocks) {
  return (size_t)count_pitch(experts) * blocks + (size_t)experts * blocks + (size_t)blocks;
}

Workspace carve(void* base, int experts, int blocks) {
  Workspace w;
  w.count = static_cast<int*>(base);
  w.p = reinterpret_cast<float*>(w.count + (size_t)count_pitch(experts) * blocks);
  w.routed = reinterpret_cast<int*>(w.p + (size_t)experts * blocks);
  return w;
}

// What a group holds of a token before it is routed.
template <class T, int V>
struct Token {
  T z[V];
  bool live;
};

// Does routing need every logit of a token?
__device__ __forceinline__ bool needs_all(const ggk_route_args& a) {
  return a.given_ids == nullptr || !a.normalize || a.loss != nullptr;
}

template <class T, int L, int V>
__device__ __forceinline__ void load_token(const ggk_route_args& a, bool vectors, int t, int last, Token<T, V>& token) {
  const bool in = t < last;
  token.live = in && (a.token_mask == nullptr || a.token_mask[t] != 0);
  if (needs_all(a)) {
    // Of a padding token too: waiting for the mask first would put one load behind the other.
    load_row<T, L, V>(static_cast<const T*>(a.logits) + (long long)(in ? t : 0) * a.ld, threadIdx.x % L,
                      in ? a.experts : 0, vectors, Logit<T>::store(-__builtin_inff()), token.z);
  }
}

// The choice: slot s of a group's token to its lane s, as the s-th best key's expert and logit.  best: the best of all.
// With few values a lane, each round looks all of them over and takes the chosen one out.
template <class T, int L, int V>
__device__ __forceinline__ void choose(int slots, uint32_t (&key)[V], uint32_t best, int& my_id, float& my_z) {
  using Z = Logit<T>;
  using C = Columns<L, V>;
  const int lane = threadIdx.x % L, base = C::expert(lane, 0);
  for (int s = 0;; ++s) {
    const bool open = best > Z::kClosed;
    uint32_t at;
    if constexpr (Z::kDistinct) {
      at = 0xffffu - (best & 0xffffu);
    } else {
      // The lowest expert among those with the best key: a lane's first, then the least over lanes.
      at = 0xffffffffu;
#pragma unroll
      for (int j = V - 1; j >= 0; --j) at = key[j] == best ? (uint32_t)C::expert(lane, j) : at;
      at = group_min<L>(at);
    }
    if (lane == s && open) {
      my_id = (int)at;
      my_z = Z::of_key(best);
    }
    if (s + 1 == slots || __ballot(open) == 0) break;
    const int here = (int)at - base;  // the value's place, if it is one of the lane's
    uint32_t next = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (Z::kDistinct) {
        key[j] = key[j] == best ? 0u : key[j];
      } else {
        key[j] = here == C::expert(0, j) ? 0u : key[j];
      }
      next = key[j] > next ? key[j] : next;
    }
    best = group_max<L>(next);
  }
}

// With many, a lane keeps its three best in order and a round looks at the first alone.  A lane that has given all
// three makes them anew, from what comes after the last choice; with 8 slots of 256 experts one token in 50 has
// such a lane.  A round of 16 values costs 30 instructions instead of 105: 65521
// tokens of 256 float logits with their softmax 36 instead of 39 us, of which 26 are vector instructions issued.
template <class T, int L, int V>
__device__ __forceinline__ void choose_queued(int slots, const uint32_t (&key)[V], uint32_t best, int& my_id, float& my_z) {
  using Z = Logit<T>;
  using C = Columns<L, V>;
  const int lane = threadIdx.x % L;
  uint32_t q0, q1, q2;
  int e0, e1, e2;
  // The best three of all keys, or of those after (key `below`, expert `after`) in the order of the choice.
  auto fill = [&](auto all, uint32_t below, int after) {
    q0 = q1 = q2 = 0;
    e0 = e1 = e2 = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = C::expert(lane, j);
      const bool in = decltype(all)::value || key[j] < below || (!Z::kDistinct && key[j] == below && e > after);
      const uint32_t k = in ? key[j] : 0u;
      if constexpr (!Z::kDistinct) {  // equal keys keep the lower expert, which comes first, ahead
        const bool b0 = k > q0, b1 = k > q1, b2 = k > q2;
        e2 = b1 ? e1 : (b2 ? e : e2);
        e1 = b0 ? e0 : (b1 ? e : e1);
        e0 = b0 ? e : e0;
      }
      const uint32_t r = min(q0, k), r1 = min(q1, r);
      q0 = max(q0, k);
      q1 = max(q1, r);
      q2 = max(q2, r1);
    }
  };
  fill(std::true_type{}, 0, 0);
  int given = 0;
  for (int s = 0;; ++s) {
    const bool open = best > Z::kClosed;
    uint32_t at;
    if constexpr (Z::kDistinct) {
      at = 0xffffu - (best & 0xffffu);
    } else {
      at = group_min<L>(q0 == best ? (uint32_t)e0 : 0xffffffffu);
    }
    if (lane == s && open) {
      my_id = (int)at;
      my_z = Z::of_key(best);
    }
    if (s + 1 == slots || __ballot(open) == 0) break;
    const bool mine = q0 == best && (Z::kDistinct || e0 == (int)at);
    q0 = mine ? q1 : q0;
    q1 = mine ? q2 : q1;
    q2 = mine ? 0u : q2;
    e0 = mine ? e1 : e0;
    e1 = mine ? e2 : e1;
    given += mine ? 1 : 0;
    if (__ballot(given == 3) != 0) {
      fill(std::false_type{}, best, (int)at);
      given = 0;
    }
    best = group_max<L>(q0);
  }
}

// One token by its group: ids and weights to memory, slots counted in s_count, p added to sums.  Every lane
// of the wave calls it; `t` at or past `last` does nothing.  Returns whether the token was routed.
template <class T, int L, int V>
__device__ __forceinline__ bool route_token(const ggk_route_args& a, const Token<T, V>& token, int t, int last,
                                            int* s_count, float (&sums)[V]) {
  using Z = Logit<T>;
  using C = Columns<L, V>;
  const int lane = threadIdx.x % L;
  const bool in = t < last, live = token.live;
  const T* row = static_cast<const T*>(a.logits) + (long long)(in ? t : 0) * a.ld;
  const long long slot0 = (long long)t * a.slots;
  uint32_t key[V], best = 0;
  T z[V];
  if (needs_all(a)) {
    const T closed = Z::store(-__builtin_inff());
#pragma unroll
    for (int j = 0; j < V; ++j) {
      z[j] = live ? token.z[j] : closed;
      key[j] = Z::key(z[j], C::expert(lane, j));
      best = key[j] > best ? key[j] : best;
    }
    best = group_max<L>(best);
  }
  int my_id = -1;
  float my_z = -__builtin_inff();
  const float top = Z::of_key(best);  // NaN where the row holds one; what follows is NaN then, as it should be
  float inv = 0.0f;
  bool routed = best > Z::kClosed;
  if (a.given_ids != nullptr) {
    if (live && lane < a.slots) {
      const int id = a.given_ids[slot0 + lane];
      if (id >= 0 && id < a.experts) {
        const T v = row[id];
        if (Z::key(v, id) > Z::kClosed) {
          my_id = id;
          my_z = Z::value(v);
        }
      }
    }
    routed = group_any<L>(my_id >= 0);
  }
  // The softmax over all experts, before the choice takes its keys away.  A token that is not routed has every expert
  // closed, or none of its own: zeros.
  if (!a.normalize || a.loss != nullptr) {
    const float shift = routed ? top : 0.0f;
    float p[V], total = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = exp_of(Z::value(z[j]) - shift);
    if (a.given_ids != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] = routed ? p[j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) total += p[j];
    total = group_sum<L>(total);
    inv = routed ? 1.0f / total : 0.0f;
    if (a.loss != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j) sums[j] = fmaf(p[j], inv, sums[j]);
    }
  }
  if (a.given_ids == nullptr) {
    if constexpr (V >= 8) {
      choose_queued<T, L, V>(a.slots, key, best, my_id, my_z);
    } else {
      choose<T, L, V>(a.slots, key, best, my_id, my_z);
    }
  }
  const bool has = my_id >= 0;
  float w;
  if (a.normalize) {
    const float peak = a.given_ids != nullptr ? group_max<L>(my_z) : top;
    const float e = has ? exp_of(my_z - peak) : 0.0f;
    w = e / group_sum<L>(e);
  } else {
    w = exp_of(my_z - top) * inv;
  }
  if (in && lane < a.slots) {
    a.weights[slot0 + lane] = has ? a.scale * w : 0.0f;
    a.ids[slot0 + lane] = my_id;
    atomicAdd(&s_count[has ? my_id : a.experts], 1);
  }
  return routed;
}

// The wave's sums of p over its groups go to its row of s_part, a row of `experts` floats a wave: stored, or added to
// what is there.
template <int L, int V>
__device__ __forceinline__ void wave_sums(const float (&sums)[V], int experts, float* s_part, bool add) {
  using C = Columns<L, V>;
  const int tid = threadIdx.x, lane = tid % L, wave = tid / kWave;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float x = sums[j];
    if constexpr (L < kWave) {
      uint2v r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const int e = C::expert(lane, j);
    if (tid % kWave < L && e < experts) s_part[wave * experts + e] = add ? s_part[wave * experts + e] + x : x;
  }
}

// Tokens [first, last) by the groups of the workgroup, each group's next logits loaded while it routes a token.
// Returns the number of tokens that this lane's group has routed.  RUNS: after every `run` tokens of a group its sums of p
// are added to s_part, which has been cleared.
template <class T, int L, int V, int THREADS, bool RUNS>
__device__ __forceinline__ int route_tokens(const ggk_route_args& a, bool vectors, int first, int last, int* s_count,
                                            float (&sums)[V], int run, float* s_part) {
  constexpr int kGroups = THREADS / L;
  const int group = threadIdx.x / L;
  int routed = 0, in_run = 0;
  Token<T, V> next;
  load_token<T, L, V>(a, vectors, first + group, last, next);
  for (int t0 = first; t0 < last; t0 += kGroups) {
    const Token<T, V> token = next;
    if (t0 + kGroups < last) load_token<T, L, V>(a, vectors, t0 + kGroups + group, last, next);
    routed += route_token<T, L, V>(a, token, t0 + group, last, s_count, sums) ? 1 : 0;
    if constexpr (RUNS) {
      if (++in_run == run) {
        wave_sums<L, V>(sums, a.experts, s_part, true);
#pragma unroll
        for (int j = 0; j < V; ++j) sums[j] = 0.0f;
        in_run = 0;
      }
    }
  }
  return routed;
}

// The block's sums of p (balance) over its groups, to out[e].  s_part: a row of `experts` floats a wave; add: with runs'
// sums in it.
template <int L, int V, int THREADS>
__device__ __forceinline__ void block_sums(const float (&sums)[V], int experts, float* s_part, float* out, bool add) {
  const int tid = threadIdx.x;
  wave_sums<L, V>(sums, experts, s_part, add);
  __syncthreads();
  for (int e = tid; e < experts; e += THREADS) {
    float x = 0.0f;
    for (int w = 0; w < THREADS / kWave; ++w) x += s_part[w * experts + e];
    out[e] = x;
  }
}

// The tokens of one block: choice, weights, counts and sums of p.  65521 tokens of 256 float logits, 8 slots, loss: 37 us
// for 67 MB, bound by vector instructions (985 a wave for its 4 tokens, 26 us); 16384 of 64: 4.7 us, start and latency.
template <class T, int L, int V, bool RUNS>
__global__ __launch_bounds__(kThreads, 4) void route_rows_kernel(ggk_route_args a, Workspace ws, Plan plan) {
  extern __shared__ int shared[];  // counts [experts + 1], routed, then (balance) `experts` floats a wave
  int* s_count = shared;
  int* s_routed = shared + a.experts + 1;
  const int tid = threadIdx.x;
  float* s_part = reinterpret_cast<float*>(shared + a.experts + 2);
  const int clear = a.experts + 2 + (RUNS ? kThreads / kWave * a.experts : 0);
  for (int e = tid; e < clear; e += kThreads) shared[e] = 0;
  __syncthreads();
  float sums[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sums[j] = 0.0f;
  const int first = blockIdx.x * plan.rows;
  const int last = min(a.tokens, first + plan.rows);
  const int routed = route_tokens<T, L, V, kThreads, RUNS>(a, plan.vectors, first, last, s_count, sums, plan.run, s_part);
  if (tid % L == 0 && routed > 0) atomicAdd(s_routed, routed);
  if (a.loss != nullptr) {
    block_sums<L, V, kThreads>(sums, a.experts, s_part, ws.p + (size_t)blockIdx.x * a.experts, RUNS);
  }
  __syncthreads();
  const int pitch = count_pitch(a.experts);
  for (int e = tid; e < pitch; e += kThreads) ws.count[(size_t)blockIdx.x * pitch + e] = e <= a.experts ? s_count[e] : 0;
  if (tid == 0) ws.routed[blockIdx.x] = *s_routed;
}

// Sums over the blocks, kColumns columns a workgroup: each column's slices of blocks are added up, then the
// counts become the sums over the blocks before, the totals go to a.counts, and the sums of p to block 0's.  5 us for
// 512 blocks of 256 experts.
constexpr int kColumns = 16;
constexpr int kSlices = kThreads / kColumns;

__global__ __launch_bounds__(kThreads) void route_columns_kernel(ggk_route_args a, Workspace ws, int blocks) {
  __shared__ int s_count[kSlices][kColumns];
  __shared__ float s_p[kSlices][kColumns];
  const int tid = threadIdx.x, c = tid % kColumns, slice = tid / kColumns;
  const int e = blockIdx.x * kColumns + c, width = a.experts + 1, pitch = count_pitch(a.experts);
  constexpr int kPer = kMaxBlocks / kSlices;
  const int each = (blocks + kSlices - 1) / kSlices;
  const int b0 = slice * each, rows = max(0, min(each, blocks - b0));
  int count[kPer], sum = 0;
  float p = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    count[i] = i < rows && e < width ? ws.count[(size_t)(b0 + i) * pitch + e] : 0;
    sum += count[i];
  }
  if (a.loss != nullptr) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) p += i < rows && e < a.experts ? ws.p[(size_t)(b0 + i) * a.experts + e] : 0.0f;
  }
  s_count[slice][c] = sum;
  s_p[slice][c] = p;
  __syncthreads();
  int before = 0, total = 0;
  p = 0.0f;
#pragma unroll
  for (int s = 0; s < kSlices; ++s) {
    before += s < slice ? s_count[s][c] : 0;
    total += s_count[s][c];
    p += s_p[s][c];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i < rows && e < width) ws.count[(size_t)(b0 + i) * pitch + e] = before;
    before += count[i];
  }
  if (slice == 0 && e < a.experts) {
    a.counts[e] = total;
    if (a.loss != nullptr) ws.p[e] = p;  // block 0's row, read above by this column's threads alone
  }
}

// Exclusive prefix sum of one value per thread in thread order; ends with a barrier.
template <int THREADS>
__device__ __forceinline__ int block_before(int v, int* s_waves) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  if (lane == kWave - 1) s_waves[wave] = x;
  __syncthreads();
  int before = x - v;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) before += w < wave ? s_waves[w] : 0;
  __syncthreads();
  return before;
}

// Turns s_at[e], the places taken before this block's slots of each expert, into places in the order, adding the
// experts before (total[e]: all slots of e; the slots without an expert come last).
template <int THREADS>
__device__ __forceinline__ void add_experts_before(int* s_at, const int* total, int experts, int* s_waves) {
  const int tid = threadIdx.x;
  constexpr int kPer = (kMaxExperts + 1 + THREADS - 1) / THREADS;
  int mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    mine[i] = e < experts ? total[e] : 0;
    sum += mine[i];
  }
  int before = block_before<THREADS>(sum, s_waves);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    if (e <= experts) s_at[e] += before;
    before += mine[i];
  }
  __syncthreads();
}

struct Run {
  long long begin, end;  // a wave's slots
};

template <int THREADS>
__device__ __forceinline__ Run run_of_wave(long long first, long long last) {
  constexpr int kWaves = THREADS / kWave;
  const long long each = ((last - first + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
  const long long begin = first + (threadIdx.x / kWave) * each;
  return {begin, min(last, begin + each)};
}

// Places the workgroup's slots by expert, in their own order within one.  s_at: the next place of each expert; s_wave:
// experts + 1 ints a wave; id0: this lane's first id, loaded before the counts were known.  Every wave takes its run
// of slots, 64 at a time: it counts its slots of each expert, the waves' counts become their first places, and a slot
// goes to its wave's next place plus the number of lanes below with the same expert.  Waves write only their own row
// of s_wave.
template <int THREADS>
__device__ __forceinline__ void place_slots(const ggk_route_args& a, const Run& run, int id0, const int* s_at,
                                            int* s_wave) {
  constexpr int kWaves = THREADS / kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, width = a.experts + 1;
  for (int i = tid; i < kWaves * width; i += THREADS) s_wave[i] = 0;
  __syncthreads();
  int* my = s_wave + wave * width;
  const int bits = 32 - __builtin_clz(a.experts);
  for (long long i = run.begin + lane; i < run.end; i += kWave) {
    const int id = i == run.begin + lane ? id0 : a.ids[i];
    atomicAdd(&my[id < 0 ? a.experts : id], 1);
  }
  __syncthreads();
  for (int e = tid; e < width; e += THREADS) {
    int at = s_at[e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int n = s_wave[w * width + e];
      s_wave[w * width + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (long long i0 = run.begin; i0 < run.end; i0 += kWave) {
    const bool in = i0 + lane < run.end;
    int id = i0 == run.begin ? id0 : (in ? a.ids[i0 + lane] : -1);
    id = id < 0 ? a.experts : id;
    unsigned long long same = __ballot(in);
    for (int bit = 0; bit < bits; ++bit) {
      const bool set = (id >> bit) & 1;
      const unsigned long long other = __ballot(set);
      same &= set ? other : ~other;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int at = my[id];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read before the first lane of each expert writes
    if (in) {
      a.order[at + rank] = (int)(i0 + lane);
      if (rank == 0) my[id] = at + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// The loss and its slopes, by one wave: p[e] sums over all tokens, counts as in a.counts.
__device__ __forceinline__ void balance_loss(const ggk_route_args& a, const float* p, const int* counts, int routed) {
  const int lane = threadIdx.x % kWave;
  int used = 0;
  for (int e = lane; e < a.experts; e += kWave) used += counts[e];
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) used += __shfl_xor(used, d, kWave);
  const float inv_used = used > 0 ? 1.0f / (float)used : 0.0f;
  const float inv_routed = routed > 0 ? 1.0f / (float)routed : 0.0f;
  float part = 0.0f;
  for (int e = lane; e < a.experts; e += kWave) {
    const float f = (float)counts[e] * inv_used;
    part += f * (p[e] * inv_routed);
    a.slope[e] = (float)a.experts * f * inv_routed;
  }
  part = group_sum<kWave>(part);
  if (lane == 0) *a.loss = (float)a.experts * part;
}

__device__ __forceinline__ int all_routed(const Workspace& ws, int blocks) {
  int routed = 0;
  for (int b = threadIdx.x % kWave; b < blocks; b += kWave) routed += ws.routed[b];
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) routed += __shfl_xor(routed, d, kWave);
  return routed;
}

// The order of one block's slots; one more block computes the loss.  Without the columns kernel every block adds up
// the counts of all blocks itself, and the last one the sums of p.  6.2 us for 16384 tokens of 2 slots on 64 experts, 9.8
// for 65521 of 8 on 256: latency of a few dependent passes, not bytes.
__global__ __launch_bounds__(kThreads) void route_order_kernel(ggk_route_args a, Workspace ws, Plan plan) {
  extern __shared__ int shared[];  // s_at, s_total [experts + 1] each, then s_wave
  __shared__ int s_waves[kThreads / kWave];
  const int tid = threadIdx.x, width = a.experts + 1, block = blockIdx.x;
  int* s_at = shared;
  int* s_total = shared + width;
  int* s_wave = shared + 2 * width;
  const bool loss_block = block == plan.blocks;
  if (loss_block && plan.columns) {
    if (tid < kWave) balance_loss(a, ws.p, a.counts, all_routed(ws, plan.blocks));
    return;
  }
  const long long first = (long long)block * plan.rows * a.slots;
  const Run run = run_of_wave<kThreads>(
      first, min((long long)a.tokens * a.slots, first + (long long)plan.rows * a.slots));
  const int id0 = !loss_block && run.begin + tid % kWave < run.end ? a.ids[run.begin + tid % kWave] : -1;
  if (plan.columns) {
    for (int e = tid; e < width; e += kThreads) s_at[e] = ws.count[(size_t)block * count_pitch(a.experts) + e];
    __syncthreads();
    add_experts_before<kThreads>(s_at, a.counts, a.experts, s_waves);
  } else {
    // Threads take four columns of a slice of the blocks; the slices are added up in LDS.
    for (int e = tid; e < 2 * width; e += kThreads) shared[e] = 0;
    __syncthreads();
    typedef struct alignas(16) {
      int v[4];
    } Four;
    const int quads = count_pitch(a.experts) / 4, slices = max(1, kThreads / quads);
    const int each = (plan.blocks + slices - 1) / slices;
    for (int i = tid; i < slices * quads; i += kThreads) {
      const int quad = i % quads, b0 = i / quads * each, b1 = min(plan.blocks, b0 + each);
      int before[4] = {0, 0, 0, 0}, total[4] = {0, 0, 0, 0};
#pragma unroll 8
      for (int b = b0; b < b1; ++b) {
        const Four n = reinterpret_cast<const Four*>(ws.count)[(size_t)b * quads + quad];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          before[c] += b < block ? n.v[c] : 0;
          total[c] += n.v[c];
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (4 * quad + c < width) {
          atomicAdd(&s_at[4 * quad + c], before[c]);
          atomicAdd(&s_total[4 * quad + c], total[c]);
        }
      }
    }
    __syncthreads();
    if (loss_block) {
      // Sums of p: slices of the blocks per expert, then the slices in their order.
      float* s_p = reinterpret_cast<float*>(s_wave);
      const int parts = min(kThreads / kWave, max(1, kThreads / a.experts)), rows = (plan.blocks + parts - 1) / parts;
      for (int i = tid; i < parts * a.experts; i += kThreads) {
        const int e = i % a.experts, b0 = i / a.experts * rows, b1 = min(plan.blocks, b0 + rows);
        float p = 0.0f;
#pragma unroll 16
        for (int b = b0; b < b1; ++b) p += ws.p[(size_t)b * a.experts + e];
        s_p[i] = p;
      }
      __syncthreads();
      for (int e = tid; e < a.experts; e += kThreads) {
        float p = s_p[e];
        for (int i = 1; i < parts; ++i) p += s_p[i * a.experts + e];
        s_p[e] = p;
      }
      __syncthreads();
      if (tid < kWave) balance_loss(a, s_p, s_total, all_routed(ws, plan.blocks));
      return;
    }
    add_experts_before<kThreads>(s_at, s_total, a.experts, s_waves);
    if (block == 0) {
      for (int e = tid; e < a.experts; e += kThreads) a.counts[e] = s_total[e];
    }
  }
  place_slots<kThreads>(a, run, id0, s_at, s_wave);
}

// All of it for a few tokens, in one workgroup.
template <class T, int L, int V>
__global__ __launch_bounds__(kSmallThreads) void route_small_kernel(ggk_route_args a, bool vectors) {
  extern __shared__ int shared[];  // counts [experts + 1], routed, s_at [experts + 1], then s_part / s_wave
  __shared__ int s_waves[kSmallThreads / kWave];
  const int tid = threadIdx.x, width = a.experts + 1;
  int* s_count = shared;
  int* s_routed = shared + width;
  int* s_at = shared + width + 1;
  int* s_rest = shared + 2 * width + 1;
  for (int e = tid; e < 2 * width + 1; e += kSmallThreads) shared[e] = 0;
  __syncthreads();
  float sums[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sums[j] = 0.0f;
  const int routed = route_tokens<T, L, V, kSmallThreads, false>(a, vectors, 0, a.tokens, s_count, sums, 0, nullptr);
  if (tid % L == 0 && routed > 0) atomicAdd(s_routed, routed);
  __syncthreads();  // ids are read back below by other threads of this workgroup
  const Run run = run_of_wave<kSmallThreads>(0, (long long)a.tokens * a.slots);
  const int id0 = run.begin + tid % kWave < run.end ? a.ids[run.begin + tid % kWave] : -1;
  if (a.loss != nullptr) {
    float* s_part = reinterpret_cast<float*>(s_rest);
    block_sums<L, V, kSmallThreads>(sums, a.experts, s_part, s_part, false);
    __syncthreads();
    if (tid < kWave) balance_loss(a, s_part, s_count, *s_routed);
    __syncthreads();
  }
  for (int e = tid; e < a.experts; e += kSmallThreads) a.counts[e] = s_count[e];
  add_experts_before<kSmallThreads>(s_at, s_count, a.experts, s_waves);
  place_slots<kSmallThreads>(a, run, id0, s_at, s_rest);
}

// ---------------------------------------------------------------- backward

// A group's row of the gradient in LDS, where the chosen experts' parts are added to it: comparing every slot's
// expert with each of a lane's takes 3 instructions for each pair, 384 a wave with 8 slots and 16 values.
template <int L, int V>
constexpr bool kRowInLds = V >= 8;

// The formulas: with a the chosen weights over scale, g = scale * dw, c_e = d_loss * slope_e and p the softmax,
//   dz_e = p_e (c_e - sum_j p_j c_j)   and   normalize: + a_s (g_s - sum_j a_j g_j) at the chosen
//                                            else:      + p_e (g_e - sum_j p_j g_j), g 0 where not chosen.
// 65521 tokens of 256 float logits: 32 us for 138 MB, near the rate of a copy.
template <class T, int L, int V>
__global__ __launch_bounds__(kThreads) void route_gradient_kernel(ggk_route_gradient_args a, bool vectors) {
  using Z = Logit<T>;
  using C = Columns<L, V>;
  constexpr int W = C::W;
  constexpr int kGroups = kThreads / L;
  __shared__ alignas(16) float s_rows[kRowInLds<L, V> ? kGroups : 1][kRowInLds<L, V> ? L * V : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float d_loss = a.d_loss != nullptr ? *a.d_loss : 0.0f;
  // Without a loss, normalized weights depend on the chosen logits alone.
  const bool softmax = a.d_loss != nullptr || !a.normalize;
  float c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = C::expert(lane, j);
    c[j] = a.d_loss != nullptr && e < a.experts ? d_loss * a.slope[e] : 0.0f;
  }
  struct Loaded {
    T z[V];
    int id;
    float g;
  };
  auto load = [&](long long t0, Loaded& x) {
    const long long t = t0 + group;
    const bool in = t < a.tokens;
    const long long slot = t * a.slots + lane;
    x.id = in && lane < a.slots ? a.ids[slot] : -1;
    x.g = in && lane < a.slots && a.d_weights != nullptr ? a.scale * a.d_weights[slot] : 0.0f;
    if (softmax) {
      load_row<T, L, V>(static_cast<const T*>(a.logits) + (in ? t : 0) * a.ld, lane, in ? a.experts : 0, vectors,
                        Z::store(-__builtin_inff()), x.z);
    }
  };
  Loaded next;
  long long t0 = (long long)blockIdx.x * kGroups;
  const long long stride = (long long)gridDim.x * kGroups;
  load(t0, next);
  for (; t0 < a.tokens; t0 += stride) {
    const Loaded now = next;
    if (t0 + stride < a.tokens) load(t0 + stride, next);
    const long long t = t0 + group;
    const bool in = t < a.tokens;
    const bool has = now.id >= 0 && now.id < a.experts;
    const bool routed = group_any<L>(has);
    const float g = has ? now.g : 0.0f;
    // The chosen logits: again from memory (the cache has them), by the lanes of the slots.
    const float my_z = has ? Z::value((static_cast<const T*>(a.logits) + t * a.ld)[now.id]) : -__builtin_inff();
    float d[V], top = 0.0f, inv = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.0f;
    if (softmax) {
      top = -__builtin_inff();
      float total = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmaxf(top, Z::value(now.z[j]));
      top = group_max<L>(top);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = routed ? exp_of(Z::value(now.z[j]) - top) : 0.0f;
        total += d[j];
      }
      total = group_sum<L>(total);
      inv = routed ? 1.0f / total : 0.0f;
    }
    float my_a;
    if (a.normalize) {
      const float peak = group_max<L>(my_z);  // by every lane: exchanges are not made under a lane's condition
      const float e = has ? exp_of(my_z - peak) : 0.0f;
      my_a = e / group_sum<L>(e);
    } else {
      my_a = exp_of(my_z - top) * inv;
    }
    const float mean = group_sum<L>(has ? my_a * g : 0.0f);
    const float my_d = has ? my_a * (a.normalize ? g - mean : g) : 0.0f;
    if (softmax) {
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] *= inv;
        dot = fmaf(d[j], c[j], dot);
      }
      dot = group_sum<L>(dot) + (a.normalize ? 0.0f : mean);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = routed ? d[j] * (c[j] - dot) : 0.0f;
    }
    if (a.d_weights != nullptr) {
      if constexpr (kRowInLds<L, V>) {
        float* row = s_rows[group];
        typedef struct alignas(16) {
          float v[4];
        } Four;
#pragma unroll
        for (int j = 0; j < V; j += 4) *reinterpret_cast<Four*>(row + C::expert(lane, j)) = {d[j], d[j + 1], d[j + 2], d[j + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (a.distinct) {
          if (has) row[now.id] += my_d;
        } else {  // one slot after the other, so that an expert named twice is added in the slots' order
          for (int s = 0; s < a.slots; ++s) {
            if (lane == s && has) row[now.id] += my_d;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const Four x = *reinterpret_cast<const Four*>(row + C::expert(lane, j));
#pragma unroll
          for (int i = 0; i < 4; ++i) d[j + i] = x.v[i];
        }
      } else {
        for (int s = 0; s < a.slots; ++s) {
          const int id = __shfl(has ? now.id : -1, s, L);
          const float part = __shfl(my_d, s, L);
#pragma unroll
          for (int j = 0; j < V; ++j) d[j] += id == C::expert(lane, j) ? part : 0.0f;
        }
      }
    }
    T* out = static_cast<T*>(a.d_logits) + t * a.experts;
    typedef struct alignas(sizeof(T) * W) {
      T v[W];
    } Vector;
#pragma unroll
    for (int j = 0; j < V; j += W) {
      const int e = C::expert(lane, j);
      if (vectors) {
        if (in && e < a.experts) {
          Vector x;
#pragma unroll
          for (int i = 0; i < W; ++i) x.v[i] = Z::store(d[j + i]);
          *reinterpret_cast<Vector*>(out + e) = x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if (in && e + i < a.experts) out[e + i] = Z::store(d[j + i]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- launches

template <class T, int L, int V>
hipError_t launch_route(const ggk_route_args& a, Plan plan, hipStream_t stream) {
  const size_t width = a.experts + 1;
  const size_t wave_row = sizeof(int) * width;  // of every wave, beside what the workgroup shares
  plan.vectors = whole_vectors<T, V>(a.logits, a.tokens > 1 ? a.ld : 0, a.experts);
  if (is_small(a.tokens, a.experts)) {
    hipLaunchKernelGGL((route_small_kernel<T, L, V>), dim3(1), dim3(kSmallThreads),
                       sizeof(int) * (2 * width + 1) + kSmallThreads / kWave * wave_row, stream, a, plan.vectors);
    return hipGetLastError();
  }
  plan.run = a.loss != nullptr ? tokens_a_run(plan.rows / (kThreads / L)) : 0;
  const Workspace ws = carve(a.workspace, a.experts, plan.blocks);
  // A kernel of its own for runs: with them the one for fewer tokens spilled or lost 1%.
  auto rows_kernel = plan.run > 0 ? route_rows_kernel<T, L, V, true> : route_rows_kernel<T, L, V, false>;
  hipLaunchKernelGGL(rows_kernel, dim3(plan.blocks), dim3(kThreads),
                     sizeof(int) * (width + 1) + (a.loss != nullptr ? kThreads / kWave * wave_row : 0), stream, a, ws, plan);
  hipError_t st = hipGetLastError();
  if (st != hipSuccess) return st;
  if (plan.columns) {
    hipLaunchKernelGGL(route_columns_kernel, dim3((a.experts + kColumns) / kColumns), dim3(kThreads), 0, stream, a, ws,
                       plan.blocks);
    st = hipGetLastError();
    if (st != hipSuccess) return st;
  }
  hipLaunchKernelGGL(route_order_kernel, dim3(plan.blocks + (a.loss != nullptr ? 1 : 0)), dim3(kThreads),
                     sizeof(int) * 2 * width + kThreads / kWave * wave_row, stream, a, ws, plan);
  return hipGetLastError();
}

template <class T, int L, int V>
hipError_t launch_gradient(const ggk_route_gradient_args& a, hipStream_t stream) {
  const int groups = kThreads / L;
  const int blocks = (int)(((long long)a.tokens + groups - 1) / groups);
  const bool vectors = whole_vectors<T, V>(a.logits, a.tokens > 1 ? a.ld : 0, a.experts) &&
                       whole_vectors<T, V>(a.d_logits, a.experts, a.experts);
  hipLaunchKernelGGL((route_gradient_kernel<T, L, V>), dim3(blocks < 1024 ? blocks : 1024), dim3(kThreads), 0, stream, a,
                     vectors);
  return hipGetLastError();
}

// Lanes a token and values a lane: 16 lanes while a token's experts fit them at 16 values each and its slots
// fit one a lane, else the wave.
#define GG_ROUTE_FORMS(T, CALL)                                      \
  if (a.experts <= 256 && a.slots <= 16) {                           \
    return a.experts <= 16 ? CALL(T, 16, 1) : a.experts <= 32 ? CALL(T, 16, 2) : a.experts <= 64 ? CALL(T, 16, 4) \
           : a.experts <= 128 ? CALL(T, 16, 8) : CALL(T, 16, 16);    \
  }                                                                  \
  return a.experts <= 256 ? CALL(T, 64, 4) : a.experts <= 512 ? CALL(T, 64, 8) : CALL(T, 64, 16);

template <class T>
hipError_t route_of_type(const ggk_route_args& a, const Plan& plan, hipStream_t stream) {
#define GG_CALL(T, L, V) launch_route<T, L, V>(a, plan, stream)
  GG_ROUTE_FORMS(T, GG_CALL)
#undef GG_CALL
}

template <class T>
hipError_t gradient_of_type(const ggk_route_gradient_args& a, hipStream_t stream) {
#define GG_CALL(T, L, V) launch_gradient<T, L, V>(a, stream)
  GG_ROUTE_FORMS(T, GG_CALL)
#undef GG_CALL
}

bool bad_sizes(int tokens, int experts, int slots, int type, long long ld) {
  return tokens < 0 || experts < 1 || experts > kMaxExperts || slots < 1 || slots > GGK_ROUTE_MAX_SLOTS ||
         (type != GGK_TYPE_F32 && type != GGK_TYPE_F16 && type != GGK_TYPE_BF16) || (tokens > 1 && ld < experts) ||
         (long long)tokens * slots > GGK_ROUTE_MAX_TOTAL_SLOTS;
}

}  // namespace

extern "C" size_t ggk_route_workspace(int tokens, int experts) {
  if (tokens < 0 || experts < 1 || experts > kMaxExperts || is_small(tokens, experts)) return 0;
  return sizeof(int) * workspace_ints(experts, plan_blocks(tokens, experts).blocks);
}

extern "C" hipError_t ggk_route_check(const ggk_route_args* args) {
  if (args == nullptr) return hipErrorInvalidValue;
  const ggk_route_args& a = *args;
  if (bad_sizes(a.tokens, a.experts, a.slots, a.type, a.ld)) return hipErrorInvalidValue;
  if (a.given_ids == nullptr && a.slots > a.experts) return hipErrorInvalidValue;
  if (a.workspace_bytes < ggk_route_workspace(a.tokens, a.experts) || reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) {
    return hipErrorInvalidValue;
  }
  if (a.counts == nullptr || (a.workspace == nullptr && !is_small(a.tokens, a.experts)) ||
      (a.loss == nullptr) != (a.slope == nullptr) ||
      (a.tokens > 0 && (a.logits == nullptr || a.weights == nullptr || a.ids == nullptr || a.order == nullptr))) {
    return hipErrorInvalidDevicePointer;
  }
  return hipSuccess;
}

extern "C" hipError_t ggk_route(const ggk_route_args* args, hipStream_t stream) {
  const hipError_t st = ggk_route_check(args);
  if (st != hipSuccess) return st;
  const ggk_route_args& a = *args;
  const Plan plan = plan_blocks(a.tokens, a.experts);
  return a.type == GGK_TYPE_F32 ? route_of_type<float>(a, plan, stream)
         : a.type == GGK_TYPE_F16 ? route_of_type<_Float16>(a, plan, stream)
                                  : route_of_type<__hip_bfloat16>(a, plan, stream);
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
  return args->type == GGK_TYPE_F32 ? gradient_of_type<float>(*args, stream)
         : args->type == GGK_TYPE_F16 ? gradient_of_type<_Float16>(*args, stream)
                                      : gradient_of_type<__hip_bfloat16>(*args, stream);
}
