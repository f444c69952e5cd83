// Router of a mixture-of-experts block: top-k gate, rows per expert and balance loss from the
// router's logits in one pass over them, and the gradient with respect to the logits.
//
// For each token t (a row of E logits l) that is not masked and has an expert above -inf:
//   score = softmax(l) or sigmoid(l),  p = score / sum(score)
//   ids   = the k largest of l (of score + bias where a bias is given), ties to the lowest index
//   w_j   = scale * score[ids_j]   (divided by the sum of the k chosen scores if renormalised)
// Over the V valid tokens: counts[e] = how often e was chosen and
//   loss  = E / (k V^2) * sum_e counts[e] * sum_t p[t, e].
// Gradient, with g_j = dL/dw_j * scale, a_e = dL/dloss * E counts[e] / (k V^2) (counts held fixed):
//   renormalised: G = scatter((g_j - sum_i g_i q_i) q_j) with q the shares, the chosen scores over their sum
//     softmax: dl_i = G_i + p_i (a_i - sum_j a_j p_j)
//     sigmoid: dl_i = (G_i + p_i (a_i - sum_j a_j p_j)) (1 - s_i)
//   not renormalised, d = scatter(g):
//     softmax: dl_i = p_i (d_i + a_i - sum_j (d_j + a_j) p_j)
//     sigmoid: dl_i = (d_i s_i + p_i (a_i - sum_j a_j p_j)) (1 - s_i)
// Scores too small for 32 bits still have shares and probabilities: sums of scores below 2^-60 are taken again
// relative to the largest logit in them (there a sigmoid is e^l within 2^-60).
//
// Sixteen lanes take a row (32 where the choice is long or the experts are many), lane l the experts l,
// l + 16, ...; a row is read once and its next row's loads are in flight meanwhile.  Bound by the latency of
// a row's chain (sort, list, rank, sums; 359 instructions): 116 registers a thread leave 16 warps an
// SM, a quarter of its slots, which issue in 59% of the cycles; DRAM is 17% busy.  One B200, calls in a row,
// 32,768 x 256 FP32, k = 8 with the balance loss 21.0 us forward (1.7 TB/s) and 17.1 us backward (4.1 TB/s),
// 22.0 and 17.4 us with sigmoid scores; 64 x 256 4.9 us and 3.2 us; 32,768 x 512, k = 16 44 and 30 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "cdg_b200.h"
#include "cdg_ptx.cuh"
#include "cdg_rows.cuh"

namespace cdg {
namespace {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 32;  // lane j keeps the row's j-th choice
constexpr unsigned kAll = 0xffffffffu;

// NaN counts as -inf (never chosen), +inf as the largest finite value, -0 as 0.
__device__ __forceinline__ float clean_logit(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX) + 0.0f; }

// Keys whose unsigned order is the values' order.  Keys below kFirstKey, that of -FLT_MAX, cannot
// be chosen (-inf, and 0 for what was taken).
constexpr uint32_t kFirstKey = 0x00800000u;
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key ^ (key & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}

// Fast exponential and division (errors of a few units in the last place): the gate's weights
// and gradients stay within 1e-6 of the exact ones.
__device__ __forceinline__ float exp_fast(float v) {
  // 2^(v log2 e), results below the normal range taken as 0: no weight or gradient needs them
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}
constexpr float kTiny = 8.673617e-19f;  // 2^-60
__device__ __forceinline__ float sigmoid_fast(float v) { return __fdividef(1.0f, 1.0f + exp_fast(-v)); }

// Sum and maximum over the lanes of a row.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// Where the lane keeps the larger value in each stage of lanes_sorted, a bit per stage.
template <int LANES>
__device__ __forceinline__ uint32_t sort_sides(int sub) {
  uint32_t sides = 0;
  int stage = 0;
#pragma unroll
  for (int size = 2; size <= LANES; size *= 2)
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2, ++stage)
      if (((sub & j) == 0) == ((sub & size & (LANES - 1)) == 0)) sides |= 1u << stage;
  return sides;
}

// One value per lane, sorted over the lanes of a row in falling order (a bitonic network).
template <int LANES>
__device__ __forceinline__ float lanes_sorted(float v, uint32_t sides) {
  int stage = 0;
#pragma unroll
  for (int size = 2; size <= LANES; size *= 2)
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2, ++stage) {
      const float other = __shfl_xor_sync(kAll, v, j);
      v = sides & (1u << stage) ? fmaxf(v, other) : fminf(v, other);
    }
  return v;
}

constexpr int kListed = 32;   // candidates of a row that are ranked by counting
constexpr int kPerLane = 7;   // of them, those of one lane
struct Candidates {
  // x the value, y the expert; a full four are compared at a time
  alignas(16) float2 listed[kListed + 4];
};

// The k experts of the largest values of a row, of equal values the lowest expert first: lane j of the
// row's LANES gets the j-th (x its value, y the expert), or y = -1 where no value that can be chosen is
// left.  v[i] is that of expert i * LANES + sub (NaN and -inf cannot be chosen, +inf counts as the
// largest finite value); most is the row's largest value and kth the k-th largest of the lanes'
// maxima, a lower bound of the k-th largest value.  Few values reach it (with 256 experts and k = 8
// about ten), so: they are listed, each with its expert; each lane takes one of the list and counts how
// many of the others go before it.  A list of more than 32, a lane with more than seven of them (many
// equal values, or k near 32) or a value of +inf is chosen from round by round, a maximum over the lanes
// each; at 32,768 x 256, k = 8 that alone took the kernel 43 us.
template <int N, int LANES>
__device__ __forceinline__ float2 choose(const float (&v)[N], float most, float kth, int k, int lane, Candidates& c) {
  const int sub = lane & (LANES - 1);
  const float bound = fmaxf(kth, -FLT_MAX);
  int reach = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) reach += v[i] >= bound ? 1 : 0;
  // the lane's place in the list: what the lanes before it have, from the bits of their counts
  const unsigned b0 = __ballot_sync(kAll, reach & 1), b1 = __ballot_sync(kAll, reach & 2), b2 = __ballot_sync(kAll, reach & 4);
  const unsigned row = LANES == 32 ? kAll : 0xFFFFu << (lane & 16), below = row & ((1u << lane) - 1u);
  const int count = __popc(b0 & row) + 2 * __popc(b1 & row) + 4 * __popc(b2 & row);
  if (!__any_sync(kAll, count > kListed || reach > kPerLane || most > FLT_MAX)) {
    int place = __popc(b0 & below) + 2 * __popc(b1 & below) + 4 * __popc(b2 & below);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[i] >= bound) c.listed[place++] = make_float2(v[i], __int_as_float(i * LANES + sub));
    if (sub < 4) c.listed[count + sub] = make_float2(-INFINITY, 0.0f);
    __syncwarp();
    float2 own[kListed / LANES];
    int before[kListed / LANES];
#pragma unroll
    for (int h = 0; h < kListed / LANES; ++h) {
      before[h] = k;
      if (h * LANES + sub < count) {
        own[h] = c.listed[h * LANES + sub];
        const int expert = __float_as_int(own[h].y);
        int n = 0;
        auto goes_before = [&](float value, float index) {
          if (value > own[h].x || (value == own[h].x && __float_as_int(index) < expert)) ++n;
        };
        for (int i = 0; i < count; i += 4) {
          const float4 two = *reinterpret_cast<const float4*>(&c.listed[i]);
          const float4 more = *reinterpret_cast<const float4*>(&c.listed[i + 2]);
          goes_before(two.x, two.y);
          goes_before(two.z, two.w);
          goes_before(more.x, more.y);
          goes_before(more.z, more.w);
        }
        before[h] = n;
      }
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < kListed / LANES; ++h)
      if (before[h] < k) c.listed[before[h]] = own[h];
    __syncwarp();
    const float2 got = sub < min(count, k) ? c.listed[sub] : make_float2(0.0f, __int_as_float(-1));
    __syncwarp();
    return got;
  }
  float2 got = make_float2(0.0f, __int_as_float(-1));
  uint32_t key[N], mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    key[i] = order_key(clean_logit(v[i]));
    mine = max(mine, key[i]);
  }
  for (int j = 0; j < k; ++j) {
    uint32_t best = mine;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(kAll, best, o));
    int winner = 0x7fffffff;
    if (best >= kFirstKey && mine == best) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (key[i] == best) winner = i * LANES + sub;
    }
    const int own = winner;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) winner = min(winner, __shfl_xor_sync(kAll, winner, o));
    if (best >= kFirstKey) {  // the warp's other row may have more or fewer
      if (own == winner) {
        mine = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i * LANES + sub == winner) key[i] = 0;
          mine = max(mine, key[i]);
        }
      }
      if (sub == j) got = make_float2(key_value(best), __int_as_float(winner));
    }
  }
  return got;
}

struct Route {
  const void* logits;
  int64_t stride;
  const uint8_t* mask;
  const float* bias;
  int64_t T;
  int E, k;
  int sigmoid, renormalize, balance, clustered;
  float scale;
  float* weights;
  int32_t *ids, *counts, *tokens;
  float* loss;
  // zeroed before the launch, unless the grid is one cluster: sum of p per expert in units of 2^-40, rows per
  // expert, valid tokens, finished CTAs
  unsigned long long* psum;
  int32_t *acc_counts, *acc_tokens, *ticket;
};

// Sums of p leave a CTA as 64-bit integers in units of 2^-40, so that the order in which the
// CTAs add them does not change the result.  2^23 tokens fit.
constexpr float kFixed = 1099511627776.0f;
constexpr unsigned kClusterCtas = 8;  // as many as a cluster may always have
constexpr int64_t kRouteMaxTokens = int64_t(1) << 23;

// Sum of one value per thread, in a fixed order; thread 0 gets it.
template <int WARPS>
__device__ double cta_sum64(double v, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < WARPS; ++i) v += scratch[i];
  return v;
}

// N experts per lane, LANES lanes per row.  Dynamic shared memory: E counts, then one row of E sums of p
// per row that the CTA works on at a time.
template <typename T, int N, int LANES, bool BIAS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, N <= 16 ? 2 : 1) moe_route_kernel(const Route a) {
  constexpr int kRows = 32 / LANES;  // per warp
  extern __shared__ int32_t route_smem[];
  __shared__ double scratch[WARPS];
  __shared__ int32_t s_tokens, s_last;
  __shared__ Candidates s_list[WARPS * kRows];
  int32_t* s_counts = route_smem;
  float* s_psum = reinterpret_cast<float*>(route_smem + a.E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LANES - 1);
  const int slot = threadIdx.x / LANES;  // of the CTA's rows
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_counts[e] = 0;
  if (threadIdx.x == 0) s_tokens = 0;
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();

  const T* logits = static_cast<const T*>(a.logits);
  const uint32_t sides = sort_sides<LANES>(sub);
  float psum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) psum[i] = 0.0f;
  int32_t tokens = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * WARPS * kRows;
  T next[N];
  const int left = a.E - sub;  // expert i * LANES + sub exists where i * LANES < left
  const bool full = a.E == N * LANES;
  auto load_row = [&](int64_t row) {
    const T* at = logits + min(row, a.T - 1) * a.stride + sub;
    if (full) {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = at[i * LANES];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = i * LANES < left ? at[i * LANES] : from_f<T>(-INFINITY);
    }
  };
  int64_t first = (static_cast<int64_t>(blockIdx.x) * WARPS + warp) * kRows;  // of the warp's rows
  if (first < a.T) load_row(first + lane / LANES);
  for (; first < a.T; first += step) {
    const int64_t row = first + lane / LANES;
    float v[N];
    float top = -INFINITY;  // fmaxf passes over NaN
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = to_f(next[i]);
      top = fmaxf(top, v[i]);
    }
    if (first + step < a.T) load_row(row + step);
    bool valid = row < a.T && (!a.mask || a.mask[row]);
    float2 got;
    float m;
    if constexpr (!BIAS) {
      top = lanes_sorted<LANES>(top, sides);
      m = __shfl_sync(kAll, top, 0, LANES);
      got = choose<N, LANES>(v, m, __shfl_sync(kAll, top, a.k - 1, LANES), a.k, lane, s_list[slot]);
    } else {
      m = lanes_max<LANES>(top);
    }
    valid = valid && m > -INFINITY;
    m = fminf(m, FLT_MAX);
    const float shift = a.sigmoid || m == -INFINITY ? 0.0f : m;
    float inv = 1.0f;   // 1 / sum of exponentials (softmax)
    float part = 0.0f;  // 1 / sum of scores
    if (a.balance || BIAS || !a.renormalize) {
      float score[N];
      float total = 0.0f;
      if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < N; ++i) total += score[i] = sigmoid_fast(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) total += score[i] = exp_fast(v[i] - shift);
      }
      total = lanes_sum<LANES>(total);
      if (__any_sync(kAll, !(total < INFINITY))) {  // NaN or +inf among the logits
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float l = row < a.T && i * LANES < left ? clean_logit(to_f(logits[row * a.stride + i * LANES + sub])) : -INFINITY;
          score[i] = a.sigmoid ? sigmoid_fast(l) : exp_fast(l - shift);
          total += score[i];
        }
        total = lanes_sum<LANES>(total);
      }
      part = total > 0.0f ? __fdividef(1.0f, total) : 0.0f;
      if (!a.sigmoid) inv = part;
      if constexpr (BIAS) {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          // NaN and -inf stay what they are: not chosen
          v[i] = v[i] >= -FLT_MAX ? clean_logit(score[i] * inv + __ldg(a.bias + i * LANES + sub)) : -INFINITY;
          top = fmaxf(top, v[i]);
        }
        top = lanes_sorted<LANES>(top, sides);
        const float most = __shfl_sync(kAll, top, 0, LANES);  // by every lane: valid differs between rows
        valid = valid && most > -INFINITY;                    // a bias of -inf may have left nothing
        got = choose<N, LANES>(v, most, __shfl_sync(kAll, top, a.k - 1, LANES), a.k, lane, s_list[slot]);
      }
      if (a.balance) {
        if (!valid) part = 0.0f;
        if (a.sigmoid && __any_sync(kAll, valid && total < kTiny)) {  // rare: every logit below -41
          float again = 0.0f;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (total < kTiny) {
              const float l = row < a.T && i * LANES < left ? clean_logit(to_f(logits[row * a.stride + i * LANES + sub])) : -INFINITY;
              score[i] = exp_fast(l - (m == -INFINITY ? 0.0f : m));
            }
            again += score[i];
          }
          again = lanes_sum<LANES>(again);
          part = valid && again > 0.0f ? __fdividef(1.0f, again) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) psum[i] = fmaf(score[i], part, psum[i]);
      }
    }
    const int32_t id = valid ? __float_as_int(got.y) : -1;
    float w = 0.0f, l = -INFINITY;
    if (id >= 0) {
      // the value is the logit itself, unless a bias went into it
      l = BIAS ? clean_logit(to_f(logits[row * a.stride + id])) : got.x;
      w = a.sigmoid ? sigmoid_fast(l) : exp_fast(l - m) * inv;
      atomicAdd(&s_counts[id], 1);
    }
    if (valid) ++tokens;
    if (a.renormalize) {
      float total = lanes_sum<LANES>(w);
      // without a bias the softmax's largest score is among the chosen
      if ((BIAS || a.sigmoid) && __any_sync(kAll, id >= 0 && total < kTiny)) {
        const float most = lanes_max<LANES>(l);
        if (id >= 0 && total < kTiny) w = exp_fast(l - most);
        total = lanes_sum<LANES>(w);
      }
      w = total <= 0.0f ? 0.0f : w == total ? 1.0f : __fdividef(w, total);  // a lone choice: 1 exactly
    }
    if (sub < a.k && row < a.T) {
      a.ids[row * a.k + sub] = id;
      a.weights[row * a.k + sub] = w * a.scale;
    }
  }

  if (sub == 0 && tokens) atomicAdd(&s_tokens, tokens);
  if (a.balance) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * LANES < left) s_psum[slot * a.E + i * LANES + sub] = psum[i];
  }
  __syncthreads();
  if (a.clustered) {  // the grid is one cluster: its first CTA reads the others' sums, in rank order
    for (int e = threadIdx.x; a.balance && e < a.E; e += blockDim.x) {
      float p = s_psum[e];
      for (int i = 1; i < WARPS * kRows; ++i) p += s_psum[i * a.E + e];
      s_psum[e] = p;
    }
    cluster_sync();
    if (blockIdx.x == 0) {
      double sum = 0.0;
      for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        int32_t count[kClusterCtas];
        float p[kClusterCtas];
#pragma unroll
        for (int r = 0; r < kClusterCtas; ++r) {
          count[r] = 0;
          p[r] = 0.0f;
          if (r < gridDim.x) {
            asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(count[r]) : "r"(cluster_addr(s_counts + e, r)));
            if (a.balance) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p[r]) : "r"(cluster_addr(s_psum + e, r)));
          }
        }
        int32_t count_all = 0;
        double p_all = 0.0;
#pragma unroll
        for (int r = 0; r < kClusterCtas; ++r) {
          count_all += count[r];
          p_all += p[r];
        }
        a.counts[e] = count_all;
        sum += p_all * count_all;
      }
      if (a.balance) sum = cta_sum64<WARPS>(sum, scratch);
      if (threadIdx.x == 0) {
        int32_t tokens_all = 0;
        for (int r = 0; r < gridDim.x; ++r) {
          int32_t n;
          asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(n) : "r"(cluster_addr(&s_tokens, r)));
          tokens_all += n;
        }
        const double n = tokens_all > 0 ? tokens_all : 1;
        *a.tokens = tokens_all;
        if (a.balance) *a.loss = static_cast<float>(sum * a.E / a.k / n / n);
      }
    }
    cluster_sync();  // no CTA leaves while its sums are read
    return;
  }
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    if (s_counts[e]) atomicAdd(&a.acc_counts[e], s_counts[e]);
    if (a.balance) {
      float p = 0.0f;
      for (int i = 0; i < WARPS * kRows; ++i) p += s_psum[i * a.E + e];
      atomicAdd(&a.psum[e], static_cast<unsigned long long>(__float2ull_rn(p * kFixed)));
    }
  }
  if (threadIdx.x == 0 && s_tokens) atomicAdd(a.acc_tokens, s_tokens);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(a.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    const int32_t count = __ldcg(a.acc_counts + e);
    a.counts[e] = count;
    if (a.balance) sum += static_cast<double>(count) * (static_cast<double>(__ldcg(a.psum + e)) / static_cast<double>(kFixed));
  }
  const int32_t tokens_all = __ldcg(a.acc_tokens);
  if (a.balance) sum = cta_sum64<WARPS>(sum, scratch);
  if (threadIdx.x == 0) {
    const double n = tokens_all > 0 ? tokens_all : 1;
    *a.tokens = tokens_all;
    if (a.balance) *a.loss = static_cast<float>(sum * a.E / a.k / n / n);
  }
}

// The workspace's sums to zero.  A kernel and not a memset, so that the next kernel starts while it runs.
__global__ void __launch_bounds__(256) route_clear_kernel(uint32_t* words, int n) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) words[i] = 0;
}

struct RouteBwd {
  const void* logits;
  int64_t stride;
  const int32_t* ids;
  const float* gw;     // [T, k] or null
  const float* gloss;  // [1] or null
  const int32_t *counts, *tokens;
  int64_t T;
  int E, k;
  int sigmoid, renormalize;
  float scale;
  void* dlogits;
  int64_t d_stride;
};

// N experts per lane, LANES lanes per row.  Dynamic shared memory: E floats per row that the CTA works on
// at a time, the scattered gradient of the chosen scores (zero between rows).
template <typename T, int N, int LANES, bool SIGMOID, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, N <= 16 ? 2 : 1) moe_route_backward_kernel(const RouteBwd a) {
  constexpr int kRows = 32 / LANES;  // per warp
  extern __shared__ float s_grad[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LANES - 1);
  float* sg = s_grad + static_cast<int>(threadIdx.x / LANES) * a.E;
  for (int e = sub; e < a.E; e += LANES) sg[e] = 0.0f;
  __syncwarp();
  grid_dependency_wait();
  grid_launch_dependents();
  const int left = a.E - sub;  // expert i * LANES + sub exists where i * LANES < left
  float load[N];               // a_e of the lane's experts
#pragma unroll
  for (int i = 0; i < N; ++i) load[i] = 0.0f;
  if (a.gloss) {
    const float n = static_cast<float>(max(*a.tokens, 1));
    const float f = *a.gloss * (static_cast<float>(a.E) / static_cast<float>(a.k)) / n / n;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * LANES < left) load[i] = f * static_cast<float>(a.counts[i * LANES + sub]);
  }
  const T* logits = static_cast<const T*>(a.logits);
  const int64_t step = static_cast<int64_t>(gridDim.x) * WARPS * kRows;
  T next[N];
  int32_t next_id = -1;
  float next_g = 0.0f;
  auto load_row = [&](int64_t row) {
    const T* at = logits + min(row, a.T - 1) * a.stride + sub;
#pragma unroll
    for (int i = 0; i < N; ++i) next[i] = i * LANES < left ? at[i * LANES] : from_f<T>(-INFINITY);
    next_id = -1;
    if (sub < a.k && row < a.T) {
      next_id = __ldg(a.ids + row * a.k + sub);
      if (a.gw) next_g = __ldg(a.gw + row * a.k + sub);
    }
  };
  int64_t first = (static_cast<int64_t>(blockIdx.x) * WARPS + warp) * kRows;  // of the warp's rows
  if (first < a.T) load_row(first + lane / LANES);
  for (; first < a.T; first += step) {
    const int64_t row = first + lane / LANES;
    float s[N];
    float m = -INFINITY;  // fmaxf passes over NaN
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = to_f(next[i]);
      m = fmaxf(m, s[i]);
    }
    const int32_t id = next_id >= 0 && next_id < a.E ? next_id : -1;
    float g = id >= 0 ? next_g * a.scale : 0.0f;
    if (first + step < a.T) load_row(row + step);
    T* out = static_cast<T*>(a.dlogits) + row * a.d_stride + sub;
    const unsigned chosen_lanes = __ballot_sync(kAll, id >= 0);
    const bool live = LANES == 32 ? chosen_lanes != 0 : (chosen_lanes & (0xFFFFu << (lane & 16))) != 0;
    if (chosen_lanes == 0) {  // masked tokens: no gradient
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * LANES < left && row < a.T) out[i * LANES] = from_f<T>(0.0f);
      continue;
    }
    float shift = 0.0f;
    if constexpr (!SIGMOID) {
      m = fminf(lanes_max<LANES>(m), FLT_MAX);
      shift = m == -INFINITY ? 0.0f : m;
    }
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) total += s[i] = SIGMOID ? sigmoid_fast(s[i]) : exp_fast(s[i] - shift);
    total = lanes_sum<LANES>(total);
    if (__any_sync(kAll, !(total < INFINITY))) {  // NaN or +inf among the logits
      total = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float l = row < a.T && i * LANES < left ? clean_logit(to_f(logits[row * a.stride + i * LANES + sub])) : -INFINITY;
        total += s[i] = SIGMOID ? sigmoid_fast(l) : exp_fast(l - shift);
      }
      total = lanes_sum<LANES>(total);
    }
    float mul = 1.0f;  // the sigmoids are s times this
    if constexpr (SIGMOID) {
      if (__any_sync(kAll, live && total < kTiny)) {  // rare: every logit below -41
        float top = -INFINITY, again = 0.0f;
        auto logit = [&](int i) {
          return row < a.T && i * LANES < left ? clean_logit(to_f(logits[row * a.stride + i * LANES + sub])) : -INFINITY;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, logit(i));
        top = lanes_max<LANES>(top);
        if (top == -INFINITY) top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (total < kTiny) s[i] = exp_fast(logit(i) - top);
          again += s[i];
        }
        again = lanes_sum<LANES>(again);
        if (total < kTiny) {
          mul = exp_fast(top);
          total = again;
        }
      }
    }
    // a row without a choice: all terms zero
    const float inv = live && total > 0.0f ? __fdividef(1.0f, total) : 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (SIGMOID)
        s[i] = live ? s[i] : 0.0f;
      else
        s[i] *= inv;  // the scores are the probabilities
    }
    if (a.gw) {
      if (a.renormalize) {
        float c = 0.0f, l = -INFINITY;
        if (id >= 0) {
          l = clean_logit(to_f(logits[row * a.stride + id]));
          c = SIGMOID ? sigmoid_fast(l) : exp_fast(l - shift) * inv;
        }
        float sum = lanes_sum<LANES>(c);
        if (__any_sync(kAll, id >= 0 && sum < kTiny)) {
          const float most = lanes_max<LANES>(l);
          if (id >= 0 && sum < kTiny && most > -INFINITY) c = exp_fast(l - most);
          sum = lanes_sum<LANES>(c);
        }
        const float share = sum <= 0.0f ? 0.0f : c == sum ? 1.0f : __fdividef(c, sum);  // nothing moves a share of 1
        g = (g - lanes_sum<LANES>(g * share)) * share;
      }
      if (id >= 0) atomicAdd(&sg[id], g);
      __syncwarp();
    }
    // SHARES: what was scattered is G of the head's formulas, else d
    auto finish = [&](auto shares) {
      constexpr bool SHARES = decltype(shares)::value;
      float d[N];
      float dot = 0.0f;  // of what meets the probabilities
#pragma unroll
      for (int i = 0; i < N; ++i) {
        d[i] = a.gw && i * LANES < left ? sg[i * LANES + sub] : 0.0f;
        if constexpr (!SIGMOID && !SHARES) d[i] += load[i];
        dot = fmaf(SIGMOID || SHARES ? load[i] : d[i], s[i], dot);
      }
      dot = lanes_sum<LANES>(dot);
      if (a.gw) {
        __syncwarp();
        if (id >= 0) sg[id] = 0.0f;
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float v;
        if constexpr (SIGMOID) {
          const float by_p = (load[i] - dot * inv) * inv;
          v = (SHARES ? fmaf(s[i], by_p, d[i]) : s[i] * fmaf(d[i], mul, by_p)) * fmaf(-s[i], mul, 1.0f);
        } else {
          v = SHARES ? fmaf(s[i], load[i] - dot, d[i]) : s[i] * (d[i] - dot);
        }
        if (i * LANES < left && row < a.T) out[i * LANES] = from_f<T>(v);
      }
    };
    if (a.gw && a.renormalize)
      finish(std::true_type());
    else
      finish(std::false_type());
  }
}

constexpr int kRouteWarps = 8;
// Lanes per row.  What a row costs beside its experts (sorting, listing and ranking, the sums) is most
// of it, and two rows to a warp share that; but 16 lanes' maxima bound only a short choice well, and
// more experts would not stay in registers.  Forward at 32,768 x 256, k = 8: 20.8 us with 16 lanes, 26.3
// with 32; at 32,768 x 32, k = 2: 12.9 and 19.8 us.
int lanes_per_row(int E, int k) { return k <= 8 && E <= 256 ? 16 : 32; }
int64_t rows_per_cta(int E, int k) { return kRouteWarps * 32 / lanes_per_row(E, k); }
// What one cluster does in one pass runs in one cluster, which needs neither zeroed sums nor a last
// CTA: 64 x 256, k = 8 in 4.9 us, over the GPU in 6.1 us; two passes cost more than the whole grid.
bool one_cluster(int64_t T, int E, int k) { return T <= int64_t(kClusterCtas) * rows_per_cta(E, k); }

// CTAs of a kernel that an SM holds at once (looked up once: the library runs on one kind of device).
template <typename K>
int resident_ctas(K kernel, int threads, size_t smem, std::atomic<int>* known) {
  int n = known->load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
    known->store(n, std::memory_order_relaxed);
  }
  return n;
}

template <typename T, int N, int LANES, bool BIAS>
int launch_route_as(const Route& a, cudaStream_t st) {
  constexpr int kRows = kRouteWarps * 32 / LANES;
  // the largest dynamic shared memory of this N, so that one look-up serves every call
  static std::atomic<int> known{0};
  const int per_sm = resident_ctas(moe_route_kernel<T, N, LANES, BIAS, kRouteWarps>, kRouteWarps * 32,
                                   size_t(N) * LANES * 4 * (kRows + 1), &known);
  const int64_t ctas = (a.T + kRows - 1) / kRows;
  const size_t smem = a.E * 4 + (a.balance ? size_t(kRows) * a.E * 4 : 0);
  const auto kernel = moe_route_kernel<T, N, LANES, BIAS, kRouteWarps>;
  if (a.clustered) {
    unsigned cluster = 1;
    while (cluster < kClusterCtas && cluster < ctas) cluster *= 2;
    return launch_clusters(kernel, dim3(cluster), cluster, kRouteWarps * 32, smem, st, a);
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ctas, int64_t(sm_count()) * per_sm));
  return launch(kernel, dim3(grid), kRouteWarps * 32, smem, st, a);
}

template <typename T, int N, int LANES>
int launch_route(const Route& a, cudaStream_t st) {
  return a.bias ? launch_route_as<T, N, LANES, true>(a, st) : launch_route_as<T, N, LANES, false>(a, st);
}

template <typename T, int N, int LANES, bool SIGMOID>
int launch_route_backward_as(const RouteBwd& a, cudaStream_t st) {
  constexpr int kRows = kRouteWarps * 32 / LANES;
  static std::atomic<int> known{0};
  const auto kernel = moe_route_backward_kernel<T, N, LANES, SIGMOID, kRouteWarps>;
  const int per_sm = resident_ctas(kernel, kRouteWarps * 32, size_t(N) * LANES * 4 * kRows, &known);
  const int64_t ctas = (a.T + kRows - 1) / kRows;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ctas, int64_t(sm_count()) * per_sm));
  return launch(kernel, dim3(grid), kRouteWarps * 32, size_t(kRows) * a.E * 4, st, a);
}

template <typename T, int N, int LANES>
int launch_route_backward(const RouteBwd& a, cudaStream_t st) {
  return a.sigmoid ? launch_route_backward_as<T, N, LANES, true>(a, st) : launch_route_backward_as<T, N, LANES, false>(a, st);
}

template <typename T>
int dispatch_route(const Route& a, cudaStream_t st) {
  if (lanes_per_row(a.E, a.k) == 16) {
    const int n = (a.E + 15) / 16;
    if (n <= 4) return launch_route<T, 4, 16>(a, st);
    if (n <= 8) return launch_route<T, 8, 16>(a, st);
    if (n <= 12) return launch_route<T, 12, 16>(a, st);
    return launch_route<T, 16, 16>(a, st);
  }
  const int n = (a.E + 31) / 32;
  if (n <= 2) return launch_route<T, 2, 32>(a, st);
  if (n <= 8) return launch_route<T, 8, 32>(a, st);
  if (n <= 16) return launch_route<T, 16, 32>(a, st);
  return launch_route<T, 32, 32>(a, st);
}

template <typename T>
int dispatch_route_backward(const RouteBwd& a, cudaStream_t st) {
  if (lanes_per_row(a.E, a.k) == 16) {
    const int n = (a.E + 15) / 16;
    if (n <= 4) return launch_route_backward<T, 4, 16>(a, st);
    if (n <= 8) return launch_route_backward<T, 8, 16>(a, st);
    if (n <= 12) return launch_route_backward<T, 12, 16>(a, st);
    return launch_route_backward<T, 16, 16>(a, st);
  }
  const int n = (a.E + 31) / 32;
  if (n <= 2) return launch_route_backward<T, 2, 32>(a, st);
  if (n <= 8) return launch_route_backward<T, 8, 32>(a, st);
  if (n <= 16) return launch_route_backward<T, 16, 32>(a, st);
  return launch_route_backward<T, 32, 32>(a, st);
}

}  // namespace
}  // namespace cdg

extern "C" {

size_t cdg_moe_route_workspace_bytes(int64_t E) {
  if (E <= 0 || E > cdg::kRouteMaxExperts) return 0;
  return static_cast<size_t>(E) * 12 + 8;
}

int cdg_moe_route(const cdg_route_args* g, void* workspace, size_t workspace_bytes, cdg_stream_t stream) {
  using namespace cdg;
  if (!g || g->T < 0 || g->E <= 0 || g->topk <= 0 || g->topk > g->E || !row_dtype(g->dtype))
    return CDG_ERR_INVALID_ARGUMENT;
  if (g->scoring != CDG_SCORE_SOFTMAX && g->scoring != CDG_SCORE_SIGMOID) return CDG_ERR_INVALID_ARGUMENT;
  if (g->E > kRouteMaxExperts || g->topk > kRouteMaxTopk || g->T > kRouteMaxTokens) return CDG_ERR_UNSUPPORTED;
  if (!g->counts || !g->tokens || (g->T > 0 && (!g->logits || !g->weights || !g->ids))) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(element_size(g->dtype), {g->logits}) ||
      !on_boundary(4, {g->bias, g->weights, g->ids, g->counts, g->tokens, g->loss}))
    return CDG_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < cdg_moe_route_workspace_bytes(g->E)) return CDG_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return CDG_ERR_ALIGNMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (g->T == 0) {
    if (cudaMemsetAsync(g->counts, 0, g->E * sizeof(int32_t), st) != cudaSuccess ||
        cudaMemsetAsync(g->tokens, 0, sizeof(int32_t), st) != cudaSuccess ||
        (g->loss && cudaMemsetAsync(g->loss, 0, sizeof(float), st) != cudaSuccess))
      return CDG_ERR_CUDA;
    return CDG_OK;
  }
  Route a{};
  a.clustered = one_cluster(g->T, static_cast<int>(g->E), static_cast<int>(g->topk));
  a.logits = g->logits;
  a.stride = g->stride;
  a.mask = g->token_mask;
  a.bias = g->bias;
  a.T = g->T;
  a.E = static_cast<int>(g->E);
  a.k = static_cast<int>(g->topk);
  a.sigmoid = g->scoring == CDG_SCORE_SIGMOID;
  a.renormalize = g->renormalize != 0;
  a.balance = g->loss != nullptr;
  a.scale = g->scale;
  a.weights = g->weights;
  a.ids = g->ids;
  a.counts = g->counts;
  a.tokens = g->tokens;
  a.loss = g->loss;
  a.psum = static_cast<unsigned long long*>(workspace);
  a.acc_counts = reinterpret_cast<int32_t*>(a.psum + a.E);
  a.acc_tokens = a.acc_counts + a.E;
  a.ticket = a.acc_tokens + 1;
  if (!a.clustered) {
    const int words = static_cast<int>(cdg_moe_route_workspace_bytes(g->E) / 4);
    const int rc = launch(route_clear_kernel, dim3((words + 255) / 256), 256, 0, st, static_cast<uint32_t*>(workspace), words);
    if (rc != CDG_OK) return rc;
  }
  if (g->dtype == CDG_DTYPE_BF16) return dispatch_route<__nv_bfloat16>(a, st);
  if (g->dtype == CDG_DTYPE_F16) return dispatch_route<__half>(a, st);
  return dispatch_route<float>(a, st);
}

int cdg_moe_route_backward(const cdg_route_backward_args* g, cdg_stream_t stream) {
  using namespace cdg;
  if (!g || g->T < 0 || g->E <= 0 || g->topk <= 0 || g->topk > g->E || !row_dtype(g->dtype))
    return CDG_ERR_INVALID_ARGUMENT;
  if (g->scoring != CDG_SCORE_SOFTMAX && g->scoring != CDG_SCORE_SIGMOID) return CDG_ERR_INVALID_ARGUMENT;
  if (g->E > kRouteMaxExperts || g->topk > kRouteMaxTopk || g->T > kRouteMaxTokens) return CDG_ERR_UNSUPPORTED;
  if (g->grad_loss && (!g->counts || !g->tokens)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->T == 0) return CDG_OK;
  if (!g->logits || !g->ids || !g->dlogits || (!g->grad_weights && !g->grad_loss)) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(element_size(g->dtype), {g->logits, g->dlogits}) ||
      !on_boundary(4, {g->ids, g->grad_weights, g->grad_loss, g->counts, g->tokens}))
    return CDG_ERR_ALIGNMENT;
  RouteBwd a{g->logits, g->stride, g->ids, g->grad_weights, g->grad_loss, g->counts, g->tokens, g->T,
             static_cast<int>(g->E), static_cast<int>(g->topk), g->scoring == CDG_SCORE_SIGMOID, g->renormalize != 0,
             g->scale, g->dlogits, g->d_stride};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (g->dtype == CDG_DTYPE_BF16) return dispatch_route_backward<__nv_bfloat16>(a, st);
  if (g->dtype == CDG_DTYPE_F16) return dispatch_route_backward<__half>(a, st);
  return dispatch_route_backward<float>(a, st);
}

}  // extern "C"
