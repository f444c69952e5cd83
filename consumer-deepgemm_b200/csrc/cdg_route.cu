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
//   renormalised: g_j <- (g_j - sum_i g_i c_i / C) / C with c the chosen scores, C their sum
//   softmax: dl_i = p_i (d_i - sum_j d_j p_j),  d = scatter(g) + a
//   sigmoid: dl_i = (scatter(g)_i + (a_i - sum_j a_j p_j) / S) s_i (1 - s_i),  S = sum s
//
// A warp takes a row, lane l the experts l, l + 32, ...; a row is read once and its next row's
// loads are in flight meanwhile.  Bound by instructions rather than memory: the choice.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>

#include "cdg_b200.h"
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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Fast exponential and division (errors of a few units in the last place): the gate's weights
// and gradients stay within 1e-6 of the exact ones.
__device__ __forceinline__ float exp_fast(float v) {
  // 2^(v log2 e), results below the normal range taken as 0 (__expf spends three instructions on them)
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float sigmoid_fast(float v) { return __fdividef(1.0f, 1.0f + exp_fast(-v)); }

// The k experts of the largest keys of a row, of equal keys the lowest first: lane j gets the j-th
// (x its key, y the expert), or y = -1 where no key that can be chosen is left.  key[i] is that of
// expert i * 32 + lane, mine the lane's largest.
//
// The k-th largest of the 32 lanes' maxima is a lower bound of the k-th largest key, and few keys
// reach it (with 256 experts and k = 8 about ten), so: the maxima are sorted across the lanes (a
// bitonic network) for the bound; the keys that reach it are listed, each with its expert; each lane
// takes one of the list and counts how many of the others go before it.  A list of more than 32, or
// a lane with more than four of them (many equal keys, or k near 32), is chosen from round by round,
// a warp-wide maximum each; at 32,768 x 256, k = 8 that alone took the kernel 43 us.
template <int N>
__device__ __forceinline__ int2 choose(uint32_t (&key)[N], uint32_t mine, int k, int lane, unsigned long long* list) {
  uint32_t top = mine;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2) {
      const uint32_t other = __shfl_xor_sync(kAll, top, j);
      top = ((lane & j) == 0) == ((lane & size) == 0) ? max(top, other) : min(top, other);  // falling order
    }
  }
  const uint32_t bound = max(__shfl_sync(kAll, top, k - 1), kFirstKey);
  int reach = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) reach += key[i] >= bound ? 1 : 0;
  const unsigned one = __ballot_sync(kAll, reach > 0), two = __ballot_sync(kAll, reach > 1),
                 three = __ballot_sync(kAll, reach > 2), four = __ballot_sync(kAll, reach > 3);
  const int count = __popc(one) + __popc(two) + __popc(three) + __popc(four);
  int2 got = make_int2(0, -1);
  if (count <= 32 && !__any_sync(kAll, reach > 4)) {
    if (reach > 0) {
      const unsigned below = (1u << lane) - 1u;
      int place = __popc(one & below) + __popc(two & below) + __popc(three & below) + __popc(four & below);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // key first, then the lower expert
        if (key[i] >= bound)
          list[place++] = (static_cast<unsigned long long>(key[i]) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i * 32 + lane));
      }
    }
    __syncwarp();
    const unsigned long long own = lane < count ? list[lane] : 0;
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) before += list[j] > own ? 1 : 0;
    __syncwarp();
    if (lane < count && before < k) list[before] = own;
    __syncwarp();
    if (lane < min(count, k)) {
      const unsigned long long v = list[lane];
      got = make_int2(static_cast<int>(v >> 32), static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(v)));
    }
    __syncwarp();
    return got;
  }
  for (int j = 0; j < k; ++j) {
    const uint32_t best = __reduce_max_sync(kAll, mine);
    if (best < kFirstKey) break;
    int e = 0x7fffffff;
    if (mine == best) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (key[i] == best) e = i * 32 + lane;
    }
    const int winner = static_cast<int>(__reduce_min_sync(kAll, static_cast<unsigned>(e)));
    if (e == winner) {
      mine = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i * 32 + lane == winner) key[i] = 0;
        mine = max(mine, key[i]);
      }
    }
    if (lane == j) got = make_int2(static_cast<int>(best), winner);
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
  int sigmoid, renormalize, balance;
  float scale;
  float* weights;
  int32_t *ids, *counts, *tokens;
  float* loss;
  // zeroed before the launch (several CTAs): sum of p per expert in units of 2^-40, rows per
  // expert, valid tokens, finished CTAs
  unsigned long long* psum;
  int32_t *acc_counts, *acc_tokens, *ticket;
};

// Sums of p leave a CTA as 64-bit integers in units of 2^-40, so that the order in which the
// CTAs add them does not change the result.  2^23 tokens fit.
constexpr float kFixed = 1099511627776.0f;
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

// N experts per lane.  Dynamic shared memory: E counts, then one row of E sums of p per warp.
template <typename T, int N, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) moe_route_kernel(const Route a) {
  extern __shared__ int32_t route_smem[];
  __shared__ double scratch[WARPS];
  __shared__ int32_t s_tokens, s_last;
  __shared__ unsigned long long s_list[WARPS][32];
  int32_t* s_counts = route_smem;
  float* s_psum = reinterpret_cast<float*>(route_smem + a.E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_counts[e] = 0;
  if (threadIdx.x == 0) s_tokens = 0;
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();

  const T* logits = static_cast<const T*>(a.logits);
  float psum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) psum[i] = 0.0f;
  int32_t tokens = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * WARPS;
  float next[N];
  const int left = a.E - lane;  // expert i * 32 + lane exists where i * 32 < left
  auto load_row = [&](int64_t row) {
    const T* at = logits + row * a.stride + lane;
    if (a.E == N * 32) {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = to_f(at[i * 32]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = i * 32 < left ? to_f(at[i * 32]) : -INFINITY;
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * WARPS + warp;
  if (row < a.T) load_row(row);
  for (; row < a.T; row += step) {
    uint32_t key[N];
    float v[N];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = clean_logit(next[i]);
      key[i] = order_key(v[i]);
      top = max(top, key[i]);
    }
    if (row + step < a.T) load_row(row + step);
    top = __reduce_max_sync(kAll, top);
    int32_t id = -1;
    float w = 0.0f;
    if (top >= kFirstKey && (!a.mask || a.mask[row])) {  // warp-uniform
      const float m = a.sigmoid ? 0.0f : key_value(top);
      float inv = 1.0f;   // 1 / sum of exponentials (softmax)
      float part = 0.0f;  // 1 / sum of scores
      if (a.balance || a.bias || !a.renormalize) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          v[i] = a.sigmoid ? sigmoid_fast(v[i]) : exp_fast(v[i] - m);
          total += v[i];
        }
        total = warp_sum(total);
        part = total > 0.0f ? __fdividef(1.0f, total) : 0.0f;
        if (!a.sigmoid) inv = part;
        if (a.bias) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (key[i] >= kFirstKey) key[i] = order_key(clean_logit(v[i] * inv + __ldg(a.bias + i * 32 + lane)));
        }
      }
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) mine = max(mine, key[i]);
      const bool valid = __any_sync(kAll, mine >= kFirstKey);  // a bias of -inf may have left nothing
      if (valid) {
        ++tokens;
        if (a.balance) {
#pragma unroll
          for (int i = 0; i < N; ++i) psum[i] = fmaf(v[i], part, psum[i]);
        }
        const int2 got = choose<N>(key, mine, a.k, lane, s_list[warp]);
        id = got.y;
        if (id >= 0) {
          // the key is that of the logit itself, unless a bias went into it
          const float l = a.bias ? clean_logit(to_f(logits[row * a.stride + id])) : key_value(got.x);
          w = a.sigmoid ? sigmoid_fast(l) : exp_fast(l - m) * inv;
          atomicAdd(&s_counts[id], 1);
        }
      }
      if (a.renormalize) {
        const float total = warp_sum(w);
        w = total > 0.0f ? __fdividef(w, total) : 0.0f;
      }
      w *= a.scale;
    }
    if (lane < a.k) {
      a.ids[row * a.k + lane] = id;
      a.weights[row * a.k + lane] = w;
    }
  }

  if (lane == 0 && tokens) atomicAdd(&s_tokens, tokens);
  if (a.balance) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < a.E) s_psum[warp * a.E + i * 32 + lane] = psum[i];
  }
  __syncthreads();
  if (gridDim.x == 1) {  // one CTA saw every row
    double sum = 0.0;
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      a.counts[e] = s_counts[e];
      if (a.balance) {
        double p = 0.0;
        for (int i = 0; i < WARPS; ++i) p += s_psum[i * a.E + e];
        sum += p * s_counts[e];
      }
    }
    const double n = s_tokens > 0 ? s_tokens : 1;
    if (a.balance) sum = cta_sum64<WARPS>(sum, scratch);
    if (threadIdx.x == 0) {
      *a.tokens = s_tokens;
      if (a.balance) *a.loss = static_cast<float>(sum * a.E / a.k / n / n);
    }
    return;
  }
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    if (s_counts[e]) atomicAdd(&a.acc_counts[e], s_counts[e]);
    if (a.balance) {
      float p = 0.0f;
      for (int i = 0; i < WARPS; ++i) p += s_psum[i * a.E + e];
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

// Dynamic shared memory: one row of E floats per warp, the scattered gradient of the chosen
// scores (zero between rows).
template <typename T, int N, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) moe_route_backward_kernel(const RouteBwd a) {
  extern __shared__ float s_grad[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* sg = s_grad + warp * a.E;
  for (int e = lane; e < a.E; e += 32) sg[e] = 0.0f;
  __syncwarp();
  grid_dependency_wait();
  grid_launch_dependents();
  float load[N];  // a_e of the lane's experts
#pragma unroll
  for (int i = 0; i < N; ++i) load[i] = 0.0f;
  if (a.gloss) {
    const float n = static_cast<float>(max(*a.tokens, 1));
    const float f = *a.gloss * (static_cast<float>(a.E) / static_cast<float>(a.k)) / n / n;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < a.E) load[i] = f * static_cast<float>(a.counts[i * 32 + lane]);
  }
  const T* logits = static_cast<const T*>(a.logits);
  const int64_t step = static_cast<int64_t>(gridDim.x) * WARPS;
  float next[N];
  int32_t next_id = -1;
  float next_g = 0.0f;
  const int left = a.E - lane;  // expert i * 32 + lane exists where i * 32 < left
  auto load_row = [&](int64_t row) {
    const T* at = logits + row * a.stride + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) next[i] = i * 32 < left ? to_f(at[i * 32]) : -INFINITY;
    if (lane < a.k) {
      next_id = __ldg(a.ids + row * a.k + lane);
      if (a.gw) next_g = __ldg(a.gw + row * a.k + lane);
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * WARPS + warp;
  if (row < a.T) load_row(row);
  for (; row < a.T; row += step) {
    float s[N];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = clean_logit(next[i]);
      m = fmaxf(m, s[i]);
    }
    const int32_t id = next_id >= 0 && next_id < a.E ? next_id : -1;
    float g = id >= 0 ? next_g * a.scale : 0.0f;
    if (row + step < a.T) load_row(row + step);
    T* out = static_cast<T*>(a.dlogits) + row * a.d_stride;
    if (!__any_sync(kAll, id >= 0)) {  // masked token: no gradient
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * 32 + lane < a.E) out[i * 32 + lane] = from_f<T>(0.0f);
      continue;
    }
    m = a.sigmoid ? 0.0f : key_value(__reduce_max_sync(kAll, order_key(m)));
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = a.sigmoid ? sigmoid_fast(s[i]) : exp_fast(s[i] - m);
      total += s[i];
    }
    total = warp_sum(total);
    const float inv = total > 0.0f ? __fdividef(1.0f, total) : 0.0f;
    if (!a.sigmoid) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] *= inv;  // the scores are the probabilities
    }
    if (a.gw) {
      if (a.renormalize) {
        float c = 0.0f;
        if (id >= 0) {
          const float l = clean_logit(to_f(logits[row * a.stride + id]));
          c = a.sigmoid ? sigmoid_fast(l) : exp_fast(l - m) * inv;
        }
        float chosen = warp_sum(c);
        chosen = chosen > 0.0f ? __fdividef(1.0f, chosen) : 1.0f;
        g = (g - warp_sum(g * c) * chosen) * chosen;
      }
      if (id >= 0) atomicAdd(&sg[id], g);
      __syncwarp();
    }
    float d[N];
    float dot = 0.0f;  // of what meets the probabilities: everything (softmax) or the loss alone
#pragma unroll
    for (int i = 0; i < N; ++i) {
      d[i] = a.gw && i * 32 < left ? sg[i * 32 + lane] : 0.0f;
      dot = fmaf(a.sigmoid ? load[i] : d[i] + load[i], s[i], dot);
    }
    dot = warp_sum(dot);
    if (a.gw) {
      __syncwarp();
      if (id >= 0) sg[id] = 0.0f;
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v;
      if (a.sigmoid)
        v = (d[i] + (load[i] - dot * inv) * inv) * s[i] * (1.0f - s[i]);
      else
        v = s[i] * (d[i] + load[i] - dot);
      if (i * 32 < left) out[i * 32 + lane] = from_f<T>(v);
    }
  }
}

constexpr int kRouteWarps = 8;
// Few tokens over few experts run in one CTA of 32 warps, which needs neither zeroed sums (a
// memset before the kernel) nor a last CTA.
constexpr int64_t kOneCtaTokens = 64;
constexpr int kOneCtaExperts = 256;
bool one_cta(int64_t T, int64_t E) { return T <= kOneCtaTokens && E <= kOneCtaExperts; }

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

template <typename T, int N>
int launch_route(const Route& a, cudaStream_t st) {
  if constexpr (N * 32 <= kOneCtaExperts) {
    if (one_cta(a.T, a.E)) {
      const size_t smem = a.E * 4 + (a.balance ? size_t(32) * a.E * 4 : 0);
      return launch(moe_route_kernel<T, N, 32>, dim3(1), 1024, smem, st, a);
    }
  }
  // the largest dynamic shared memory of this N, so that one look-up serves every call
  static std::atomic<int> known{0};
  const int per_sm = resident_ctas(moe_route_kernel<T, N, kRouteWarps>, kRouteWarps * 32,
                                   size_t(N) * 32 * 4 * (kRouteWarps + 1), &known);
  const int64_t ctas = (a.T + kRouteWarps - 1) / kRouteWarps;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ctas, int64_t(sm_count()) * per_sm));
  const size_t smem = a.E * 4 + (a.balance ? size_t(kRouteWarps) * a.E * 4 : 0);
  return launch(moe_route_kernel<T, N, kRouteWarps>, dim3(grid), kRouteWarps * 32, smem, st, a);
}

template <typename T, int N>
int launch_route_backward(const RouteBwd& a, cudaStream_t st) {
  static std::atomic<int> known{0};
  const int per_sm = resident_ctas(moe_route_backward_kernel<T, N, kRouteWarps>, kRouteWarps * 32,
                                   size_t(N) * 32 * 4 * kRouteWarps, &known);
  const int64_t ctas = (a.T + kRouteWarps - 1) / kRouteWarps;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ctas, int64_t(sm_count()) * per_sm));
  return launch(moe_route_backward_kernel<T, N, kRouteWarps>, dim3(grid), kRouteWarps * 32, size_t(kRouteWarps) * a.E * 4, st,
                a);
}

template <typename T>
int dispatch_route(const Route& a, cudaStream_t st) {
  const int n = (a.E + 31) / 32;
  if (n <= 1) return launch_route<T, 1>(a, st);
  if (n <= 2) return launch_route<T, 2>(a, st);
  if (n <= 4) return launch_route<T, 4>(a, st);
  if (n <= 8) return launch_route<T, 8>(a, st);
  if (n <= 16) return launch_route<T, 16>(a, st);
  return launch_route<T, 32>(a, st);
}

template <typename T>
int dispatch_route_backward(const RouteBwd& a, cudaStream_t st) {
  const int n = (a.E + 31) / 32;
  if (n <= 1) return launch_route_backward<T, 1>(a, st);
  if (n <= 2) return launch_route_backward<T, 2>(a, st);
  if (n <= 4) return launch_route_backward<T, 4>(a, st);
  if (n <= 8) return launch_route_backward<T, 8>(a, st);
  if (n <= 16) return launch_route_backward<T, 16>(a, st);
  return launch_route_backward<T, 32>(a, st);
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
  if (!one_cta(g->T, g->E) &&
      cudaMemsetAsync(workspace, 0, cdg_moe_route_workspace_bytes(g->E), st) != cudaSuccess)
    return CDG_ERR_CUDA;
  Route a{};
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
  RouteBwd a{g->logits, g->stride, g->ids, g->grad_weights, g->grad_loss, g->counts, g->tokens, g->T,
             static_cast<int>(g->E), static_cast<int>(g->topk), g->scoring == CDG_SCORE_SIGMOID, g->renormalize != 0,
             g->scale, g->dlogits, g->d_stride};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (g->dtype == CDG_DTYPE_BF16) return dispatch_route_backward<__nv_bfloat16>(a, st);
  if (g->dtype == CDG_DTYPE_F16) return dispatch_route_backward<__half>(a, st);
  return dispatch_route_backward<float>(a, st);
}

}  // extern "C"
