// Root-mean-square norm with the residual's addition, an e4m3 output with 1x128 scales, and
// its gradient.
//
//   h = x + r                      (32 bits; stored once in x's type)
//   s = 1 / sqrt(mean(h^2) + eps)
//   y = h * s * w                  (from the 32-bit h; stored once in x's type)
//   q, scale = 1x128 e4m3 quantisation of the 32-bit y (the recipes of cdg_quant_fp8_rows)
//
//   u = w * dy,  dx = dh + s * (u - h * s^2 * mean(u * h)),  dw[c] = sum_t dy[t, c] * h[t, c] * s[t]
//
// Both directions are bound by memory: the forward pass reads x and r once and writes h, y, q and
// the scales once, the backward pass reads dy, h and dh once and writes dx once.  A row stays in
// its CTA's registers between the sum of squares and the stores.  One B200: 32,768 x 4096 BF16 with
// residual and codes 194 us (6.2 TB/s; a plain copy 6.5), 8 x 4096 2.3 us; backward of 16,384 x 4096
// with dh 94 us (5.7 TB/s) with the sums of dw.  Rows off 16-byte boundaries move by single elements: 6007 x
// 2503 BF16 with residual and codes 44 us (3.1 TB/s), backward 55 us (2.2 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "cdg_b200.h"
#include "cdg_rows.cuh"

namespace cdg {
namespace {

// The norm's weights: of the rows' type or FP32.
template <typename T, bool WIDE>
__device__ __forceinline__ void load_weight8(const void* w, bool w_f32, int64_t chunk, int lane, int64_t H,
                                             float (&v)[8]) {
  if (w_f32) {
    unpack8<float>(load8<float, WIDE>(static_cast<const float*>(w), chunk, lane, H), v);
  } else {
    unpack8<T>(load8<T, WIDE>(static_cast<const T*>(w), chunk, lane, H), v);
  }
}

// Sum over the CTA's warps of one value per thread (every thread gets it).  `slot` holds one
// value per warp; one barrier, so a caller that comes again alternates between two slots.
__device__ __forceinline__ float cta_sum(float v, float* slot, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  float t = lane < warps ? slot[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// Scale and factor of a 128-column block with the largest magnitude `amax`.
// The scale is that of cdg_quant_fp8_rows bit for bit, and a code is e4m3 of y times the factor.
// Both are correctly rounded quotients: the FP32 recipe's code can differ from e4m3(y / amax * 448) only
// where a rounding point of e4m3 lies within 4 * 2^-24 of the value.  A NaN among the values does not
// reach the scale (fmaxf passes over it); its own code is NaN.  With the FP32 recipe even lanes divide
// for the scale, which is theirs alone, and odd ones for the factor: calls of 32,768 x 4096 BF16 take
// 1.3% longer than with approximate divisions, 2.0% with two divisions a lane.
__device__ __forceinline__ float block_scale(float amax, int pow2, int lane, float& factor) {
  amax = fmaxf(amax, 1e-12f);
  if (pow2) {
    uint32_t b = __float_as_uint(amax / 448.0f);
    if (b & 0x007FFFFFu) b = (b & 0xFF800000u) + 0x00800000u;
    factor = 1.0f / __uint_as_float(b);
    return __uint_as_float(b);
  }
  const bool odd = lane & 1;
  const float quotient = (odd ? 448.0f : amax) / (odd ? amax : 448.0f);
  factor = __shfl_sync(0xffffffffu, quotient, lane | 1);
  return quotient;
}

struct NormFwd {
  const void *x, *r, *w;
  void *h, *y;
  uint8_t* q;
  float* s;
  int64_t x_stride, r_stride, h_stride, y_stride, q_stride, s_stride_m, s_stride_k;
  int64_t T, H;
  float eps, inv_h;
  int w_f32, pow2;
};

// Quantise one chunk of y and store codes and scales.
template <bool WIDE>
__device__ __forceinline__ void quant_chunk(const NormFwd& a, int64_t row, int64_t chunk, int lane,
                                            const float (&y)[8]) {
  uint8_t* q = a.q + row * a.q_stride;
  float* s = a.s + row * a.s_stride_m;
  const int64_t kb = chunk * 2;
  if constexpr (WIDE) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(y[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float f;
    const float scale = block_scale(m, a.pow2, lane, f);
    const int64_t c = column<true>(chunk, lane, 0);
    if (c >= a.H) return;
    uint32_t p[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * k] * f, y[4 * k + 1] * f), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi =
          __nv_cvt_float2_to_fp8x2(make_float2(y[4 * k + 2] * f, y[4 * k + 3] * f), __NV_SATFINITE, __NV_E4M3);
      p[k] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(q + c) = make_uint2(p[0], p[1]);
    if ((lane & 15) == 0) s[(kb + (lane >> 4)) * a.s_stride_k] = scale;
  } else {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(y[4 * b + j]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float f;
      const float scale = block_scale(m, a.pow2, lane, f);
      uint8_t* to = q + column<false>(chunk, lane, 4 * b);
      const bool full = (kb + b + 1) * 128 <= a.H;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const uint32_t two =
            __nv_cvt_float2_to_fp8x2(make_float2(y[4 * b + j] * f, y[4 * b + j + 1] * f), __NV_SATFINITE, __NV_E4M3);
        if (full || column<false>(chunk, lane, 4 * b + j) < a.H) to[j * 32] = static_cast<uint8_t>(two);
        if (full || column<false>(chunk, lane, 4 * b + j + 1) < a.H) to[(j + 1) * 32] = static_cast<uint8_t>(two >> 8);
      }
      if (lane == 0 && (kb + b) * 128 < a.H) s[(kb + b) * a.s_stride_k] = scale;
    }
  }
}

// One row per CTA (one per warp where a warp holds a whole row: warps_per_row == 1); warp w of a
// row's warps takes chunks w, w + warps, ... and keeps its ITER chunks of h in registers.
template <typename T, bool WIDE, int ITER, int THREADS>
__global__ void __launch_bounds__(THREADS) add_rms_norm_kernel(const NormFwd a, int warps_per_row) {
  __shared__ float slot[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t row = blockIdx.x;
  int w = warp;
  if (warps_per_row == 1) {
    row = row * (blockDim.x >> 5) + warp;
    w = 0;
    if (row >= a.T) return;  // no barrier follows where a warp holds the row
  }
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  Raw<T> rx[ITER], rr[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) rx[i] = load8<T, WIDE>(x, i * warps_per_row + w, lane, a.H);
  if (a.r) {
    const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
#pragma unroll
    for (int i = 0; i < ITER; ++i) rr[i] = load8<T, WIDE>(r, i * warps_per_row + w, lane, a.H);
  }
  float h[ITER][8];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    unpack8<T>(rx[i], h[i]);
    if (a.r) {
      float b[8];
      unpack8<T>(rr[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += b[j];
    }
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) part = fmaf(h[i][j], h[i][j], part);
    sum += part;
  }
  if (a.h) {
#pragma unroll
    for (int i = 0; i < ITER; ++i)
      store8<T, WIDE>(static_cast<T*>(a.h) + row * a.h_stride, i * warps_per_row + w, lane, a.H, h[i]);
  }
  sum = cta_sum(sum, slot, warps_per_row);
  const float rstd = rsqrtf(fmaf(sum, a.inv_h, a.eps));
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int64_t chunk = i * warps_per_row + w;
    if (chunk * 256 >= a.H) break;  // warp-uniform
    float wv[8];
    load_weight8<T, WIDE>(a.w, a.w_f32, chunk, lane, a.H, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) wv[j] *= h[i][j] * rstd;
    if (a.y) store8<T, WIDE>(static_cast<T*>(a.y) + row * a.y_stride, chunk, lane, a.H, wv);
    if (a.q) quant_chunk<WIDE>(a, row, chunk, lane, wv);
  }
}

constexpr int kRingMax = 8;  // rows in flight per CTA of the ring kernel

struct NormBwd {
  const void *dy, *h, *w, *dh;
  void* dx;
  float* partial;  // [gridDim.x][H]: each CTA's sum over its rows of dy * h * s
  int64_t dy_stride, h_stride, dh_stride, dx_stride;
  int64_t T, H;
  float eps;
  int w_f32;
};

// CTA b takes rows b, b + grid, ...; warp w of it takes chunks w, w + warps, ... of every row and
// sums their weight gradients in registers.  The next row's loads are issued before this row's
// barrier, so that they cross it.  Both sums over the row (h^2 and u * h) share one barrier.
template <typename T, bool WIDE, int ITER, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_backward_kernel(const NormBwd a) {
  __shared__ float2 slot[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const T* dy = static_cast<const T*>(a.dy);
  const T* h = static_cast<const T*>(a.h);
  const T* dh = static_cast<const T*>(a.dh);
  float acc[ITER][8] = {};
  Raw<T> rdy[ITER], rh[ITER], rdh[ITER];
  auto load_row = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int64_t chunk = i * warps + warp;
      rh[i] = load8<T, WIDE>(h + row * a.h_stride, chunk, lane, a.H);
      rdy[i] = load8<T, WIDE>(dy + row * a.dy_stride, chunk, lane, a.H);
      if (dh) rdh[i] = load8<T, WIDE>(dh + row * a.dh_stride, chunk, lane, a.H);
    }
  };
  int64_t row = blockIdx.x;
  if (row < a.T) load_row(row);
  for (int turn = 0; row < a.T; row += gridDim.x, turn ^= 1) {
    Raw<T> cdy[ITER], ch[ITER], cdh[ITER];
    float sq = 0.0f, uh = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      cdy[i] = rdy[i]; ch[i] = rh[i]; cdh[i] = rdh[i];
    }
    if (row + gridDim.x < a.T) load_row(row + gridDim.x);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      float hv[8], g[8], wv[8];
      unpack8<T>(ch[i], hv);
      unpack8<T>(cdy[i], g);
      load_weight8<T, WIDE>(a.w, a.w_f32, i * warps + warp, lane, a.H, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq = fmaf(hv[j], hv[j], sq);
        uh = fmaf(g[j] * wv[j], hv[j], uh);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
      uh += __shfl_xor_sync(0xffffffffu, uh, o);
    }
    if (lane == 0) slot[turn][warp] = make_float2(sq, uh);
    __syncthreads();
    const float2 t = lane < warps ? slot[turn][lane] : make_float2(0.0f, 0.0f);
    sq = t.x;
    uh = t.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
      uh += __shfl_xor_sync(0xffffffffu, uh, o);
    }
    const float inv = 1.0f / static_cast<float>(a.H);
    const float rstd = rsqrtf(fmaf(sq, inv, a.eps));
    const float k = uh * inv * rstd * rstd;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int64_t chunk = i * warps + warp;
      float hv[8], g[8], wv[8];
      unpack8<T>(ch[i], hv);
      unpack8<T>(cdy[i], g);
      load_weight8<T, WIDE>(a.w, a.w_f32, chunk, lane, a.H, wv);
      float out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = fmaf(g[j], hv[j] * rstd, acc[i][j]);
        out[j] = rstd * fmaf(-hv[j], k, g[j] * wv[j]);
      }
      if (dh) {
        float d[8];
        unpack8<T>(cdh[i], d);
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] += d[j];
      }
      store8<T, WIDE>(static_cast<T*>(a.dx) + row * a.dx_stride, chunk, lane, a.H, out);
    }
  }
  float* partial = a.partial + static_cast<int64_t>(blockIdx.x) * a.H;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = column<WIDE>(i * warps + warp, lane, j);
      if (c < a.H) partial[c] = acc[i][j];
    }
  }
}

// The same with the rows brought into shared memory by bulk copies, for rows on 16-byte boundaries
// of up to 8192 columns: warp w holds chunks w and w + warps of every row of its CTA, and a ring of
// `slots` rows (h, dy and dh side by side) keeps the loads of the next rows in flight whatever the
// registers hold.  At 16,384 x 4096 BF16 with dh (537 MB) it takes 93 us, 5.8 TB/s; with one chunk a
// warp, twice the warps at each row's barrier, 110 us; the register form at its best shape 137 us.
template <typename T>
__global__ void __launch_bounds__(512) rms_norm_backward_ring_kernel(const NormBwd a, const int slots) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float2 slot_sum[2][32];
  __shared__ __align__(8) uint64_t full[kRingMax];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const uint32_t row_bytes = static_cast<uint32_t>(a.H * sizeof(T));
  const int arrays = a.dh ? 3 : 2;
  const T* h = static_cast<const T*>(a.h);
  const T* dy = static_cast<const T*>(a.dy);
  const T* dh = static_cast<const T*>(a.dh);
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i) mbar_init(&full[i], 1);
    fence_mbarrier_init();
  }
  __syncthreads();
  auto load_row = [&](int64_t row, int s) {  // by thread 0
    uint8_t* at = ring + static_cast<size_t>(s) * arrays * row_bytes;
    mbar_arrive_expect_tx(&full[s], arrays * row_bytes);
    bulk_load(at, h + row * a.h_stride, row_bytes, &full[s]);
    bulk_load(at + row_bytes, dy + row * a.dy_stride, row_bytes, &full[s]);
    if (dh) bulk_load(at + 2 * row_bytes, dh + row * a.dh_stride, row_bytes, &full[s]);
  };
  const int64_t step = gridDim.x;
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i)
      if (blockIdx.x + i * step < a.T) load_row(blockIdx.x + i * step, i);
  }
  constexpr int V = 2;  // chunks of a warp
  float w[V][8], acc[V][8] = {};
#pragma unroll
  for (int u = 0; u < V; ++u) load_weight8<T, true>(a.w, a.w_f32, u * warps + warp, lane, a.H, w[u]);
  const float inv = 1.0f / static_cast<float>(a.H);
  int s = 0, turn = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t row = blockIdx.x; row < a.T; row += step, turn ^= 1) {
    ok = mbar_wait_cta(&full[s], phase, nullptr, wait_code(1, 1, s, phase, static_cast<int>(row)));
    const uint8_t* at = ring + static_cast<size_t>(s) * arrays * row_bytes;
    float hv[V][8] = {}, g[V][8] = {}, d[V][8] = {};
    float sq = 0.0f, uh = 0.0f;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int64_t c = column<true>(u * warps + warp, lane, 0);
      if (c < a.H) {
        const uint8_t* p = at + c * sizeof(T);
        unpack8<T>(*reinterpret_cast<const Raw<T>*>(p), hv[u]);
        unpack8<T>(*reinterpret_cast<const Raw<T>*>(p + row_bytes), g[u]);
        if (dh) unpack8<T>(*reinterpret_cast<const Raw<T>*>(p + 2 * row_bytes), d[u]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq = fmaf(hv[u][j], hv[u][j], sq);
        uh = fmaf(g[u][j] * w[u][j], hv[u][j], uh);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
      uh += __shfl_xor_sync(0xffffffffu, uh, o);
    }
    if (lane == 0) slot_sum[turn][warp] = make_float2(sq, uh);
    // also: every thread has taken its columns out of the slot; a wait that gave up ends the CTA
    if (__syncthreads_or(!ok)) {
      // copies issued before it still land: give them time before exit
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) __nanosleep(20000);
      return;
    }
    if (threadIdx.x == 0 && row + slots * step < a.T) load_row(row + slots * step, s);
    const float2 t = lane < warps ? slot_sum[turn][lane] : make_float2(0.0f, 0.0f);
    sq = t.x;
    uh = t.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
      uh += __shfl_xor_sync(0xffffffffu, uh, o);
    }
    const float rstd = rsqrtf(fmaf(sq, inv, a.eps));
    const float k = uh * inv * rstd * rstd;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      float out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[u][j] = fmaf(g[u][j], hv[u][j] * rstd, acc[u][j]);
        out[j] = fmaf(rstd, fmaf(-hv[u][j], k, g[u][j] * w[u][j]), d[u][j]);
      }
      store8<T, true>(static_cast<T*>(a.dx) + row * a.dx_stride, u * warps + warp, lane, a.H, out);
    }
    if (++s == slots) { s = 0; phase ^= 1; }
  }
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int64_t c = column<true>(u * warps + warp, lane, 0);
    if (c < a.H) {
      float4* partial = reinterpret_cast<float4*>(a.partial + static_cast<int64_t>(blockIdx.x) * a.H + c);
      partial[0] = make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
      partial[1] = make_float4(acc[u][4], acc[u][5], acc[u][6], acc[u][7]);
    }
  }
}

}  // namespace

// Row widths up to this one fit the registers of one CTA (32 warps of four 256-column chunks).
constexpr int64_t kNormMaxH = 32768;

namespace {

template <typename T, bool WIDE>
int launch_norm(const NormFwd& a, cudaStream_t st) {
  const int chunks = static_cast<int>((a.H + 255) / 256);
  // Few rows are spread over as many warps as they have chunks (latency).  Otherwise a warp holds
  // two chunks: 32,768 x 4096 BF16 with residual and codes takes 192 us so; in one comparison, single
  // launches, 203 us, 259 us with one (more warps wait at each row's barrier) and 236 us with four (100
  // registers a thread leave too few warps to cover the loads); 65,536 x 1024 96 us, 118 us and 119 us.  Only rows of more
  // than 16,384 columns need four, with some spilling.
  const int iter = chunks <= 32 && a.T <= 2 * sm_count() ? 1 : chunks > 64 ? 4 : chunks >= 2 ? 2 : 1;
  const int warps = (chunks + iter - 1) / iter;
  const int rows = warps == 1 ? 4 : 1;  // rows per CTA
  const unsigned grid = static_cast<unsigned>((a.T + rows - 1) / rows);
  auto kernel = iter == 1   ? add_rms_norm_kernel<T, WIDE, 1, 1024>
                : iter == 2 ? add_rms_norm_kernel<T, WIDE, 2, 1024>
                            : add_rms_norm_kernel<T, WIDE, 4, 1024>;
  return launch(kernel, dim3(grid), warps * rows * 32, 0, st, a, warps);
}

// CTAs of the backward kernels: every SM filled, each CTA taking several rows where there are
// that many, because each writes one row of partial weight gradients.
struct BwdShape {
  int warps, grid;
};

constexpr int64_t kRingMaxH = 8192;  // 16 warps of two chunks

// Two chunks a warp and sixteen warps an SM (16,384 x 4096 BF16: 93 us; eight warps leave the loads
// waiting, 128 us, 24 and more gain nothing, 96 to 122 us), but for 16-bit rows on odd boundaries, whose
// loads of single elements want warps rather than registers: one chunk and 32 (6007 x 2503: 53 us
// against 75).  Rows of more than 8192 columns take four chunks a warp and spill most of them (1 to 2.4 KB
// a thread): 8192 x 9216 BF16 1.97 ms, 0.3 TB/s.  From nine warps on, 4097 to 7680 columns, an SM holds
// one CTA: 8192 x 4352 73 us (3.9 TB/s), 16,384 x 5120 144 us (4.7 TB/s).
BwdShape backward_shape(int64_t T, int64_t H, bool single) {
  const int chunks = static_cast<int>((H + 255) / 256);
  BwdShape s;
  s.warps = H > kRingMaxH ? (chunks + 3) / 4 : single ? chunks : (chunks + 1) / 2;
  const int per_sm = std::max(1, std::min(16, (single ? 32 : 16) / s.warps));
  s.grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(T, int64_t(sm_count()) * per_sm)));
  return s;
}

template <typename T>
int launch_norm_backward(const NormBwd& a, const BwdShape& s, bool wide, cudaStream_t st) {
  if (wide && a.H <= kRingMaxH) {
    const int64_t row = a.H * static_cast<int64_t>(sizeof(T)) * (a.dh ? 3 : 2);
    const int per_sm = std::max(1, std::min(16, 16 / s.warps));
    const int slots = static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(kRingMax, 200 * 1024 / per_sm / row)));
    static std::once_flag flags[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CDG_ERR_CUDA;
    std::call_once(flags[dev], [] {
      (void)cudaFuncSetAttribute(rms_norm_backward_ring_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 200 * 1024);
    });
    return launch(rms_norm_backward_ring_kernel<T>, dim3(s.grid), s.warps * 32, slots * row, st, a, slots);
  }
  auto kernel = wide ? rms_norm_backward_kernel<T, true, 4, 1024> : rms_norm_backward_kernel<T, false, 4, 1024>;
  if (a.H <= kRingMaxH) {
    if constexpr (sizeof(T) == 2)
      kernel = rms_norm_backward_kernel<T, false, 1, 1024>;
    else
      kernel = rms_norm_backward_kernel<T, false, 2, 512>;
  }
  return launch(kernel, dim3(s.grid), s.warps * 32, 0, st, a);
}

}  // namespace

// This unit's record of waits that gave up (cdg_device_status reads it with the others').
int norm_sticky_status(int clear, int32_t* out) { return read_sticky(g_sticky_status, clear, out); }

}  // namespace cdg

extern "C" {

int cdg_add_rms_norm(const cdg_norm_args* g, cdg_stream_t stream) {
  using namespace cdg;
  if (!g || g->T < 0 || g->H <= 0 || !row_dtype(g->dtype)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->w_dtype != g->dtype && g->w_dtype != CDG_DTYPE_F32) return CDG_ERR_INVALID_ARGUMENT;
  if (g->scale_fmt != CDG_SCALE_FP32 && g->scale_fmt != CDG_SCALE_POW2) return CDG_ERR_INVALID_ARGUMENT;
  if (!(g->eps >= 0.0f)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->H > kNormMaxH || g->T >= int64_t(1) << 31) return CDG_ERR_UNSUPPORTED;
  if (g->T == 0) return CDG_OK;
  if (!g->x || !g->w || (g->q && !g->s) || (!g->y && !g->q && !g->h)) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(element_size(g->dtype), {g->x, g->r, g->h, g->y}) || !on_boundary(element_size(g->w_dtype), {g->w}) ||
      !on_boundary(4, {g->s}))
    return CDG_ERR_ALIGNMENT;
  NormFwd a{g->x, g->r, g->w, g->h, g->y, g->q, g->s, g->x_stride, g->r_stride, g->h_stride, g->y_stride, g->q_stride,
            g->s_stride_m, g->s_stride_k, g->T, g->H, g->eps, 1.0f / static_cast<float>(g->H), g->w_dtype == CDG_DTYPE_F32, g->scale_fmt};
  const int64_t e = element_size(g->dtype);
  const bool wide = g->H % 8 == 0 && wide_rows(a.x, a.x_stride, e) && wide_rows(a.r, a.r_stride, e) &&
                    wide_rows(a.h, a.h_stride, e) && wide_rows(a.y, a.y_stride, e) && wide_rows(a.w, 0, e) &&
                    (!a.q || (reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.q_stride % 8 == 0));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (g->dtype == CDG_DTYPE_BF16)
    return wide ? launch_norm<__nv_bfloat16, true>(a, st) : launch_norm<__nv_bfloat16, false>(a, st);
  if (g->dtype == CDG_DTYPE_F16) return wide ? launch_norm<__half, true>(a, st) : launch_norm<__half, false>(a, st);
  return wide ? launch_norm<float, true>(a, st) : launch_norm<float, false>(a, st);
}

size_t cdg_rms_norm_backward_workspace_bytes(int64_t T, int64_t H) {
  if (T < 0 || H <= 0 || H > cdg::kNormMaxH) return 0;
  // whichever form the rows' type and boundaries select
  return static_cast<size_t>(std::max(cdg::backward_shape(T, H, false).grid, cdg::backward_shape(T, H, true).grid)) * H *
         sizeof(float);
}

int cdg_rms_norm_backward(const cdg_norm_backward_args* g, void* workspace, size_t workspace_bytes,
                          cdg_stream_t stream) {
  using namespace cdg;
  if (!g || g->T < 0 || g->H <= 0 || !row_dtype(g->dtype)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->w_dtype != g->dtype && g->w_dtype != CDG_DTYPE_F32) return CDG_ERR_INVALID_ARGUMENT;
  if (!(g->eps >= 0.0f) || !g->w || !g->dw) return CDG_ERR_INVALID_ARGUMENT;
  if (g->H > kNormMaxH || g->T >= int64_t(1) << 31) return CDG_ERR_UNSUPPORTED;
  if (g->T > 0 && (!g->dy || !g->h || !g->dx)) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(element_size(g->dtype), {g->dy, g->h, g->dh, g->dx}) ||
      !on_boundary(element_size(g->w_dtype), {g->w, g->dw}))
    return CDG_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < cdg_rms_norm_backward_workspace_bytes(g->T, g->H)) return CDG_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return CDG_ERR_ALIGNMENT;  // sums leave four at a time
  NormBwd a{g->dy, g->h, g->w, g->dh, g->dx, static_cast<float*>(workspace), g->dy_stride, g->h_stride, g->dh_stride,
            g->dx_stride, g->T, g->H, g->eps, g->w_dtype == CDG_DTYPE_F32};
  const int64_t e = element_size(g->dtype);
  const bool wide = g->H % 8 == 0 && wide_rows(a.dy, a.dy_stride, e) && wide_rows(a.h, a.h_stride, e) &&
                    wide_rows(a.dh, a.dh_stride, e) && wide_rows(a.dx, a.dx_stride, e) && wide_rows(a.w, 0, e);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const BwdShape s = backward_shape(g->T, g->H, !wide && e == 2);
  int rc;
  if (g->dtype == CDG_DTYPE_BF16)
    rc = launch_norm_backward<__nv_bfloat16>(a, s, wide, st);
  else if (g->dtype == CDG_DTYPE_F16)
    rc = launch_norm_backward<__half>(a, s, wide, st);
  else
    rc = launch_norm_backward<float>(a, s, wide, st);
  if (rc != CDG_OK) return rc;
  const unsigned grid = static_cast<unsigned>((g->H + 31) / 32);
  if (g->w_dtype == CDG_DTYPE_BF16)
    return launch(column_sum_kernel<__nv_bfloat16>, dim3(grid), 1024, 0, st, a.partial, s.grid, g->H, static_cast<__nv_bfloat16*>(g->dw));
  if (g->w_dtype == CDG_DTYPE_F16)
    return launch(column_sum_kernel<__half>, dim3(grid), 1024, 0, st, a.partial, s.grid, g->H, static_cast<__half*>(g->dw));
  return launch(column_sum_kernel<float>, dim3(grid), 1024, 0, st, a.partial, s.grid, g->H, static_cast<float*>(g->dw));
}

}  // extern "C"
