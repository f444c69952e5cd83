// Dense product on the tensor cores with a fused epilogue: D = epilogue(A . B^T), A [M, K] and
// B [N, K] BF16 or FP16, FP32 accumulation.
//
//   z = sum_k A[m, k] B[n, k] + bias[n];   y = act(z) + residual[m, n]
//
// Each operand lies in memory either K-major (rows of K) or MN-major (K rows of M or N), so that
// one kernel serves x . W^T, dz . W and dz^T . x.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "cdg_ptx.cuh"
#include "cdg_rows.cuh"

namespace cdg {
namespace {

// ---------------------------------------------------------------- instructions
// D[tmem] (+)= A[smem] . B[smem], 16-bit operands, by the lane elect.sync picks of a whole warp.
__device__ __forceinline__ void tc_mma_f16_warp(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tc_commit_warp(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar))
      : "memory");
}

// Operand tiles of one K step (64 columns of K) in shared memory, 128-byte swizzle:
//   K-major:  [rows][64 k], 8-row groups 1024 bytes apart;
//   MN-major: chunks of 64 rows, each [64 k][64 rows] (8192 bytes); the 8-k groups of a chunk
//             are 1024 bytes apart, the chunks 8192.
// One MMA takes 16 of K: 32 bytes further on in the swizzled rows, or two 8-k groups.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn_major) {
  uint64_t d = smem_desc_sw128(addr);
  if (mn_major) d |= static_cast<uint64_t>((8192u >> 4) & 0x3FFFu) << 16;  // leading byte offset: chunk to chunk
  return d;
}

__device__ __forceinline__ uint32_t operand_k_step(bool mn_major) { return mn_major ? 2048u >> 4 : 32u >> 4; }

// Instruction descriptor of tcgen05.mma kind::f16 with FP32 accumulation.
__host__ __device__ __forceinline__ uint32_t idesc_f16(bool bf16, bool a_mn, bool b_mn, uint32_t m, uint32_t n) {
  uint32_t d = 1u << 4;  // D is FP32
  d |= (bf16 ? 1u : 0u) << 7;
  d |= (bf16 ? 1u : 0u) << 10;
  d |= (a_mn ? 1u : 0u) << 15;
  d |= (b_mn ? 1u : 0u) << 16;
  d |= ((n >> 3) & 0x3Fu) << 17;
  d |= ((m >> 4) & 0x1Fu) << 24;
  return d;
}

// ---------------------------------------------------------------- epilogue arithmetic
// Activations in FP32, with the fast exponential: exp(x) is within 2 + 1.173 |x| units in the last place and
// x is rounded a few times, so an activation's relative error is below 2^-19 + 2^-21 |x|, x the exponent
// that it takes (z, z^2 / 2 or u2 below): less than a 16-bit result's rounding.
__device__ __forceinline__ float fast_sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// Phi(-|z|), the normal distribution's tail, as exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.306 |z|).  The factor
// Phi(-a) exp(a^2 / 2) is smooth and falls as 1 / a, which t P(t) follows: P, of degree 7, has the least
// largest relative error on 0 <= a <= 14.5 (least squares with Lawson's weights), 1.1e-7 with these FP32
// coefficients; beyond, the exponential is 0.  The tail itself, not 1 + erf, so that nothing cancels: far
// below zero z Phi(z) is as exact, relative to itself, as the exponential.
__device__ __forceinline__ float normal_tail(float z) {
  const float a = fabsf(z);
  const float t = __fdividef(1.0f, fmaf(0.306f, a, 1.0f));
  float p = fmaf(t, 0.0365378037f, -0.150699764f);
  p = fmaf(t, p, 0.179384798f);
  p = fmaf(t, p, -0.0330358259f);
  p = fmaf(t, p, 0.118629217f);
  p = fmaf(t, p, 0.10436748f);
  p = fmaf(t, p, 0.122772254f);
  p = fmaf(t, p, 0.122044094f);
  return t * p * __expf(-0.5f * a * a);
}

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case CDG_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
    case CDG_ACT_SILU: return __fdividef(z, 1.0f + __expf(-z));
    case CDG_ACT_GELU: {
      const float tail = normal_tail(z);
      return z * (z < 0.0f ? tail : 1.0f - tail);
    }
    case CDG_ACT_GELU_TANH: {
      // 0.5 (1 + tanh u) = sigmoid(2u), u = sqrt(2 / pi) (z + 0.044715 z^3)
      const float u2 = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      return __fdividef(z, 1.0f + __expf(-u2));
    }
    default: return z;
  }
}

// d act(z) / dz
__device__ __forceinline__ float activate_slope(float z, int act) {
  switch (act) {
    case CDG_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case CDG_ACT_SILU: {
      const float s = fast_sigmoid(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case CDG_ACT_GELU: {
      const float tail = normal_tail(z);
      return (z < 0.0f ? tail : 1.0f - tail) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    }
    case CDG_ACT_GELU_TANH: {
      // with s = sigmoid(2u): z s' + s, s' = s (1 - s) d(2u)/dz
      const float s = fast_sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));
      // z^2 kept finite: far from zero s (1 - s) is 0, and so is the term
      return s + z * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * fminf(z * z, 1e30f));
    }
    default: return 1.0f;
  }
}

// The activation of C values, with one test for all of them.
template <int C>
__device__ __forceinline__ void activate_all(float (&v)[C], int act) {
  switch (act) {
    case CDG_ACT_RELU:
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = activate(v[j], CDG_ACT_RELU);
      break;
    case CDG_ACT_SILU:
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = activate(v[j], CDG_ACT_SILU);
      break;
    case CDG_ACT_GELU:
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = activate(v[j], CDG_ACT_GELU);
      break;
    case CDG_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = activate(v[j], CDG_ACT_GELU_TANH);
      break;
    default: break;
  }
}

struct Epilogue {
  const void* bias;
  const void* residual;
  void* y;
  void* z;  // the value before the activation, in the operands' type; NULL = not stored
  int64_t residual_stride, y_stride, z_stride;
  int bias_f32, residual_f32, act;
  int wide;       // y, z and residual rows on 16-byte boundaries
  int wide_bias;  // bias of the operands' type, on a 16-byte boundary
  int staged;     // pair kernel: y and residual through shared memory, by TMA (1) or by the warps (2)
};

// An element of a bias or of a residual, by the read-only path: loads of several elements may then
// be in flight across the stores between them.
template <typename T>
__device__ __forceinline__ float load_any(const void* p, int64_t i, int f32) {
  if (f32) return __ldg(static_cast<const float*>(p) + i);
  const unsigned short raw = __ldg(static_cast<const unsigned short*>(p) + i);
  return to_f(*reinterpret_cast<const T*>(&raw));
}

// Adds the residual to eight consecutive columns [n, n + 8) of row m, clipped at N, and stores them.
template <typename T, typename O>
__device__ __forceinline__ void add_residual_and_store8(const Epilogue& e, int64_t m, int64_t n, int64_t N,
                                                        float (&v)[8]) {
  const bool full = e.wide && n + 8 <= N;
  if (e.residual) {
    if (full && !e.residual_f32) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(e.residual) + m * e.residual_stride + n));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2(w[j], T());
        v[2 * j] += f.x;
        v[2 * j + 1] += f.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < N) v[j] += load_any<T>(e.residual, m * e.residual_stride + n + j, e.residual_f32);
    }
  }
  O* y = static_cast<O*>(e.y) + m * e.y_stride + n;
  if (full) {
    if constexpr (sizeof(O) == 4) {
      reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(y) = make_uint4(pack2(v[0], v[1], O()), pack2(v[2], v[3], O()),
                                                pack2(v[4], v[5], O()), pack2(v[6], v[7], O()));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n + j < N) y[j] = from_f<O>(v[j]);
  }
}

// The whole epilogue of eight consecutive columns [n, n + 8) of row m, clipped at N; `bias` holds
// theirs, or zeros.
template <typename T, typename O>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t m, int64_t n, int64_t N, const float (&bias)[8],
                                        float (&v)[8]) {
  const bool full = e.wide && n + 8 <= N;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += bias[j];
  if (e.z) {
    T* z = static_cast<T*>(e.z) + m * e.z_stride + n;
    if (full) {
      *reinterpret_cast<uint4*>(z) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()),
                                                pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < N) z[j] = from_f<T>(v[j]);
    }
  }
  activate_all<8>(v, e.act);
  add_residual_and_store8<T, O>(e, m, n, N, v);
}

// v[j] += bias[n + j] (the same for every lane).
template <typename T, int CH>
__device__ __forceinline__ void add_bias(const Epilogue& e, int64_t n, int64_t N, float (&v)[CH]) {
  if (e.bias) {
    if (e.wide_bias && n + CH <= N) {
#pragma unroll
      for (int g = 0; g < CH / 8; ++g) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(e.bias) + n) + g);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2(w[j], T());
          v[g * 8 + 2 * j] += f.x;
          v[g * 8 + 2 * j + 1] += f.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j)
        if (n + j < N) v[j] += load_any<T>(e.bias, n + j, e.bias_f32);
    }
  }
}

// Epilogues take 16 columns at a time in loops that are not unrolled: with 64 unrolled columns and
// five activations the code outgrew the instruction cache, and a tile that no other product hides
// spent most of its epilogue fetching instructions.
constexpr int kTurnFloats = 32 * 17;

// 32 rows x 16 columns of a warp, lane = row, turned in shared memory (kTurnFloats of the warp's own)
// so that the lanes store along the rows.
__device__ __forceinline__ void turn16(const float (&v)[16], float* turn, int lane) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 16; ++j) turn[lane * 17 + j] = v[j];
  __syncwarp();
}

// The epilogue of 32 rows x 16 columns from the accumulator, lane = row.  Bias and activation come
// before the turn, where a lane has 16 independent values; then two lanes with eight columns each
// take a row, or, where rows do not start on 16-byte boundaries, 16 lanes with one column each.
template <typename T, typename O>
__device__ __forceinline__ void finish_turned(const Epilogue& e, int64_t m0, int64_t M, int64_t n0, int64_t N,
                                              float (&v)[16], float* turn, int lane) {
  add_bias<T, 16>(e, n0, N, v);
  const int64_t n = n0 + (lane & 15);
  const int rows = n < N ? static_cast<int>(M - m0 < 32 ? M - m0 : 32) : 0;
  if (e.z) {
    turn16(v, turn, lane);
    T* z = static_cast<T*>(e.z) + m0 * e.z_stride + n;
#pragma unroll 4
    for (int row = lane >> 4; row < rows; row += 2) z[row * e.z_stride] = from_f<T>(turn[row * 17 + (lane & 15)]);
  }
  activate_all<16>(v, e.act);
  turn16(v, turn, lane);
  if (e.wide) {
    const int64_t n8 = n0 + (lane & 1) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = i * 16 + (lane >> 1);
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = turn[row * 17 + (lane & 1) * 8 + j];
      if (m0 + row < M && n8 < N) add_residual_and_store8<T, O>(e, m0 + row, n8, N, w);
    }
    return;
  }
  O* y = static_cast<O*>(e.y) + m0 * e.y_stride + n;
  const int64_t r0 = m0 * e.residual_stride + n;
#pragma unroll 1
  for (int row = lane >> 4; row < rows; row += 16) {  // eight rows of the lane's column at a time
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = e.residual && row + 2 * i < rows ? load_any<T>(e.residual, r0 + (row + 2 * i) * e.residual_stride, e.residual_f32) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row + 2 * i < rows) y[(row + 2 * i) * e.y_stride] = from_f<O>(f[i] + turn[(row + 2 * i) * 17 + (lane & 15)]);
  }
}

// Rows of 16-bit values that start on any boundary of two bytes, 64 columns (or the first `len` of
// them) by a warp, in words of four bytes: lane l has columns 2l (low half) and 2l + 1.  A row on an odd
// boundary is read and written in words that straddle two lanes' columns; nothing outside the
// columns is touched.  Reading is in two steps, so that the loads of several rows are in flight
// before the first is used; no step branches.  Every lane calls (shuffles).
struct RowWord {
  // the lane's word, where the row has both of its columns; the one column where it has one; column
  // 63 of a row on an odd boundary (lane 31).  Registers of their own: a load into one that another
  // load may still write would wait for it.
  uint32_t both, one, last;
};

__device__ __forceinline__ int odd_row(const uint16_t* row) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1;
}

__device__ __forceinline__ RowWord load_row_word(const uint16_t* row, int len, int lane) {
  const int odd = odd_row(row), low = 2 * lane - odd;
  const bool has_low = low >= 0 && low < len, has_high = low + 1 < len;
  RowWord r{0, 0, 0};
  if (has_low && has_high) r.both = __ldg(reinterpret_cast<const uint32_t*>(row + low));
  if (has_low != has_high) r.one = __ldg(row + (has_low ? low : low + 1));
  if (lane == 31 && 63 < len && odd) r.last = __ldg(row + 63);
  return r;
}

__device__ __forceinline__ uint32_t row_columns(const RowWord& r, int odd, int lane) {
  // a lone column is the high half only in lane 0 of an odd row
  const uint32_t w = r.both | (odd && lane == 0 ? r.one << 16 : r.one);
  const uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
  return odd ? (w >> 16) | ((lane == 31 ? r.last : next) << 16) : w;
}

__device__ __forceinline__ void store_row_word(uint16_t* row, int len, int lane, uint32_t columns) {
  const int odd = odd_row(row), low = 2 * lane - odd;
  const uint32_t before = __shfl_up_sync(0xffffffffu, columns, 1);
  const uint32_t w = odd ? (before >> 16) | (columns << 16) : columns;
  const bool has_low = low >= 0 && low < len, has_high = low + 1 < len;
  if (has_low && has_high) *reinterpret_cast<uint32_t*>(row + low) = w;
  if (has_low && !has_high) row[low] = static_cast<uint16_t>(w);
  if (!has_low && has_high) row[low + 1] = static_cast<uint16_t>(w >> 16);
  if (lane == 31 && 63 < len && odd) row[63] = static_cast<uint16_t>(columns >> 16);
}

// The same for up to 32 rows of 64 columns, word(r) being where the lane's word of row r is kept: the rows
// that start on words and those that do not each in a loop of their own, without tests per row; a row's
// single columns at its ends are lane r's.  Reading is in two steps, so that all rows are on their way
// at once (asynchronous copies of words, which lie one column too far left in odd rows until the
// second step).  With tests per row and eight rows at a time 10,861 x 3278 x 48 took 65 us, with a residual 134
// us; now 38 and 75 us (odd rows, N = 3279: 43 and 89 us; rows that TMA stores, N = 3280: 26 and 43 us).
template <typename W>
__device__ __forceinline__ void store_rows(uint16_t* first, int64_t stride, int rows, int lane, const uint8_t* tile, const W& word) {
  const int classes = 1 + static_cast<int>(stride & 1);
  const int64_t step = stride * classes;  // even
#pragma unroll 1
  for (int c = 0; c < classes; ++c) {
    uint16_t* row = first + c * stride;
    if (!odd_row(row)) {
      uint32_t* to = reinterpret_cast<uint32_t*>(row) + lane;
#pragma unroll 8
      for (int r = c; r < rows; r += classes, to += step / 2) *to = *word(r);
    } else {
      uint32_t* to = reinterpret_cast<uint32_t*>(row - 1) + lane;  // lane 0's is half another's: not stored
#pragma unroll 8
      for (int r = c; r < rows; r += classes, to += step / 2) {
        const uint32_t columns = *word(r), before = __shfl_up_sync(0xffffffffu, columns, 1);
        if (lane > 0) *to = (before >> 16) | (columns << 16);
      }
    }
  }
  uint16_t* own = first + lane * stride;
  if (lane < rows && odd_row(own)) {
    own[0] = *reinterpret_cast<const uint16_t*>(tile + lane * 128 + ((lane & 7) << 4));
    own[63] = *reinterpret_cast<const uint16_t*>(tile + lane * 128 + ((7 ^ (lane & 7)) << 4) + 14);
  }
}

// First step; the result is the lane's row's first (low half) and last column, where it starts on an odd one.
template <typename W>
__device__ __forceinline__ uint32_t begin_rows(const uint16_t* first, int64_t stride, int rows, int lane, const W& word) {
  uint32_t ends = 0;
  const uint16_t* own = first + lane * stride;
  if (lane < rows && odd_row(own)) ends = __ldg(own) | static_cast<uint32_t>(__ldg(own + 63)) << 16;
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    const int odd = odd_row(first + r * stride);
    const uint32_t* from = reinterpret_cast<const uint32_t*>(first + r * stride - odd) + lane;
    if (lane >= odd)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(word(r))), "l"(from) : "memory");
  }
  return ends;
}
template <typename W>
__device__ __forceinline__ void finish_rows(const uint16_t* first, int64_t stride, int rows, int lane, uint32_t ends, const W& word) {
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    if (!odd_row(first + r * stride)) continue;  // warp-uniform
    const uint32_t end = __shfl_sync(0xffffffffu, ends, r);
    const uint32_t mine = lane == 0 ? end << 16 : *word(r), next = __shfl_down_sync(0xffffffffu, mine, 1);
    *word(r) = (mine >> 16) | (lane == 31 ? end & 0xffff0000u : next << 16);
  }
  __syncwarp();
}

struct LinearShape {
  int64_t M, N;
  int k_steps;         // of 64 columns of K
  int m_tiles, n_tiles;
  int a_rows;          // rows of A's box: 128, or M rounded up to 8 where M is smaller (K-major)
  int a_mn, b_mn, bf16;
  int stages;          // of the tile kernel
};

// ---------------------------------------------------------------- one tile per CTA, K split over a cluster
// Tile 128 x BN.  gridDim.x = tiles * splits; the CTAs of a cluster share a tile and take
// consecutive parts of K, then each sums a share of the tile's columns over all of them through
// distributed shared memory, in rank order (deterministic).  Two CTAs fit an SM, so that one's
// epilogue overlaps another's products.
// PROMOTE (32-bit outputs): the tensor core's running sum loses about one part in 2^20 over a
// few thousand terms (its additions truncate), which 16-bit outputs do not see; here a sum
// covers 512 of K at most, and FP32 registers add those up.
// SWAP (few rows of x): A is the weight and B is x, so that 128 rows of the weight meet 16 or 32
// rows of x without tiles that are mostly padding; the epilogue's roles of rows and columns change
// places with them (M and N here are those of the swapped product).
// Epilogue: four warps bring the accumulator to shared memory, [column][129] floats so that threads
// may read it along either dimension; then all ten warps take rows or elements of it along y's rows,
// each thread with a column (and its bias) of its own.  A tile that no other product hides is bound by
// the latency of its epilogue's few warps: with four warps alone, one lane per row, 2910 x 94 x 192
// with a residual took 26 us.
// Warps: 0-3 accumulator (one per TMEM lane quadrant), 4 TMA producer, 5 MMA issuer and TMEM owner.
// Threads: the ten warps named above; swapped tiles have few columns to finish and start sooner with six.
template <bool SWAP>
constexpr int kThreadsOf = SWAP ? 192 : 320;
constexpr int kPartStride = 129;

template <int BN, bool PROMOTE>
struct TileSmem {
  static constexpr int kA = 128 * 128;
  static constexpr int kB = BN * 128;
  static constexpr int kStageBytes = kA + kB;
  // stages where two CTAs share an SM, and where a CTA has one alone: more loads in flight then
  // make up for the second CTA's (1110 cycles per K step of 128 x 128 with three stages)
  static constexpr int kStages = BN >= 128 ? 3 : BN == 64 ? 4 : BN == 32 ? 5 : 6;
  static constexpr int kStagesAlone = BN >= 128 ? 6 : 8;
  // after the stages: full, empty [stages]; tfull, tempty [2]; TMEM address
  static constexpr int bytes(int stages) { return stages * kStageBytes + (2 * stages + 4) * 8 + 16 + 1024; }
  static constexpr int kBytes = bytes(kStages);
  static constexpr int kAccs = PROMOTE ? 2 : 1;
  static constexpr int kTmemCols = kAccs * BN < 32 ? 32 : kAccs * BN;
  static_assert(kPartStride * BN * 4 <= kStages * kStageBytes, "the accumulator's copy reuses the stages");
  static_assert(2 * kBytes <= 228 * 1024, "two CTAs per SM");
  static_assert(bytes(kStagesAlone) <= 232448, "shared memory per CTA");
};

constexpr int kPromoteSteps = 8;  // K steps of 64 per running sum

template <typename T, typename O, int BN, bool PROMOTE, bool SWAP>
__global__ void __launch_bounds__(kThreadsOf<SWAP>)
    cdg_linear_tile_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                           const LinearShape s, const Epilogue e, const int splits) {
  using L = TileSmem<BN, PROMOTE>;
  const int S = s.stages;
  constexpr int CC = 16;  // columns taken out of TMEM at a time
  constexpr int kTileThreads = kThreadsOf<SWAP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * L::kStageBytes);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = static_cast<int>(blockIdx.x) / splits, split = static_cast<int>(blockIdx.x) % splits;
  const int m0 = (tile % s.m_tiles) * 128, n0 = (tile / s.m_tiles) * BN;
  const int k_first = static_cast<int>(static_cast<int64_t>(s.k_steps) * split / splits);
  const int k_last = static_cast<int>(static_cast<int64_t>(s.k_steps) * (split + 1) / splits);
  const int sums = PROMOTE ? (k_last - k_first + kPromoteSteps - 1) / kPromoteSteps : (k_last > k_first ? 1 : 0);

  if (warp == 4 && lane == 0) {
    if (s.k_steps > 0) {  // K = 0 has no operands and no maps
      prefetch_tmap(&tmap_a);
      prefetch_tmap(&tmap_b);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 128);
    }
    fence_mbarrier_init();
  }
  // operands may be the previous kernel's results; nor does this kernel take TMEM from it
  grid_dependency_wait();
  grid_launch_dependents();
  if (warp == 5) {
    tmem_alloc(tmem_holder, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  bool ok = true;
  float acc[PROMOTE ? BN : 1];

  if (warp == 4) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      // boxes past M (MN-major, in chunks of 64) are not loaded: their rows of the result are not stored
      const int a_chunks = s.a_mn ? (s.M - m0 > 64 ? 2 : 1) : 0;
      const uint32_t bytes = (s.a_mn ? a_chunks * 8192u : static_cast<uint32_t>(s.a_rows) * 128u) + L::kB;
      for (int k = k_first; k < k_last; ++k) {
        if (!mbar_wait_cta(&empty[stage], phase ^ 1, nullptr, wait_code(1, 0, stage, phase ^ 1, k))) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], bytes);
        uint8_t* a = smem + stage * L::kStageBytes;
        uint8_t* b = a + L::kA;
        if (s.a_mn) {
          for (int c = 0; c < a_chunks; ++c) tma_load_2d(a + c * 8192, &tmap_a, &full[stage], m0 + c * 64, k * 64);
        } else {
          tma_load_2d(a, &tmap_a, &full[stage], k * 64, m0);
        }
        if (s.b_mn) {
#pragma unroll
          for (int c = 0; c < (BN + 63) / 64; ++c)
            tma_load_2d(b + c * 8192, &tmap_b, &full[stage], n0 + c * 64, k * 64);  // BN of 64 or 128 alone
        } else {
          tma_load_2d(b, &tmap_b, &full[stage], k * 64, n0);
        }
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    const uint32_t idesc = idesc_f16(s.bf16, s.a_mn, s.b_mn, 128, BN);
    const uint32_t a_step = operand_k_step(s.a_mn), b_step = operand_k_step(s.b_mn);
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0, k = k_first; i < sums && ok; ++i) {
      const int buf = PROMOTE ? i & 1 : 0;
      if (PROMOTE && !mbar_wait_cta_warp(&tempty[buf], ((i >> 1) & 1) ^ 1, nullptr, wait_code(2, 0, buf, i, k))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int end = PROMOTE ? min(k_last, k + kPromoteSteps) : k_last;
      for (bool first = true; k < end; ++k) {
        if (!mbar_wait_cta_warp(&full[stage], phase, nullptr, wait_code(3, 0, stage, phase, k))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t base = smem_u32(smem + stage * L::kStageBytes);
        const uint64_t ad = operand_desc(base, s.a_mn), bd = operand_desc(base + L::kA, s.b_mn);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          tc_mma_f16_warp(tmem + buf * BN, ad + j * a_step, bd + j * b_step, idesc, first ? 0u : 1u);
          first = false;
        }
        tc_commit_warp(&empty[stage]);
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
      if (ok) tc_commit_warp(&tfull[buf]);
    }
  } else if (warp < 4) {
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // every product of this CTA has completed before anything is written here: the stages are free
    float* part = reinterpret_cast<float*>(smem) + warp * 32 + lane;
    if constexpr (PROMOTE) {
#pragma unroll
      for (int j = 0; j < BN; ++j) acc[j] = 0.0f;
      for (int i = 0; i < sums && ok; ++i) {
        const int buf = i & 1;
        if (!mbar_wait_cta_warp(&tfull[buf], (i >> 1) & 1, nullptr, wait_code(4, 0, buf, i >> 1, i))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < BN / CC; ++c) {
          uint32_t r[CC];
          tmem_ld16(lanes + buf * BN + c * CC, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < CC; ++j) acc[c * CC + j] += __uint_as_float(r[j]);
        }
        tc_fence_before();
        mbar_arrive(&tempty[buf]);
      }
    } else {
      if (sums && !mbar_wait_cta_warp(&tfull[0], 0, nullptr, wait_code(4, 0, 0, 0, 0))) ok = false;
      tc_fence_after();
    }
    if (ok) {
      if constexpr (PROMOTE) {
#pragma unroll
        for (int j = 0; j < BN; ++j) part[j * kPartStride] = acc[j];
      } else {
#pragma unroll 1
        for (int at = 0; at < BN; at += CC) {
          uint32_t r[CC];
          tmem_ld16(lanes + at, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < CC; ++j)
            part[(at + j) * kPartStride] = sums ? __uint_as_float(r[j]) : 0.0f;  // K = 0: nothing was summed
        }
      }
    }
  }

  // every thread takes part from here on, also where a wait gave up (the sums are then wrong, and the
  // device record says so)
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  const int t = threadIdx.x;
  const int share = 128 / splits, row0 = split * share;  // this CTA's rows of the tile
  const int rows = static_cast<int>(s.M - m0 - row0 < share ? s.M - m0 - row0 : share);  // below 1: none
  const int cols = static_cast<int>(s.N - n0 < BN ? s.N - n0 : BN);
  // The accumulator at one place: the sum over the cluster's CTAs (eight at most), in rank order, all
  // of the (remote) reads in flight together.
  auto total = [&](const float* at) {
    if (splits == 1) return *at;
    float f[8], v = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      f[r] = 0.0f;
      if (r < splits) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[r]) : "r"(cluster_addr(at, r)));
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) v += f[r];
    return v;
  };
  // The accumulator at eight places: each the sum over the cluster's CTAs, in rank order; the eight
  // (remote) reads of a CTA are in flight together.
  auto totals = [&](const float* at, int step, int count, float (&v)[8]) {
    if (splits == 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < count ? at[j * step] : 0.0f;
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
#pragma unroll 2
    for (int r = 0; r < splits; ++r) {
      const uint32_t base = cluster_addr(at, r);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = 0.0f;
        if (j < count) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[j]) : "r"(base + j * step * 4));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += f[j];
    }
  };
  if constexpr (SWAP) {
    // rows of the weight run along y: a thread keeps one of this CTA's and takes columns, two at a time
    // where K is split (it mostly has one; eight cost 1.4 us of predicated work), else eight, so that
    // their residual loads are in flight together
    const int row = row0 + t % share, lanes = kTileThreads / share;
    const int64_t n = m0 + row;
    auto columns = [&](auto width) {
      constexpr int U = decltype(width)::value;
      const float bias = e.bias ? load_any<T>(e.bias, n, e.bias_f32) : 0.0f;
      for (int c = t / share; c < cols; c += lanes * U) {
        float v[U], r[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int col = c + j * lanes;
          r[j] = e.residual && col < cols ? load_any<T>(e.residual, (n0 + col) * e.residual_stride + n, e.residual_f32) : 0.0f;
          v[j] = bias + (col < cols ? total(part + col * kPartStride + row) : 0.0f);
        }
        if (e.z) {
#pragma unroll
          for (int j = 0; j < U; ++j)
            if (c + j * lanes < cols) static_cast<T*>(e.z)[(n0 + c + j * lanes) * e.z_stride + n] = from_f<T>(v[j]);
        }
        activate_all<U>(v, e.act);
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (c + j * lanes < cols) static_cast<O*>(e.y)[(n0 + c + j * lanes) * e.y_stride + n] = from_f<O>(v[j] + r[j]);
      }
    };
    if (n < s.M && t < lanes * share) {
      if (splits == 1)
        columns(std::integral_constant<int, 8>());
      else
        columns(std::integral_constant<int, 2>());
    }
  } else if (e.wide && splits > 1) {
    // consecutive threads take consecutive rows, so that remote reads are contiguous
    for (int item = t; item < share * (BN / 8); item += kTileThreads) {
      const int row = item % share, col = item / share * 8;
      if (row >= rows || col >= cols) continue;
      float bias[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) bias[j] = e.bias && col + j < cols ? load_any<T>(e.bias, n0 + col + j, e.bias_f32) : 0.0f;
      totals(part + col * kPartStride + row0 + row, kPartStride, 8, v);
      finish8<T, O>(e, m0 + row0 + row, n0 + col, s.N, bias, v);
    }
  } else if (e.wide) {
    // a thread keeps eight columns (and their bias) and takes rows, along y's rows
    constexpr int kGroups = BN / 8;
    const int col = t % kGroups * 8;
    if (col < cols) {
      float bias[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) bias[j] = e.bias && col + j < cols ? load_any<T>(e.bias, n0 + col + j, e.bias_f32) : 0.0f;
#pragma unroll 2
      for (int row = t / kGroups; row < rows; row += kTileThreads / kGroups) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = part[(col + j) * kPartStride + row];
        finish8<T, O>(e, m0 + row, n0 + col, s.N, bias, v);
      }
    }
  } else {
    if (splits > 1) {
      // the sums in place: only this CTA reads these rows of its own copy
      for (int item = t; item < share * (BN / 8); item += kTileThreads) {
        float* at = part + item / share * 8 * kPartStride + row0 + item % share;
        float v[8];
        totals(at, kPartStride, 8, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) at[j * kPartStride] = v[j];
      }
      __syncthreads();
    }
    // a warp takes rows; a lane keeps two columns of 64 (16-bit results), or every 32nd (FP32)
    if constexpr (sizeof(O) == 2) {
      for (int c0 = 0; c0 < cols; c0 += 64) {
        const int len = cols - c0 < 64 ? cols - c0 : 64;
        const int64_t n = n0 + c0;
        float bias[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) bias[j] = e.bias && 2 * lane + j < len ? load_any<T>(e.bias, n + 2 * lane + j, e.bias_f32) : 0.0f;
        constexpr int U = 4;  // rows at a time
        for (int row = warp; row < rows; row += U * (kTileThreads / 32)) {
          RowWord raw[U];
          float r[U][2];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int64_t m = m0 + row0 + row + i * (kTileThreads / 32);
            const int l = row + i * (kTileThreads / 32) < rows ? len : 0;
            r[i][0] = r[i][1] = 0.0f;
            if (e.residual && !e.residual_f32) {
              raw[i] = load_row_word(static_cast<const uint16_t*>(e.residual) + m * e.residual_stride + n, l, lane);
            } else if (e.residual) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (2 * lane + j < l) r[i][j] = load_any<T>(e.residual, m * e.residual_stride + n + 2 * lane + j, 1);
            }
          }
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int at = row + i * (kTileThreads / 32);
            if (at >= rows) break;  // warp-uniform
            const int64_t m = m0 + row0 + at;
            if (e.residual && !e.residual_f32) {
              const uint16_t* from = static_cast<const uint16_t*>(e.residual) + m * e.residual_stride + n;
              const float2 f = unpack2(row_columns(raw[i], odd_row(from), lane), T());
              r[i][0] = f.x;
              r[i][1] = f.y;
            }
            float v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] = part[(c0 + 2 * lane + j) * kPartStride + row0 + at] + bias[j];
            if (e.z) store_row_word(static_cast<uint16_t*>(e.z) + m * e.z_stride + n, len, lane, pack2(v[0], v[1], T()));
            activate_all<2>(v, e.act);
            store_row_word(static_cast<uint16_t*>(e.y) + m * e.y_stride + n, len, lane,
                           pack2(v[0] + r[i][0], v[1] + r[i][1], O()));
          }
        }
      }
    } else {
      for (int c = lane; c < cols; c += 32) {
        const int64_t n = n0 + c;
        const float bias = e.bias ? load_any<T>(e.bias, n, e.bias_f32) : 0.0f;
#pragma unroll 4
        for (int row = warp; row < rows; row += kTileThreads / 32) {
          const int64_t m = m0 + row0 + row;
          const float r = e.residual ? load_any<T>(e.residual, m * e.residual_stride + n, e.residual_f32) : 0.0f;
          float v[1] = {part[c * kPartStride + row0 + row] + bias};
          if (e.z) static_cast<T*>(e.z)[m * e.z_stride + n] = from_f<T>(v[0]);
          activate_all<1>(v, e.act);
          static_cast<O*>(e.y)[m * e.y_stride + n] = v[0] + r;
        }
      }
    }
  }
  if (splits > 1) cluster_sync();  // no CTA leaves while another reads its shared memory
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    // after a wait that gave up, copies issued before it still land: give them time before exit
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(20000);
  }
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// ---------------------------------------------------------------- CTA pairs, persistent, for many tiles
// A pair of CTAs takes tiles of 256 x BN (256) in turn: CTA r of it holds rows 128r .. 128r + 127 of A and
// of the result and half of B's rows.  The tensor cores fill one of two accumulators in TMEM while
// sixteen epilogue warps per CTA empty the other (warp w: the 32 lanes of quadrant w % 4, a quarter of
// the columns; eight warps of half the columns each, two per scheduler, waited for their own
// instructions and took 4.3 us a tile, more than the products of K = 512).  Staged (y, and the
// residual where there is one, of the output's type and on 16-byte rows, z not stored): each epilogue
// warp has the residual brought into its own shared-memory tile of 32 rows x 128 bytes by TMA, ahead
// of the accumulator, adds it in place and has the result stored from there, so that global memory
// sees whole tiles; clipping at M and N is TMA's.  Where rows start or end on other boundaries, the warp
// itself copies the residual's rows in and the result's out, in whole words (10,861 x 3279 x 48 with a
// residual: 226 us with single elements, 89 us so).  With z, or a residual of another type, its lanes turn
// their columns and store along the rows.
// Warps: 0 TMA producer, 1 MMA issuer (even CTA) and TMEM owner, 4-19 epilogue.
template <int BN>
struct PairTileSmem {
  static constexpr int kA = 128 * 128;
  static constexpr int kB = BN / 2 * 128;
  static constexpr int kStageBytes = kA + kB;
  static constexpr int kStages = 5;
  static constexpr int kEpiWarps = 16;
  static constexpr int kStaging = kStages * kStageBytes;      // [warp] tiles of 4096 bytes
  static constexpr int kBars = kStaging + kEpiWarps * 4096;
  // full, empty [kStages]; tfull, tempty [2]; done; residual [warp]; TMEM address
  static constexpr int kBytes = kBars + (2 * kStages + 5 + kEpiWarps) * 8 + 16 + 1024;
  static_assert(kTurnFloats * 4 <= 4096, "a warp turns its columns in its staged tile");
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static_assert(kBytes <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ void tc_mma_f16_pair_warp(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                     uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 2-D tiled store of one box from shared memory (bulk group of the issuing thread).
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// The stores issued by this thread have read their shared memory / have completed.
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Tile t of a grid of m_tiles x n_tiles: bands of kBand row tiles, column by column, so that the
// tiles in flight share their operands in L2.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int band = t / (kBand * n_tiles), first = band * kBand;
  const int height = min(kBand, m_tiles - first), in = t - band * kBand * n_tiles;
  mt = first + in % height;
  nt = in / height;
}

// The epilogue of 32 consecutive columns from n on of the lane's row, in place of the residual in
// the staged tile (row `lane`, 128 bytes, 16-byte pieces XORed with the row's low three bits: the
// 128-byte swizzle); `first` is the columns' first piece.
template <typename T, typename O>
__device__ __forceinline__ void finish_staged(const Epilogue& e, int64_t n, int64_t N, float (&v)[32], uint8_t* tile,
                                              int first, int lane) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(O));  // columns per 16-byte piece
  add_bias<T, 32>(e, n, N, v);
  activate_all<32>(v, e.act);
#pragma unroll
  for (int c = 0; c < 32 / kPer; ++c) {
    uint4* at = reinterpret_cast<uint4*>(tile + lane * 128 + (((first + c) ^ (lane & 7)) << 4));
    if constexpr (sizeof(O) == 4) {
      *at = make_uint4(__float_as_uint(v[c * 4]), __float_as_uint(v[c * 4 + 1]), __float_as_uint(v[c * 4 + 2]),
                       __float_as_uint(v[c * 4 + 3]));
    } else {
      if (e.residual) {
        const uint4 r = *at;
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2(w[j], O());
          v[c * 8 + 2 * j] += f.x;
          v[c * 8 + 2 * j + 1] += f.y;
        }
      }
      *at = make_uint4(pack2(v[c * 8], v[c * 8 + 1], O()), pack2(v[c * 8 + 2], v[c * 8 + 3], O()),
                       pack2(v[c * 8 + 4], v[c * 8 + 5], O()), pack2(v[c * 8 + 6], v[c * 8 + 7], O()));
    }
  }
}

template <typename T, typename O, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairTileSmem<BN>::kThreads, 1)
    cdg_linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                           const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ CUtensorMap tmap_r,
                           const LinearShape s, const Epilogue e) {
  using L = PairTileSmem<BN>;
  constexpr bool PROMOTE = sizeof(O) == 4;
  constexpr int S = L::kStages;
  constexpr int CH = 128 / static_cast<int>(sizeof(O));  // columns of a staged tile
  constexpr int kCols = BN / 4;                          // columns of an epilogue warp: CH, or 2 CH in FP32
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;
  uint64_t* rfull = done + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(rfull + L::kEpiWarps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
  const int tiles = s.m_tiles * s.n_tiles;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * 32 * L::kEpiWarps);
    }
    mbar_init(done, 1);
    for (int i = 0; i < L::kEpiWarps; ++i) mbar_init(&rfull[i], 1);
    fence_mbarrier_init();
  }
  // operands may be the previous kernel's results; nor does this kernel take TMEM from it
  grid_dependency_wait();
  grid_launch_dependents();
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers ready before any copy or commit reaches them
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t full0 = cluster_addr(&full[0], 0);
      for (int t = pair; t < tiles && ok; t += pairs) {
        int mt, nt;
        tile_at(t, s.m_tiles, s.n_tiles, mt, nt);
        const int m0 = mt * 256 + static_cast<int>(rank) * 128, n0 = nt * BN + static_cast<int>(rank) * (BN / 2);
        for (int k = 0; k < s.k_steps; ++k) {
          if (!mbar_wait_cluster(&empty[stage], phase ^ 1, nullptr, wait_code(1, static_cast<int>(rank), stage, phase ^ 1, k))) {
            ok = false;
            break;
          }
          const uint32_t fb = full0 + stage * 8;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2u * L::kStageBytes);
          uint8_t* a = smem + stage * L::kStageBytes;
          uint8_t* b = a + L::kA;
          if (s.a_mn) {
            tma_load_2d_pair(a, &tmap_a, fb, m0, k * 64);
            tma_load_2d_pair(a + 8192, &tmap_a, fb, m0 + 64, k * 64);
          } else {
            tma_load_2d_pair(a, &tmap_a, fb, k * 64, m0);
          }
          if (s.b_mn) {
#pragma unroll
            for (int c = 0; c < BN / 128; ++c) tma_load_2d_pair(b + c * 8192, &tmap_b, fb, n0 + c * 64, k * 64);
          } else {
            tma_load_2d_pair(b, &tmap_b, fb, k * 64, n0);
          }
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = idesc_f16(s.bf16, s.a_mn, s.b_mn, 256, BN);
      const uint32_t a_step = operand_k_step(s.a_mn), b_step = operand_k_step(s.b_mn);
      int stage = 0, sum = 0;
      uint32_t phase = 0;
      for (int t = pair; t < tiles && ok; t += pairs) {
        for (int k = 0; k < s.k_steps && ok; ++sum) {
          const int buf = sum & 1;
          if (!mbar_wait_cluster_warp(&tempty[buf], ((sum >> 1) & 1) ^ 1, nullptr, wait_code(2, 0, buf, sum >> 1, k))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int end = PROMOTE ? min(s.k_steps, k + kPromoteSteps) : s.k_steps;
          for (uint32_t more = 0; k < end; ++k) {
            if (!mbar_wait_cta_warp(&full[stage], phase, nullptr, wait_code(3, 0, stage, phase, k))) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t base = smem_u32(smem + stage * L::kStageBytes);
            const uint64_t ad = operand_desc(base, s.a_mn), bd = operand_desc(base + L::kA, s.b_mn);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              tc_mma_f16_pair_warp(tmem + buf * BN, ad + j * a_step, bd + j * b_step, idesc, more);
              more = 1;
            }
            tc_commit_pair_warp(&empty[stage], 0x3);
            if (++stage == S) { stage = 0; phase ^= 1; }
          }
          if (ok) tc_commit_pair_warp(&tfull[buf], 0x3);
        }
      }
      tc_commit_pair_warp(done, 0x1);  // every product completes before teardown
      mbar_wait_cluster_warp(done, 0, nullptr, wait_code(5, 0, 0, 0, 0));
    }
  } else if (warp >= 4) {
    const int w = warp - 4, quarter = w >> 2, q = warp & 3;
    const uint32_t tempty0 = cluster_addr(&tempty[0], 0);
    uint8_t* tile = smem + L::kStaging + w * 4096;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16) + quarter * kCols;
    int sum = 0;
    uint32_t turn = 0;  // phase of the staged tile's residual barrier
    for (int t = pair; t < tiles && ok; t += pairs) {
      int mt, nt;
      tile_at(t, s.m_tiles, s.n_tiles, mt, nt);
      const int row0 = mt * 256 + static_cast<int>(rank) * 128 + q * 32, col0 = nt * BN + quarter * kCols;
      const bool any = row0 < s.M && col0 < s.N;  // a warp past the edges only keeps the barriers moving
      if (e.staged && any) {
        if (lane == 0) {
          bulk_wait_read();  // the last tile's store has read the staged tile
          if (e.residual && e.staged == 1) {  // with 16-bit results alone
            mbar_arrive_expect_tx(&rfull[w], 4096);
            tma_load_2d(tile, &tmap_r, &rfull[w], col0, row0);
          }
        }
        __syncwarp();
      }
      // the rows and (staged) columns of this warp that exist
      const int rows = any ? static_cast<int>(s.M - row0 < 32 ? s.M - row0 : 32) : 0;
      const int len = any ? static_cast<int>(s.N - col0 < CH ? s.N - col0 : CH) : 0;
      // word l of row r of the staged tile
      auto word = [&](int r) { return reinterpret_cast<uint32_t*>(tile + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4); };
      uint32_t ends = 0;
      const uint16_t* r0 = static_cast<const uint16_t*>(e.residual) + row0 * e.residual_stride + col0;
      if (!PROMOTE && e.staged == 2 && e.residual) {
        if (len == CH) {
          ends = begin_rows(r0, e.residual_stride, rows, lane, word);
        } else {
#pragma unroll 1
          for (int r = 0; r < rows; r += 8) {
            RowWord raw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = load_row_word(r0 + (r + i) * e.residual_stride, r + i < rows ? len : 0, lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) *word(r + i) = row_columns(raw[i], odd_row(r0 + (r + i) * e.residual_stride), lane);
          }
          __syncwarp();
        }
      }
      if constexpr (PROMOTE) {
        float acc[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) acc[j] = 0.0f;
        for (int k = 0; k < s.k_steps; k += kPromoteSteps, ++sum) {
          const int buf = sum & 1;
          if (!mbar_wait_cluster_warp(&tfull[buf], (sum >> 1) & 1, nullptr, wait_code(4, static_cast<int>(rank), buf, sum >> 1, k))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kCols / 16; ++c) {
            uint32_t r[16];
            tmem_ld16(lanes + buf * BN + c * 16, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c * 16 + j] += __uint_as_float(r[j]);
          }
          tc_fence_before();
          if (rank == 0) mbar_arrive(&tempty[buf]); else mbar_arrive_cluster(tempty0 + buf * 8);
        }
        if (!ok) break;
        if (!any) continue;
        if (e.staged) {
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c) {
            const int n = col0 + c * 32;
            if (n >= s.N) break;
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = acc[c * 32 + j];
            if (c > 0) {
              if (lane == 0) bulk_wait_read();
              __syncwarp();
            }
            finish_staged<T, O>(e, n, s.N, v, tile, 0, lane);
            if (e.staged == 2) {
              __syncwarp();
              float* y0 = static_cast<float*>(e.y) + row0 * e.y_stride + n + lane;
              if (n + lane < s.N) {
#pragma unroll 4
                for (int r = 0; r < rows; ++r) y0[r * e.y_stride] = __uint_as_float(*word(r));
              }
              __syncwarp();
              continue;
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_y, tile, n, row0);
              bulk_commit();
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < kCols / 16; ++c) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = acc[c * 16 + j];
            if (col0 + c * 16 < s.N)
              finish_turned<T, O>(e, row0, s.M, col0 + c * 16, s.N, v, reinterpret_cast<float*>(tile), lane);
          }
        }
      } else {
        const int buf = sum & 1;
        if (!mbar_wait_cluster_warp(&tfull[buf], (sum >> 1) & 1, nullptr, wait_code(4, static_cast<int>(rank), buf, sum >> 1, 0))) {
          ok = false;
          break;
        }
        ++sum;
        tc_fence_after();
        auto drained = [&]() {  // this thread has taken its part of the accumulator
          tc_fence_before();
          if (rank == 0) mbar_arrive(&tempty[buf]); else mbar_arrive_cluster(tempty0 + buf * 8);
        };
        if (!any) {
          drained();
          continue;
        }
        if (e.staged) {
          if (e.residual && e.staged == 1) {
            if (!mbar_wait_cta_warp(&rfull[w], turn, nullptr, wait_code(4, 8 + w % 8, w, turn, 0))) ok = false;
            turn ^= 1;
          }
          if (e.residual && e.staged == 2 && len == CH) finish_rows(r0, e.residual_stride, rows, lane, ends, word);
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            uint32_t r[2][16];
            tmem_ld16(lanes + buf * BN + c, r[0]);
            tmem_ld16(lanes + buf * BN + c + 16, r[1]);
            tmem_ld_wait();
            if (c + 32 >= kCols) drained();
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j / 16][j % 16]);
            if (col0 + c < s.N) finish_staged<T, O>(e, col0 + c, s.N, v, tile, c * static_cast<int>(sizeof(O)) / 16, lane);
          }
          if (e.staged == 2) {
            __syncwarp();
            uint16_t* y0 = static_cast<uint16_t*>(e.y) + row0 * e.y_stride + col0;
            if (len == CH) {
              store_rows(y0, e.y_stride, rows, lane, tile, word);
            } else {
#pragma unroll 4
              for (int r = 0; r < rows; ++r) store_row_word(y0 + r * e.y_stride, len, lane, *word(r));
            }
            __syncwarp();
            continue;
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmap_y, tile, col0, row0);
            bulk_commit();
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kCols; c += 16) {
            uint32_t r[16];
            tmem_ld16(lanes + buf * BN + c, r);
            tmem_ld_wait();
            if (c + 16 >= kCols) drained();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
            if (col0 + c < s.N)
              finish_turned<T, O>(e, row0, s.M, col0 + c, s.N, v, reinterpret_cast<float*>(tile), lane);
          }
        }
      }
    }
    if (e.staged && lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  const int any_fail = __syncthreads_or(!ok);
  cluster_sync();  // no CTA releases TMEM or exits while its pair still uses it
  if (any_fail) {
    // after a wait that gave up, copies issued before it still land: give them time before exit
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(20000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

}  // namespace
}  // namespace cdg
