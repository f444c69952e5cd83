// Host side of the dense product (cdg_linear, cdg_linear_backward) and its elementwise kernels.
//
//   forward   y = act(x W^T + b) + r                                   one product
//   backward  dz = dy * act'(z), db = sum over rows of dz, dx = dz W, dW = dz^T x
//             one elementwise pass (dz in the operands' 16 bits, since it is an operand of both
//             products; db from its 32-bit values), then two products that read W and dz across
//             their rows (MN-major operands), so nothing is transposed in memory
//
// Operands whose rows do not start on 16-byte boundaries cannot be loaded by TMA: they are copied
// once into the workspace with padded rows.
//
// One B200, short replays: 8192 x 4096 x 4096 with bias, GELU and residual 200 us (1.38 PFLOP/s), gradient of
// 8192 x 2048 x 4096 with SiLU and bias 223 us; 32,768 x 256 x 4096 with FP32 results 68 us; 1 x 4096 x 4096
// 10 us.  Back to back for seconds the power limit lowers the clock: the first takes 233 us (1.18
// PFLOP/s) then, the bare product 213 us, the library's 216 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "cdg_b200.h"
#include "cdg_linear.cuh"

namespace cdg {
namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Copies rows of 16-bit values to rows of `out_stride` columns, zeros past `cols`; one or two
// matrices (blockIdx.y).  A warp takes 256 columns of a row, so that few long rows are as many warps as
// many short ones (with a warp per row, 192 x 5729 took 27 us, now 4); a row on an odd boundary is read in the
// words that its columns share.
struct Repack {
  const uint16_t* in;
  int64_t in_stride, rows, cols;
  uint16_t* out;
  int64_t out_stride;
  int64_t parts;  // of 256 columns per row
};

__global__ void __launch_bounds__(256) repack_rows_kernel(const Repack first, const Repack second) {
  grid_dependency_wait();  // the workspace may still be in the previous kernel's use
  grid_launch_dependents();
  const Repack p = blockIdx.y == 0 ? first : second;
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < p.rows * p.parts; item += warps) {
    const int64_t r = item / p.parts, c = (item - r * p.parts) * 256 + lane * 8;
    if (c >= p.out_stride) continue;
    const uint16_t* from = p.in + r * p.in_stride + c;
    const bool odd = reinterpret_cast<uintptr_t>(from) % 4 != 0;
    uint32_t w[4];
    if (!odd && c + 8 <= p.cols) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint32_t*>(from) + j);
    } else if (odd && c > 0 && c + 9 <= p.cols) {
      uint32_t shared[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) shared[j] = __ldg(reinterpret_cast<const uint32_t*>(from - 1) + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (shared[j] >> 16) | (shared[j + 1] << 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < p.cols ? from[2 * j] : 0, hi = c + 2 * j + 1 < p.cols ? from[2 * j + 1] : 0;
        w[j] = lo | (hi << 16);
      }
    }
    *reinterpret_cast<uint4*>(p.out + r * p.out_stride + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// dz = dy * act'(z) and partial column sums of it.  A CTA takes 256 columns (eight per lane of
// each of its eight warps) and every gridDim.y-th group of eight rows; its sums go to
// partial[blockIdx.y][N].  dz or partial may be NULL.  Bound by memory: 8192 x 2048 BF16 (101 MB) in
// 19.5 us, 5.2 TB/s.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) linear_dz_kernel(const T* dy, int64_t dy_stride, const T* z, int64_t z_stride,
                                                        int act, int64_t M, int64_t N, T* dz, int64_t dz_stride,
                                                        float* partial) {
  __shared__ float sums[8][256];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t chunk = blockIdx.x;
  float acc[8] = {};
  for (int64_t m = static_cast<int64_t>(blockIdx.y) * 8 + warp; m < M; m += static_cast<int64_t>(gridDim.y) * 8) {
    float g[8];
    unpack8<T>(load8<T, WIDE>(dy + m * dy_stride, chunk, lane, N), g);
    if (z) {
      float v[8];
      unpack8<T>(load8<T, WIDE>(z + m * z_stride, chunk, lane, N), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] *= activate_slope(v[j], act);
    }
    if (dz) store8<T, WIDE>(dz + m * dz_stride, chunk, lane, N, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += g[j];
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[warp][column<WIDE>(0, lane, j)] = acc[j];
  __syncthreads();
  const int64_t n = chunk * 256 + threadIdx.x;
  if (n < N) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sums[i][threadIdx.x];
    partial[static_cast<int64_t>(blockIdx.y) * N + n] = v;
  }
}

// ------------------------------------------------------------------ host
template <typename T, typename O, int BN, bool SWAP>
bool allow_smem() {
  constexpr bool PROMOTE = sizeof(O) == 4;
  using L = TileSmem<BN, PROMOTE>;
  return cudaFuncSetAttribute(cdg_linear_tile_kernel<T, O, BN, PROMOTE, SWAP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              std::max(L::kBytes, L::bytes(L::kStagesAlone))) == cudaSuccess;
}

template <typename T, typename O, int BN>
bool allow_pair_smem() {
  return cudaFuncSetAttribute(cdg_linear_pair_kernel<T, O, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              PairTileSmem<BN>::kBytes) == cudaSuccess;
}

template <typename T, typename O>
bool allow_smem_for() {
  return allow_pair_smem<T, O, 256>() && allow_smem<T, O, 64, false>() && allow_smem<T, O, 128, false>() &&
         allow_smem<T, O, 16, true>() && allow_smem<T, O, 32, true>();
}

template <typename T>
bool allow_smem_of() {
  return allow_smem_for<T, T>() && allow_smem_for<T, float>();
}

// Compute capability and kernel attributes, once per device.
int device_ready() {
  static std::once_flag flags[kMaxDevices];
  static int state[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CDG_ERR_CUDA;
  std::call_once(flags[dev], [dev] {
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
      state[dev] = CDG_ERR_CUDA;
    else if (major != 10)
      state[dev] = CDG_ERR_NO_SM100;
    else
      state[dev] = allow_smem_of<__nv_bfloat16>() && allow_smem_of<__half>() ? CDG_OK : CDG_ERR_CUDA;
  });
  return state[dev];
}

// A 16-bit matrix as it lies in memory: `rows` rows of `cols` columns.
struct Matrix {
  const void* p;
  int64_t stride, rows, cols;
};

int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

// Rows that TMA can load: on 16-byte boundaries and apart (a broadcast row has stride 0).
bool tma_rows(const Matrix& m) {
  return m.rows == 0 || (reinterpret_cast<uintptr_t>(m.p) % 16 == 0 &&
                         (m.rows == 1 || (m.stride % 8 == 0 && m.stride >= m.cols)));
}

size_t repack_bytes(const Matrix& m) {
  return tma_rows(m) ? 0 : (static_cast<size_t>(m.rows) * padded(m.cols) * 2 + 255) / 256 * 256;
}

// Replaces the operands that TMA cannot load (b may be NULL) by copies in the workspace.
int repack(Matrix* a, Matrix* b, uint8_t*& ws, cudaStream_t st) {
  Repack todo[2];
  int n = 0;
  int64_t most = 0;
  for (Matrix* m : {a, b}) {
    if (!m || tma_rows(*m)) continue;
    const int64_t stride = padded(m->cols);
    const int64_t parts = (stride + 255) / 256;
    todo[n++] = Repack{static_cast<const uint16_t*>(m->p), m->stride, m->rows, m->cols, reinterpret_cast<uint16_t*>(ws), stride, parts};
    most = std::max(most, m->rows * parts);
    const size_t bytes = repack_bytes(*m);
    m->p = ws;
    m->stride = stride;
    ws += bytes;
  }
  if (n == 0 || most == 0) return CDG_OK;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((most + 7) / 8, int64_t(sm_count()) * 16)), n);
  return launch(repack_rows_kernel, grid, 256, 0, st, todo[0], n == 2 ? todo[1] : todo[0]);
}

// Boxes of 128 bytes x box_rows in the 128-byte swizzle.
int make_map(CUtensorMap* map, const Matrix& m, int dtype, uint32_t box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return CDG_ERR_CUDA;
  const int64_t e = element_size(dtype);
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(m.cols), static_cast<cuuint64_t>(m.rows)};
  // one row may have any stride; the map wants a multiple of 16 bytes all the same
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(m.rows > 1 ? m.stride : padded(m.cols)) * e};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / e), box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = dtype == CDG_DTYPE_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : dtype == CDG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return enc(map, type, 2, const_cast<void*>(m.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? CDG_OK
             : CDG_ERR_CUDA;
}

template <typename T, typename O, int BN, bool SWAP>
int launch_tiles(const CUtensorMap& ta, const CUtensorMap& tb, LinearShape s, const Epilogue& e, int splits,
                 cudaStream_t st) {
  constexpr bool PROMOTE = sizeof(O) == 4;
  using L = TileSmem<BN, PROMOTE>;
  const int64_t ctas = int64_t(s.m_tiles) * s.n_tiles * splits;
  s.stages = ctas <= sm_count() ? L::kStagesAlone : L::kStages;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreadsOf<SWAP>);
  cfg.dynamicSmemBytes = L::bytes(s.stages);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch()
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = cdg_get_pdl() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, cdg_linear_tile_kernel<T, O, BN, PROMOTE, SWAP>, ta, tb, s, e, splits) == cudaSuccess
             ? CDG_OK
             : CDG_ERR_CUDA;
}

template <typename T, typename O, int BN>
int launch_pairs(const Matrix& A, const Matrix& B, const LinearShape& s, Epilogue e, int64_t M, int64_t N,
                 cudaStream_t st) {
  constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? CDG_DTYPE_BF16 : CDG_DTYPE_F16;
  constexpr int kOut = sizeof(O) == 4 ? CDG_DTYPE_F32 : kType;
  CUtensorMap ta{}, tb{}, ty{}, tr{};
  int rc = make_map(&ta, A, kType, s.a_mn ? 64 : 128);
  if (rc == CDG_OK) rc = make_map(&tb, B, kType, s.b_mn ? 64 : BN / 2);
  // a box of y or of the residual is one warp's 32 rows x 128 bytes
  const Matrix y{e.y, e.y_stride, M, N}, r{e.residual, e.residual_stride, M, N};
  const bool apart = M == 1 || (y.stride >= N && (!e.residual || r.stride >= N));
  // TMA stores whole pieces of 16 bytes: where a row ends inside one, the rest of it is not this row's to write
  const bool whole = N * static_cast<int64_t>(sizeof(O)) % 16 == 0;
  // (FP32 results have four chunks a warp and tile, and no staged residual)
  e.staged = e.z || (e.residual && (sizeof(O) == 4 || e.residual_f32)) ? 0 : e.wide && apart && whole ? 1 : 2;
  if (rc == CDG_OK && e.staged == 1) rc = make_map(&ty, y, kOut, 32);
  if (rc == CDG_OK && e.staged == 1 && e.residual) rc = make_map(&tr, r, kOut, 32);
  if (rc != CDG_OK) return rc;
  // The plan is made for the whole GPU, so that a limit on the SMs does not change the result's bits.
  const unsigned grid =
      static_cast<unsigned>(2 * std::min<int64_t>(int64_t(s.m_tiles) * s.n_tiles, std::max(1, usable_sms() / 2)));
  return launch(cdg_linear_pair_kernel<T, O, BN>, dim3(grid), PairTileSmem<BN>::kThreads, PairTileSmem<BN>::kBytes, st, ta, tb,
                ty, tr, s, e);
}

// How a product is cut: pairs (256 x 256 tiles), tiles (128 x 64 or 128 x 128, K split or not), or
// swapped tiles (up to 32 rows of x).  The costs are microseconds, fitted to the GPU times of 24
// shapes under every cut, from 64 x 512 x 512 to 16,384 x 64 x 1024 (one B200, calls in a row).  What they
// decide, for instance: 128 x 4096 x 4096 pairs 26.2, 128 x 64 in 2 parts 14.0 us; 1024 x 2048 x 2048 pairs
// 16.8, 128 x 128 13.7, 128 x 64 15.2 us; 300 x 8192 x 512 pairs 9.9, 128 x 64 12.9 us; 3000 x 3000 x 256
// pairs 12.0, 128 x 128 16.9 us; 2910 x 94 x 192 128 x 64 7.8, pairs 8.3, 128 x 128 11.8 us.
struct Plan {
  enum Kind { kPairs, kTiles, kSwapped } kind;
  int bn, splits;
};

// Whether K may go to clusters of `parts` CTAs: two CTAs per SM, but clusters of eight, which few SMs
// can hold at the same time, on half the SMs only (1 x 256 x 4096 in 4 parts 7.2, in 8 5.2 us;
// 8 x 2048 x 8192 in 4 parts 12.0, in 8, 128 CTAs, 16.8 us).
bool may_split(int64_t ctas, int parts, int sms) {
  return parts <= 4 ? ctas <= 2 * sms : parts == 8 && ctas <= sms / 2;
}

Plan make_plan(int64_t M, int64_t N, int64_t k_steps, bool narrow, int sms) {
  if (M <= 32) {
    Plan p{Plan::kSwapped, M <= 16 ? 16 : 32, 1};
    const int64_t tiles = (N + 127) / 128;
    while (may_split(tiles * p.splits * 2, p.splits * 2, sms) && k_steps / (p.splits * 2) >= 4) p.splits *= 2;
    return p;
  }
  Plan best{Plan::kTiles, 64, 1};
  double least = 1e300;
  for (int bn : {64, 128}) {
    for (int s = 1; s <= 8; s *= 2) {
      const int64_t ctas = (M + 127) / 128 * ((N + bn - 1) / bn) * s;
      if (s > 1 && (!may_split(ctas, s, sms) || k_steps / s < 2)) break;
      const double steps = static_cast<double>((k_steps + s - 1) / s);
      const double waves = static_cast<double>((ctas + 2 * sms - 1) / (2 * sms));
      double cost;
      if (ctas <= sms)  // a CTA has its SM alone
        cost = bn == 64 ? 4.0 + 0.235 * steps : 4.9 + 0.245 * steps;
      else
        cost = 1.0 + waves * (bn == 64 ? 4.7 + 0.3 * steps : 6.5 + 0.41 * steps);
      if (s > 1) cost += (bn == 64 ? 0.8 : 2.5) + 0.2 * s + (ctas > sms ? 1.0 : 0.0);
      if (narrow) cost += waves * (bn == 64 ? 3.0 : 6.0);
      if (cost < least) {
        least = cost;
        best = Plan{Plan::kTiles, bn, s};
      }
    }
  }
  const int64_t pairs = std::max(1, sms / 2), pair_tiles = (M + 255) / 256 * ((N + 255) / 256);
  const double waves = static_cast<double>((pair_tiles + pairs - 1) / pairs);
  if (k_steps > 0 && 4.0 + waves * (2.6 + 0.293 * static_cast<double>(k_steps) + (narrow ? 3.0 : 0.0)) < least)
    best.kind = Plan::kPairs;
  return best;
}

// D [M, N] = epilogue(sum over K of A and B); a_mn: A lies as [K, M], else [M, K]; b_mn: B lies as
// [K, N], else [N, K].  Rows of both on 16-byte boundaries.
template <typename T, typename O>
int product(const Matrix& A, bool a_mn, const Matrix& B, bool b_mn, int64_t M, int64_t N, int64_t K,
            const Epilogue& e, cudaStream_t st) {
  constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? CDG_DTYPE_BF16 : CDG_DTYPE_F16;
  if (M == 0 || N == 0) return CDG_OK;
  LinearShape s{};
  s.M = M;
  s.N = N;
  s.k_steps = static_cast<int>((K + 63) / 64);
  s.a_mn = a_mn;
  s.b_mn = b_mn;
  s.bf16 = kType == CDG_DTYPE_BF16;
  s.a_rows = static_cast<int>(std::min<int64_t>(128, (M + 7) / 8 * 8));
  Plan p = make_plan(M, N, s.k_steps, !e.wide, sm_count());
  if (p.kind == Plan::kSwapped && a_mn) {  // x's place is loaded in boxes of 16 to 64 rows, K-major
    p.kind = Plan::kTiles;
    p.bn = 64;
  }
  const int64_t tm = p.kind == Plan::kPairs ? 256 : 128, tn = p.kind == Plan::kPairs ? 256 : p.bn;
  const int64_t rows = p.kind == Plan::kSwapped ? N : M, cols = p.kind == Plan::kSwapped ? M : N;
  const int64_t m_tiles = (rows + tm - 1) / tm, n_tiles = (cols + tn - 1) / tn;
  if (m_tiles * n_tiles * 8 > 0x7fffffff) return CDG_ERR_UNSUPPORTED;
  s.m_tiles = static_cast<int>(m_tiles);
  s.n_tiles = static_cast<int>(n_tiles);
  if (p.kind == Plan::kPairs) return launch_pairs<T, O, 256>(A, B, s, e, M, N, st);
  CUtensorMap ta{}, tb{};
  if (p.kind == Plan::kSwapped) {
    std::swap(s.M, s.N);
    s.a_mn = b_mn;
    s.b_mn = 0;
    s.a_rows = static_cast<int>(std::min<int64_t>(128, (s.M + 7) / 8 * 8));
    if (K > 0) {
      int rc = make_map(&ta, B, kType, b_mn ? 64 : s.a_rows);
      if (rc == CDG_OK) rc = make_map(&tb, A, kType, p.bn);
      if (rc != CDG_OK) return rc;
    }
    return p.bn == 16 ? launch_tiles<T, O, 16, true>(ta, tb, s, e, p.splits, st)
                      : launch_tiles<T, O, 32, true>(ta, tb, s, e, p.splits, st);
  }
  if (K > 0) {
    int rc = make_map(&ta, A, kType, a_mn ? 64 : s.a_rows);
    if (rc == CDG_OK) rc = make_map(&tb, B, kType, b_mn ? 64 : p.bn);
    if (rc != CDG_OK) return rc;
  }
  return p.bn == 128 ? launch_tiles<T, O, 128, false>(ta, tb, s, e, p.splits, st)
                     : launch_tiles<T, O, 64, false>(ta, tb, s, e, p.splits, st);
}

bool operand_dtype(int dtype) { return dtype == CDG_DTYPE_BF16 || dtype == CDG_DTYPE_F16; }

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M <= (int64_t(1) << 30) && N <= (int64_t(1) << 30) && K <= (int64_t(1) << 30);
}

// 16-byte rows of an output or residual that the epilogue reads and writes eight columns at a time.
bool wide_columns(const void* p, int64_t stride, int64_t bytes) { return wide_rows(p, stride, bytes); }

template <typename T>
int forward(const cdg_linear_args* g, uint8_t* ws, cudaStream_t st) {
  Matrix x{g->x, g->x_stride, g->M, g->K}, w{g->w, g->w_stride, g->N, g->K};
  int rc = CDG_OK;
  if (g->K > 0) {
    rc = repack(&x, &w, ws, st);
    if (rc != CDG_OK) return rc;
  }
  Epilogue e{};
  e.bias = g->bias;
  e.bias_f32 = g->bias_dtype == CDG_DTYPE_F32;
  e.residual = g->residual;
  e.residual_stride = g->residual_stride;
  e.residual_f32 = g->residual_dtype == CDG_DTYPE_F32;
  e.act = g->activation;
  e.y = g->y;
  e.y_stride = g->y_stride;
  e.z = g->z_out;
  e.z_stride = g->z_stride;
  e.wide_bias = e.bias && !e.bias_f32 && reinterpret_cast<uintptr_t>(e.bias) % 16 == 0;
  e.wide = wide_columns(e.y, e.y_stride, element_size(g->out_dtype)) && wide_columns(e.z, e.z_stride, 2) &&
           wide_columns(e.residual, e.residual_stride, e.residual_f32 ? 4 : 2);
  return g->out_dtype == CDG_DTYPE_F32 ? product<T, float>(x, false, w, false, g->M, g->N, g->K, e, st)
                                       : product<T, T>(x, false, w, false, g->M, g->N, g->K, e, st);
}

// Row groups of the elementwise backward pass: a few CTAs per SM, each summing many rows.
int dz_groups(int64_t M, int64_t N) {
  const int64_t chunks = std::max<int64_t>(1, (N + 255) / 256);
  const int64_t want = std::max<int64_t>(1, int64_t(sm_count()) * 4 / chunks);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, (M + 7) / 8, 1024})));
}

bool needs_dz(const cdg_linear_backward_args* g) {
  if (g->M == 0 || g->N == 0) return false;  // no elements (and torch gives [M, 0] a row stride of 1)
  return g->activation != CDG_ACT_NONE || !tma_rows(Matrix{g->dy, g->dy_stride, g->M, g->N});
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

template <typename T>
int backward(const cdg_linear_backward_args* g, uint8_t* ws, cudaStream_t st) {
  Matrix x{g->x, g->x_stride, g->M, g->K}, w{g->w, g->w_stride, g->N, g->K};
  Matrix dz{g->dy, g->dy_stride, g->M, g->N};
  const bool store = needs_dz(g) && (g->dx || g->dw);
  if ((store || g->db) && g->M > 0 && g->N > 0) {
    T* out = nullptr;
    const int64_t stride = padded(g->N);
    if (store) {
      out = reinterpret_cast<T*>(ws);
      ws += align256(static_cast<size_t>(g->M) * stride * 2);
    }
    const int groups = dz_groups(g->M, g->N);
    float* partial = nullptr;
    if (g->db) {
      partial = reinterpret_cast<float*>(ws);
      ws += align256(static_cast<size_t>(groups) * g->N * 4);
    }
    const T* z = g->activation != CDG_ACT_NONE ? static_cast<const T*>(g->z) : nullptr;
    const bool wide = g->N % 8 == 0 && wide_rows(g->dy, g->dy_stride, 2) && (!z || wide_rows(z, g->z_stride, 2));
    const dim3 grid(static_cast<unsigned>((g->N + 255) / 256), static_cast<unsigned>(groups));
    int rc = launch(wide ? linear_dz_kernel<T, true> : linear_dz_kernel<T, false>, grid, 256, 0, st, static_cast<const T*>(g->dy),
                    g->dy_stride, z, g->z_stride, g->activation, g->M, g->N, out, stride, partial);
    if (rc != CDG_OK) return rc;
    if (g->db) {
      const unsigned blocks = static_cast<unsigned>((g->N + 31) / 32);
      rc = g->db_dtype == CDG_DTYPE_F32
               ? launch(column_sum_kernel<float>, dim3(blocks), 1024, 0, st, partial, groups, g->N, static_cast<float*>(g->db))
               : launch(column_sum_kernel<T>, dim3(blocks), 1024, 0, st, partial, groups, g->N, static_cast<T*>(g->db));
      if (rc != CDG_OK) return rc;
    }
    if (store) {
      dz.p = out;
      dz.stride = stride;
    }
  } else if (g->db && g->N > 0) {
    if (cudaMemsetAsync(g->db, 0, g->N * element_size(g->db_dtype), st) != cudaSuccess) return CDG_ERR_CUDA;
  }
  if (g->dx) {
    int rc = g->N > 0 && g->M > 0 ? repack(&w, nullptr, ws, st) : CDG_OK;
    Epilogue e{};
    e.y = g->dx;
    e.y_stride = g->dx_stride;
    e.wide = wide_columns(e.y, e.y_stride, 2);
    if (rc == CDG_OK) rc = product<T, T>(dz, false, w, true, g->M, g->K, g->N, e, st);
    if (rc != CDG_OK) return rc;
  }
  if (g->dw) {
    int rc = g->M > 0 ? repack(&x, nullptr, ws, st) : CDG_OK;
    Epilogue e{};
    e.y = g->dw;
    e.y_stride = g->dw_stride;
    e.wide = wide_columns(e.y, e.y_stride, 2);
    if (rc == CDG_OK) rc = product<T, T>(dz, true, x, true, g->N, g->K, g->M, e, st);
    if (rc != CDG_OK) return rc;
  }
  return CDG_OK;
}

int check_forward(const cdg_linear_args* g) {
  if (!g || g->M < 0 || g->N < 0 || g->K < 0 || !operand_dtype(g->dtype)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->out_dtype != g->dtype && g->out_dtype != CDG_DTYPE_F32) return CDG_ERR_INVALID_ARGUMENT;
  if (g->activation < CDG_ACT_NONE || g->activation > CDG_ACT_GELU_TANH) return CDG_ERR_INVALID_ARGUMENT;
  if (g->bias && g->bias_dtype != g->dtype && g->bias_dtype != CDG_DTYPE_F32) return CDG_ERR_INVALID_ARGUMENT;
  if (g->residual && g->residual_dtype != g->dtype && g->residual_dtype != CDG_DTYPE_F32)
    return CDG_ERR_INVALID_ARGUMENT;
  if (g->M > 0 && g->N > 0 && (!g->y || (g->K > 0 && (!g->x || !g->w)))) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(2, {g->x, g->w, g->z_out}) || !on_boundary(element_size(g->out_dtype), {g->y}) ||
      (g->bias && !on_boundary(element_size(g->bias_dtype), {g->bias})) ||
      (g->residual && !on_boundary(element_size(g->residual_dtype), {g->residual})))
    return CDG_ERR_ALIGNMENT;
  return sizes_ok(g->M, g->N, g->K) ? CDG_OK : CDG_ERR_UNSUPPORTED;
}

int check_backward(const cdg_linear_backward_args* g) {
  if (!g || g->M < 0 || g->N < 0 || g->K < 0 || !operand_dtype(g->dtype)) return CDG_ERR_INVALID_ARGUMENT;
  if (g->activation < CDG_ACT_NONE || g->activation > CDG_ACT_GELU_TANH) return CDG_ERR_INVALID_ARGUMENT;
  if (g->db && g->db_dtype != g->dtype && g->db_dtype != CDG_DTYPE_F32) return CDG_ERR_INVALID_ARGUMENT;
  if (g->M > 0 && g->N > 0 && (!g->dy || (g->activation != CDG_ACT_NONE && !g->z))) return CDG_ERR_INVALID_ARGUMENT;
  if (g->dx && g->N > 0 && g->K > 0 && g->M > 0 && !g->w) return CDG_ERR_INVALID_ARGUMENT;
  if (g->dw && g->M > 0 && g->K > 0 && g->N > 0 && !g->x) return CDG_ERR_INVALID_ARGUMENT;
  if (!on_boundary(2, {g->dy, g->x, g->w, g->z, g->dx, g->dw}) || (g->db && !on_boundary(element_size(g->db_dtype), {g->db})))
    return CDG_ERR_ALIGNMENT;
  return sizes_ok(g->M, g->N, g->K) ? CDG_OK : CDG_ERR_UNSUPPORTED;
}

}  // namespace

// This unit's record of waits that gave up (cdg_device_status reads it with the others').
int linear_sticky_status(int clear, int32_t* out) { return read_sticky(g_sticky_status, clear, out); }

}  // namespace cdg

extern "C" {

size_t cdg_linear_workspace_bytes(const cdg_linear_args* g) {
  using namespace cdg;
  if (check_forward(g) != CDG_OK) return 0;
  return repack_bytes(Matrix{g->x, g->x_stride, g->M, g->K}) + repack_bytes(Matrix{g->w, g->w_stride, g->N, g->K});
}

int cdg_linear(const cdg_linear_args* g, void* workspace, size_t workspace_bytes, cdg_stream_t stream) {
  using namespace cdg;
  int rc = check_forward(g);
  if (rc != CDG_OK) return rc;
  if (g->M == 0 || g->N == 0) return CDG_OK;
  const size_t need = cdg_linear_workspace_bytes(g);
  if (need && (!workspace || workspace_bytes < need)) return CDG_ERR_WORKSPACE;
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16) return CDG_ERR_ALIGNMENT;
  rc = device_ready();
  if (rc != CDG_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return g->dtype == CDG_DTYPE_BF16 ? forward<__nv_bfloat16>(g, ws, st) : forward<__half>(g, ws, st);
}

size_t cdg_linear_backward_workspace_bytes(const cdg_linear_backward_args* g) {
  using namespace cdg;
  if (check_backward(g) != CDG_OK) return 0;
  size_t n = 0;
  if (needs_dz(g) && (g->dx || g->dw)) n += align256(static_cast<size_t>(g->M) * padded(g->N) * 2);
  if (g->M > 0 && g->N > 0 && g->db) n += align256(static_cast<size_t>(dz_groups(g->M, g->N)) * g->N * 4);
  if (g->dx) n += repack_bytes(Matrix{g->w, g->w_stride, g->N, g->K});
  if (g->dw) n += repack_bytes(Matrix{g->x, g->x_stride, g->M, g->K});
  return n;
}

int cdg_linear_backward(const cdg_linear_backward_args* g, void* workspace, size_t workspace_bytes,
                        cdg_stream_t stream) {
  using namespace cdg;
  int rc = check_backward(g);
  if (rc != CDG_OK) return rc;
  const size_t need = cdg_linear_backward_workspace_bytes(g);
  if (need && (!workspace || workspace_bytes < need)) return CDG_ERR_WORKSPACE;
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16) return CDG_ERR_ALIGNMENT;
  rc = device_ready();
  if (rc != CDG_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return g->dtype == CDG_DTYPE_BF16 ? backward<__nv_bfloat16>(g, ws, st) : backward<__half>(g, ws, st);
}

}  // extern "C"
