// Rows of BF16, FP16 or FP32 values as the row-wise kernels read and write them, and the host
// helpers those kernels' launchers share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "cdg_b200.h"
#include "cdg_ptx.cuh"

namespace cdg {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// A warp takes 256 columns at a time, eight per lane.  Wide (rows on 16-byte boundaries, H a
// multiple of 8): lane l holds columns 8l .. 8l+7, one 128-column scale block per half warp.
// Narrow (anything else): lane l holds columns l, l + 32, ..., so that each load of the warp
// stays contiguous; the first four are in the first scale block, the others in the second.
template <bool WIDE>
__device__ __forceinline__ int64_t column(int64_t chunk, int lane, int j) {
  return chunk * 256 + (WIDE ? lane * 8 + j : j * 32 + lane);
}

// The lane's eight elements of a chunk as they lie in memory.
template <typename T>
struct alignas(16) Raw {
  static constexpr int kWords = static_cast<int>(sizeof(T)) * 2;
  uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ void unpack8(const Raw<T>& raw, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2(raw.w[j], T());
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ Raw<T> load8(const T* row, int64_t chunk, int lane, int64_t H) {
  Raw<T> raw;
#pragma unroll
  for (int j = 0; j < Raw<T>::kWords; ++j) raw.w[j] = 0;
  if constexpr (WIDE) {
    const int64_t c = column<true>(chunk, lane, 0);
    if (c < H) {
      const uint4* p = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
      for (int k = 0; k < Raw<T>::kWords / 4; ++k) {
        const uint4 t = p[k];
        raw.w[4 * k] = t.x; raw.w[4 * k + 1] = t.y; raw.w[4 * k + 2] = t.z; raw.w[4 * k + 3] = t.w;
      }
    }
  } else {
    // a chunk that lies in the row needs no test per column
    const T* from = row + column<false>(chunk, lane, 0);
    const int left = static_cast<int>(H - chunk * 256 < 256 ? H - chunk * 256 : 256);
    if (left == 256) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4)
          raw.w[j] = reinterpret_cast<const uint32_t*>(from)[j * 32];
        else
          raw.w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[j * 32]) << (16 * (j & 1));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j * 32 + lane < left) {
          if constexpr (sizeof(T) == 4)
            raw.w[j] = reinterpret_cast<const uint32_t*>(from)[j * 32];
          else
            raw.w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[j * 32]) << (16 * (j & 1));
        }
      }
    }
  }
  return raw;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store8(T* row, int64_t chunk, int lane, int64_t H, const float (&v)[8]) {
  if constexpr (WIDE) {
    const int64_t c = column<true>(chunk, lane, 0);
    if (c >= H) return;
    uint4* p = reinterpret_cast<uint4*>(row + c);
    if constexpr (sizeof(T) == 4) {
      p[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      p[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
      p[0] = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
  } else {
    T* to = row + column<false>(chunk, lane, 0);
    const int left = static_cast<int>(H - chunk * 256 < 256 ? H - chunk * 256 : 256);
    if (left == 256) {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j * 32] = from_f<T>(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j * 32 + lane < left) to[j * 32] = from_f<T>(v[j]);
    }
  }
}

// out[c] = the sum of `parts` rows of partial column sums, every 32nd row per thread and then over
// the 32 threads of a column: the same order every time.  1024 threads.
template <typename W>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partial, int parts, int64_t H, W* out) {
  __shared__ float sums[32][33];
  grid_dependency_wait();  // the partial sums are the previous kernel's
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float v = 0.0f;
  if (c < H) {
#pragma unroll 8
    for (int p = g; p < parts; p += 32) v += partial[static_cast<int64_t>(p) * H + c];
  }
  sums[g][lane] = v;
  __syncthreads();
  // warp g sums column g of the block
  v = sums[lane][g];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t out_c = static_cast<int64_t>(blockIdx.x) * 32 + g;
  if (lane == 0 && out_c < H) out[out_c] = from_f<W>(v);
}

// ------------------------------------------------------------------ host
// Launch with programmatic stream serialization (unless cdg_set_pdl(0)): the kernel may be scheduled
// while its predecessor on the stream, of this call or of another, drains; it waits for the
// predecessor's end (griddepcontrol.wait) before it touches global memory.  Calls of a few
// microseconds in a row lose about one less between them.  cluster: CTAs of a cluster, 0 as the
// kernel says.
template <typename... K, typename... A>
inline int launch_clusters(void (*kernel)(K...), dim3 grid, unsigned cluster, unsigned block, size_t smem, cudaStream_t st,
                           A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  unsigned n = 0;
  if (cluster > 0) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = 1;
  }
  if (cdg_get_pdl()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...) == cudaSuccess ? CDG_OK : CDG_ERR_CUDA;
}
template <typename... K, typename... A>
inline int launch(void (*kernel)(K...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, A&&... args) {
  return launch_clusters(kernel, grid, 0, block, smem, st, static_cast<A&&>(args)...);
}

// SM count of the current device (looked up at each call: a cheap attribute query).
inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n > 0 ? n : 148;
}

// SMs a persistent GEMM kernel may use (cdg_set_num_sms; read at every launch).
inline int usable_sms() {
  const int limit = cdg_get_num_sms(), all = sm_count();
  return limit > 0 && limit < all ? limit : all;
}

constexpr int kMaxDevices = 64;

// Reads a unit's device-side error record (two words) into `out`, and clears it if asked.
inline int read_sticky(const int (&record)[2], int clear, int32_t* out) {
  if (cudaMemcpyFromSymbol(out, record, 2 * sizeof(int32_t)) != cudaSuccess) return CDG_ERR_CUDA;
  if (clear && (out[0] || out[1])) {
    const int32_t z[2] = {0, 0};
    if (cudaMemcpyToSymbol(record, z, sizeof(z)) != cudaSuccess) return CDG_ERR_CUDA;
  }
  return CDG_OK;
}

inline int element_size(int dtype) { return dtype == CDG_DTYPE_F32 ? 4 : 2; }

inline bool row_dtype(int dtype) {
  return dtype == CDG_DTYPE_BF16 || dtype == CDG_DTYPE_F16 || dtype == CDG_DTYPE_F32;
}

// Whether each pointer lies on a boundary of its type's `bytes` (absent ones do): what a kernel's loads and
// stores of single elements need.
inline bool on_boundary(int64_t bytes, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  return true;
}

// Whether every row of a tensor starts on a 16-byte boundary (absent tensors do).
inline bool wide_rows(const void* p, int64_t stride, int64_t bytes) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0);
}

}  // namespace
}  // namespace cdg
