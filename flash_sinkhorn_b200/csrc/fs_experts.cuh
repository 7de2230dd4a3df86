// What the kernels of routed experts share (fs_experts.cu: routing, gated activation, sums back into tokens;
// fs_group.cu: matrix products grouped by expert): loads and stores of 16- and 32-bit values, checks of the host side.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "../../include/flash_sinkhorn_b200.h"

namespace fs {
int report_error(int code, const char* msg);  // fs_api.cu: records the calling thread's error text
void count_launches(int k);                   // fs_api.cu: adds to the count behind fs_launch_count()

namespace ex {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values as one load or store of up to 16 bytes each; the pointer is aligned to N values (at most 16 bytes).
// Held as 32-bit words (two 16-bit values each): as an array of values each would take a register.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  static constexpr bool kWords = N * sizeof(T) % 4 == 0;
  static constexpr int kCount = kWords ? (int)(N * sizeof(T) / 4) : N;
  typename std::conditional<kWords, uint32_t, T>::type w[kCount];
};
__device__ __forceinline__ void two_f32(uint32_t w, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void two_f32(uint32_t w, float& lo, float& hi, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ uint32_t from_two(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t from_two(float lo, float hi, __half) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& q, float (&out)[N]) {
  if constexpr (!Pack<T, N>::kWords) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_f32(q.w[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = __uint_as_float(q.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) two_f32(q.w[i], out[2 * i], out[2 * i + 1], T());
  }
}
// From global memory that nothing writes meanwhile: such loads may move ahead of stores to other arrays.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> read_only(const T* p) {
  Pack<T, N> q;
  constexpr int kBytes = N * sizeof(T);
  if constexpr (kBytes % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      q.w[4 * i] = v.x;
      q.w[4 * i + 1] = v.y;
      q.w[4 * i + 2] = v.z;
      q.w[4 * i + 3] = v.w;
    }
  } else if constexpr (kBytes == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    q.w[0] = v.x;
    q.w[1] = v.y;
  } else if constexpr (kBytes == 4) {
    q.w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else {
    const unsigned short v = __ldg(reinterpret_cast<const unsigned short*>(p));
    memcpy(&q.w[0], &v, 2);
  }
  return q;
}
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[N]) {
  unpack<T, N>(*reinterpret_cast<const Pack<T, N>*>(p), out);
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[N]) {
  Pack<T, N> q;
  if constexpr (!Pack<T, N>::kWords) {
#pragma unroll
    for (int i = 0; i < N; ++i) q.w[i] = from_f32<T>(in[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) q.w[i] = __float_as_uint(in[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) q.w[i] = from_two(in[2 * i], in[2 * i + 1], T());
  }
  *reinterpret_cast<Pack<T, N>*>(p) = q;
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline int type_bytes(int type) { return type == FS_TYPE_F32 ? 4 : 2; }

inline int check_device() {
  static std::atomic<uint64_t> fits{0};  // devices that have been looked at
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return report_error(FS_ERR_CUDA, "cannot query the current CUDA device");
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (fits.load(std::memory_order_relaxed) & bit) return FS_OK;
  const int arch = fs_device_arch();
  if (arch < 0) return report_error(FS_ERR_CUDA, "cannot query the current CUDA device");
  if (arch / 10 != 10) return report_error(FS_ERR_UNSUPPORTED, "this library is built for sm_100a only");
  fits.fetch_or(bit, std::memory_order_relaxed);
  return FS_OK;
}
inline int launched(int kernels) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  count_launches(kernels);
  return FS_OK;
}

}  // namespace
}  // namespace ex
}  // namespace fs
