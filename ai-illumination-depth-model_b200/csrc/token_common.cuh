// Loads, stores and reductions shared by the token operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace illumina {
namespace gpu {
namespace tok {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float &d, float v) { d = v; }
__device__ __forceinline__ void from_f32(bf16 &d, float v) { d = __float2bfloat16_rn(v); }

// VW consecutive elements as floats: one load when VW fills 8 or 16 bytes
// (the caller guarantees the alignment).
template <typename T, int VW>
struct Pack {
  static_assert(VW == 1 || VW * sizeof(T) == 16 || VW * sizeof(T) == 8, "16- or 8-byte vectors, or scalars");
  static __device__ __forceinline__ void load(const T *p, float (&o)[VW]) {
    if constexpr (VW == 1) {
      o[0] = to_f32(*p);
    } else if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p);
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
      uint32_t w[VW / 2];
      if constexpr (VW == 8)
        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p);
      else
        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
      for (int i = 0; i < VW / 2; i++) {
        o[2 * i] = __uint_as_float(w[i] << 16);
        o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ void store(T *p, const float (&o)[VW]) {
    if constexpr (VW == 1) {
      from_f32(*p, o[0]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4 *>(p) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
      uint32_t w[VW / 2];
#pragma unroll
      for (int i = 0; i < VW / 2; i++) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
      }
      if constexpr (VW == 8)
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(w);
      else
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(w);
    }
  }
};

// VW consecutive elements as they lie in memory, and their values.
template <typename T, int VW>
struct RawPack;
template <>
struct RawPack<float, 4> {
  typedef float4 type;
  static __device__ __forceinline__ void unpack(float4 v, float (&o)[4]) { o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w; }
};
template <>
struct RawPack<bf16, 4> {
  typedef uint2 type;
  static __device__ __forceinline__ void unpack(uint2 v, float (&o)[4]) {
    o[0] = __uint_as_float(v.x << 16), o[1] = __uint_as_float(v.x & 0xffff0000u);
    o[2] = __uint_as_float(v.y << 16), o[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <typename T>
struct RawPack<T, 1> {
  typedef T type;
  static __device__ __forceinline__ void unpack(T v, float (&o)[1]) { o[0] = to_f32(v); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Lets kernel K use `bytes` of dynamic shared memory on the current device;
// the runtime is asked once a device.
template <auto K>
cudaError_t allow_smem(size_t bytes) {
  static std::atomic<uint64_t> seen{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && seen.load(std::memory_order_relaxed) >> dev & 1)) return e;
  e = cudaFuncSetAttribute((const void *)K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) seen.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

// A kernel that follows another on its stream and needs its results: it may
// start, and set itself up, while the last CTAs of the one before are at work,
// if that one's CTAs called cudaTriggerProgrammaticLaunchCompletion. At least
// one thread of each of its CTAs calls cudaGridDependencySynchronize, so that
// what follows on the stream finds both finished.
template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), long long grid, int threads, size_t smem, cudaStream_t st, const A &...args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid), c.blockDim = dim3(threads), c.dynamicSmemBytes = smem, c.stream = st;
  c.attrs = &early, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace tok
}  // namespace gpu
}  // namespace illumina
