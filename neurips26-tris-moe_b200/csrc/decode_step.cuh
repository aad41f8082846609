// What the kernels of the decode step around the experts share (paged_kv.cu, paged_attention.cu, rms_norm.cu, logit_controls.cu):
// element types, conversions and stores of eight values, quotients by a scale.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"

namespace tris {

constexpr float kE4m3Max = 448.f;

template <typename T>
struct Pair;  // two elements of a 16-bit type in one register
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ void store_float(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_float(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_float(__nv_fp8_e4m3* p, float v) { p->__x = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// Eight elements that have been read, and stored by one access of 16 bytes (8 of e4m3).
template <typename T>
__device__ __forceinline__ void unpack_8(const uint4& raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Pair<T>::unpack(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void store_8(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]), Pair<T>::pack(v[4], v[5]), Pair<T>::pack(v[6], v[7]));
}
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ void store_8(__nv_fp8_e4m3* p, const float (&v)[8]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(e4m3_pack4(v[0], v[1], v[2], v[3]), e4m3_pack4(v[4], v[5], v[6], v[7]));
}

// 1 / v to a rounding.
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Two products, and sums with them, by one instruction.
__device__ __forceinline__ uint64_t pack_2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
// x / s of many x by one s, rounded to 32 bits as a division rounds it (but for quotients within some 2^-46 of half way between two numbers, none
// of which is one): the reciprocal in two parts, one instruction an element where a division takes some ten.  Scales for which the parts are not exact are
// brought by 2^64 into the range where they are, together with x; infinite numbers have no sum of two products.
// (Prompts of 8188 tokens, 48 heads of 128, to e4m3: 32.2 us, 41.3 with divisions; 31.6 by the reciprocal alone, which is one step of e4m3 off
// where it falls on the other side of half way.)
struct DivideBy {
  float hi, lo, lift;
  template <int N>
  static __device__ __forceinline__ void by_parts(float (&x)[N], float hi, float lo) {
    const uint64_t his = pack_2(hi, hi), los = pack_2(lo, lo);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t v = pack_2(x[i], x[i + 1]), q = fma_2(v, his, mul_2(v, los));
      asm("mov.b64 {%0, %1}, %2;" : "=f"(x[i]), "=f"(x[i + 1]) : "l"(q));
    }
  }
  static __device__ __forceinline__ float second_part(float hi, float s) { return fmaf(-hi, s, 1.f) * hi; }
  __device__ __forceinline__ explicit DivideBy(float s) {
    lift = fabsf(s) < 0x1p-80f ? 0x1p64f : fabsf(s) > 0x1p80f ? 0x1p-64f : 1.f;
    s *= lift;
    hi = reciprocal(s);
    lo = second_part(hi, s);
  }
  template <int N>
  __device__ __forceinline__ void operator()(float (&x)[N], float top) const {  // top: the largest magnitude, or more
    if (lift == 1.f && top < INFINITY) {
      by_parts(x, hi, lo);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = x[i] * lift, q = v * hi;
        x[i] = fabsf(q) < INFINITY && lo == lo ? fmaf(v, hi, v * lo) : q;  // of a scale of 0 or without end, lo is none
      }
    }
  }
};

// launch_kernel, by the plain launch where nothing else is asked for: 0.6 us less of the host's time (2.8 against 3.4).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_step(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl, int cluster_z, Args&&... args) {
  if (pdl || cluster_z > 1) return launch_kernel(kernel, grid, block, smem, stream, pdl, cluster_z, static_cast<Args&&>(args)...);
  return [&](KArgs... held) {
    void* params[] = {&held...};
    return cudaLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, params, smem, stream);
  }(static_cast<KArgs>(args)...);
}
// Lets a kernel use that much dynamic shared memory; asked of the driver once a device (0.5 us a call).
template <auto KERNEL>
inline int allow_shared_memory(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  TRIS_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return TRIS_OK;
  TRIS_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return TRIS_OK;
}
// SMs of the current device, 0 where there is none; asked of the driver once a device.
inline int sm_count() {
  static std::atomic<int> count[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = count[dev].load(std::memory_order_relaxed);
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) count[dev].store(n, std::memory_order_relaxed);
  return n;
}
inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline int dtype_size(int dtype) { return dtype == TRIS_DTYPE_F32 ? 4 : dtype == TRIS_DTYPE_E4M3 ? 1 : 2; }
int validate_paged_kv(const TrisPagedKv* cache, const char* what);  // paged_kv.cu

}  // namespace tris
