// Rows and weights to e4m3, with a scale for each 128 columns of a row or for each block of 128 x 128.
//
// s = max |x| / 448 of a group, and x / s, both rounded as divisions round them.  Bound by bytes (2 read and 1 written an element), by latency for a few
// rows.  A quarter-warp has 128 columns of a row; for blocks a CTA has all of one in its registers, so that x is read once.
// Replayed, bf16: rows of 4096, 64 of them 1.8 us, 1024 3.6, 8192 18.5 (101 MB, 5.5 TB/s); blocks of 14336 x 4096 30 to 35 us (176 MB, 5.0 to 5.9 TB/s).
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 128, kLanes = kGroup / 8;  // columns of a scale, and lanes that have them
constexpr int kRowLanes = 8;  // of a group of one row

struct QuantizeArgs {
  TrisQuantizeE4m3 q;
  int groups;        // scales of a row
  int wide;          // whether eight elements can be read, and eight results written, at once
  int64_t units;     // groups of all rows
};

// Eight columns from `column` on, zeros behind the last.
template <typename T>
__device__ __forceinline__ uint4 fetch_8(const QuantizeArgs& a, int64_t row, int column) {
  const T* p = static_cast<const T*>(a.q.x) + row * a.q.x_stride + column;
  if (a.wide && column + 8 <= a.q.columns) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = column + 2 * i < a.q.columns ? *reinterpret_cast<const uint16_t*>(p + 2 * i) : 0;
    const uint32_t hi = column + 2 * i + 1 < a.q.columns ? *reinterpret_cast<const uint16_t*>(p + 2 * i + 1) : 0;
    w[i] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void put_8(const QuantizeArgs& a, int64_t row, int column, const float (&v)[8]) {
  __nv_fp8_e4m3* p = static_cast<__nv_fp8_e4m3*>(a.q.values) + row * a.q.values_stride + column;
  if (a.wide && column + 8 <= a.q.columns) {
    store_8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (column + i < a.q.columns) store_float(p + i, v[i]);
  }
}
// The largest magnitude of eight elements, as a float's bits; a NaN is the largest.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const uint4& raw) {
  uint32_t top = __vmaxu2(__vmaxu2(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu), __vmaxu2(raw.z & 0x7FFF7FFFu, raw.w & 0x7FFF7FFFu));
  top = max(top & 0xFFFFu, top >> 16);
  return __float_as_uint(Pair<T>::unpack(top).x);
}

// A quarter-warp has a group of one row, a lane two vectors of it.  (us for 64 and for 8192 rows of 4096: 16 lanes to a group 1.6 and 24.0, eight 1.8 and 18.5, four 2.2 and 17.3; four
// groups of sixteen lanes each, one after the other, 3.2 and 27.5.)
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ QuantizeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int l = threadIdx.x % kRowLanes;
  const int64_t unit = blockIdx.x * static_cast<int64_t>(kThreads / kRowLanes) + threadIdx.x / kRowLanes, here = min(unit, a.units - 1), row = here / a.groups;
  const int group = static_cast<int>(here - row * a.groups);
  constexpr int kSteps = kLanes / kRowLanes;
  uint4 raw[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) raw[i] = fetch_8<T>(a, row, group * kGroup + 8 * (i * kRowLanes + l));
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) top = max(top, top_of<T>(raw[i]));
#pragma unroll
  for (int d = 1; d < kRowLanes; d <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  if (unit >= a.units) return;
  float scale = 0.f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float v[8];
    unpack_8<T>(raw[i], v);
    scale = quantize_8(v, top);
    put_8(a, row, group * kGroup + 8 * (i * kRowLanes + l), v);
  }
  if (l == 0) a.q.scales[row * a.q.scales_stride + group] = scale;
}

// A CTA has a block of 128 x 128.  (Five CTAs an SM 29.8 us for 14336 x 4096; four 31.8, six 32.5, eight, which leave too few registers, 40.8.)
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) quantize_blocks_kernel(const __grid_constant__ QuantizeArgs a) {
  __shared__ uint32_t tops[kThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kRows = kThreads / kLanes, kSteps = kGroup / kRows;
  const int l = threadIdx.x % kLanes, column = blockIdx.x * kGroup + 8 * l;
  const int64_t row0 = blockIdx.y * static_cast<int64_t>(kGroup) + threadIdx.x / kLanes;
  uint4 raw[kSteps];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row0 + i * kRows < a.q.rows) raw[i] = fetch_8<T>(a, row0 + i * kRows, column);
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) top = max(top, top_of<T>(raw[i]));
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, tops[i]);
  float scale = 0.f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float v[8];
    unpack_8<T>(raw[i], v);
    scale = quantize_8(v, top);
    if (row0 + i * kRows < a.q.rows) put_8(a, row0 + i * kRows, column, v);
  }
  if (threadIdx.x == 0) a.q.scales[blockIdx.y * a.q.scales_stride + blockIdx.x] = scale;
}

template <typename T>
int launch_quantize(const QuantizeArgs& a, cudaStream_t stream) {
  const bool pdl = programmatic_launch_default();
  if (a.q.group_rows > 1) {
    TRIS_CUDA(launch_step(quantize_blocks_kernel<T>, dim3(a.groups, ceil_div(a.q.rows, kGroup)), dim3(kThreads), 0, stream, pdl, 1, a));
    return TRIS_OK;
  }
  constexpr int kPerCta = kThreads / kRowLanes;
  TRIS_CUDA(launch_step(quantize_rows_kernel<T>, dim3(static_cast<unsigned>((a.units + kPerCta - 1) / kPerCta)), dim3(kThreads), 0, stream, pdl, 1, a));
  return TRIS_OK;
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_quantize_e4m3(const TrisQuantizeE4m3* args, void* stream) {
  TRIS_REQUIRE(args, TRIS_ERR_INVALID_ARG, "quantize_e4m3: null arguments");
  const TrisQuantizeE4m3& q = *args;
  TRIS_REQUIRE(q.dtype == TRIS_DTYPE_F16 || q.dtype == TRIS_DTYPE_BF16, TRIS_ERR_INVALID_ARG, "quantize_e4m3: x is fp16 or bf16");
  TRIS_REQUIRE(q.group_rows == 1 || q.group_rows == kGroup, TRIS_ERR_INVALID_ARG, "quantize_e4m3: a scale is for 1 or %d rows, not %d", kGroup, q.group_rows);
  TRIS_REQUIRE(q.rows >= 0 && q.columns >= 0, TRIS_ERR_INVALID_ARG, "quantize_e4m3: negative sizes");
  if (q.rows == 0 || q.columns == 0) return TRIS_OK;
  TRIS_REQUIRE(q.x && q.values && q.scales, TRIS_ERR_INVALID_ARG, "quantize_e4m3: null x, values or scales");
  TRIS_REQUIRE(q.columns <= (1 << 30), TRIS_ERR_UNSUPPORTED, "quantize_e4m3: more than 2^30 columns");
  QuantizeArgs a{q};
  a.groups = ceil_div(q.columns, kGroup);
  TRIS_REQUIRE(q.rows == 1 || (q.values_stride >= q.columns && q.scales_stride >= a.groups), TRIS_ERR_INVALID_ARG, "quantize_e4m3: rows of values or scales overlap");
  a.units = static_cast<int64_t>(q.rows) * a.groups;
  TRIS_REQUIRE(q.group_rows > 1 ? ceil_div(q.rows, kGroup) <= 65535 : a.units < (1ll << 34), TRIS_ERR_UNSUPPORTED, "quantize_e4m3: too many rows");
  a.wide = aligned_to(q.x, 16) && aligned_to(q.values, 8) && (q.rows == 1 || (q.x_stride % 8 == 0 && q.values_stride % 8 == 0));
  return q.dtype == TRIS_DTYPE_F16 ? launch_quantize<__half>(a, static_cast<cudaStream_t>(stream)) : launch_quantize<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream));
}
