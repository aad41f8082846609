// Residual addition and root-mean-square norm of rows in one pass, with an output in the rows' type or in e4m3 with scales.
//
// h = residual + x; y = h * w / sqrt(mean(h^2) + eps).  The mean needs the whole row before the first output, so a row stays in the registers of
// the CTA that reads it: x and residual are read once, h and y written once.  Bound by bytes for many rows, by the chain load -> sum -> store for one.
// CTAs take several rows, evenly, and ask for the next row before they add up the one they have; the weights stay in registers.
// 2047 x 4096 bf16 to e4m3 with a scale for 128 columns: 12.7 us, 9.0 of them its 59 MB at the rate of a copy; in bf16 10.0 us (67 MB).
// The sums are fp32, h is not rounded before it is squared or scaled.  e4m3: y / s with s = max |y| / 448 of the group, so the group's largest
// element is representable and none saturates; a second exchange between threads gives the maxima.
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kMaxVectors = 4;  // of 8 columns that a thread keeps
constexpr int most_threads(int vectors) { return vectors >= 4 ? 512 : 1024; }  // whose rows fit the registers
// With two registers more for one vector a thread, an SM would have four CTAs of 256 in place of five (2047 x 2048 to e4m3: 8.1 us, 7.2 so).
constexpr int registers(int vectors) { return vectors >= 4 ? 128 : vectors == 2 ? 64 : 48; }
constexpr int threads_on_sm(int vectors) { return 65536 / registers(vectors) / 256 * 256; }

struct NormArgs {
  TrisAddRmsNorm a;
  float inv_hidden;
  int groups;       // scales of a row
  int group_shift;  // log2 of the vectors of a group where that is a power of two up to a warp's lanes, else -1
};

// Over the CTA, for all threads; red has a place for every warp.  A barrier lies between two uses of one red (two of them take turns).
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : 0.f;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_max_sync(0xFFFFFFFFu, lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : 0);
}
// Rows of at most 8 * VECS * blockDim columns, all pointers and strides at 16-byte boundaries.
template <typename T, bool FP8, int VECS>
__global__ void __maxnreg__(registers(VECS)) add_rms_norm_kernel(const __grid_constant__ NormArgs args) {
  const TrisAddRmsNorm& a = args.a;
  __shared__ float red[2][32];
  __shared__ uint32_t red_max[2][32];
  extern __shared__ uint32_t vector_max[];  // groups that do not fit a warp: largest element of every vector
  const int tid = threadIdx.x, vectors = a.hidden_size / 8;
  uint4 w[VECS], x[VECS], r[VECS];
  pdl_wait();  // ahead of the weight, too: it may be what the launch before has made (1 + w)
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = tid + i * blockDim.x;
    w[i] = r[i] = make_uint4(0, 0, 0, 0);
    if (v < vectors) w[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.weight) + 8 * v);
  }
  auto fetch = [&](int64_t row) {
    const T* xs = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* rs = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = tid + i * blockDim.x;
      x[i] = make_uint4(0, 0, 0, 0);
      if (v < vectors) {
        x[i] = *reinterpret_cast<const uint4*>(xs + 8 * v);
        if (a.residual) r[i] = *reinterpret_cast<const uint4*>(rs + 8 * v);
      }
    }
  };
  fetch(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float h[VECS][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      unpack_8<T>(x[i], h[i]);
      if (a.residual) {
        float f[8];
        unpack_8<T>(r[i], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i][k] += f[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += h[i][k] * h[i][k];
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    if (a.residual_out) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int v = tid + i * blockDim.x;
        if (v < vectors) store_8(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + 8 * v, h[i]);
      }
    }
    sum = block_sum(sum, red[turn]);
    const float inv = rsqrtf(sum * args.inv_hidden + a.eps);
    uint32_t top[VECS];  // largest magnitude
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      float f[8];
      unpack_8<T>(w[i], f);
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        h[i][k] = h[i][k] * inv * f[k];
        if (FP8) most = max_or_nan(most, h[i][k]);
      }
      top[i] = magnitude(most);
    }
    if constexpr (!FP8) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int v = tid + i * blockDim.x;
        if (v < vectors) store_8(static_cast<T*>(a.y) + row * a.y_stride + 8 * v, h[i]);
      }
    } else {
      const int per_group = a.group_size / 8;  // vectors
      if (a.group_size == a.hidden_size) {
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < VECS; ++i)
          if (tid + i * blockDim.x < vectors) all = max(all, top[i]);
        all = block_max(all, red_max[turn]);
#pragma unroll
        for (int i = 0; i < VECS; ++i) top[i] = all;
      } else if (args.group_shift >= 0) {
        // neighbours in a warp; vectors past the row only meet one another
#pragma unroll
        for (int d = 16; d; d >>= 1)
          if (d < per_group) {
#pragma unroll
            for (int i = 0; i < VECS; ++i) top[i] = max(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], d));
          }
      } else {
        __syncthreads();  // the row before has been read
#pragma unroll
        for (int i = 0; i < VECS; ++i)
          if (tid + i * blockDim.x < vectors) vector_max[tid + i * blockDim.x] = top[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
          const int v = tid + i * blockDim.x;
          if (v < vectors)
            for (int k = v / per_group * per_group, e = k + per_group; k < e; ++k) top[i] = max(top[i], vector_max[k]);
        }
      }
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int v = tid + i * blockDim.x;
        if (v < vectors) {
          const float scale = quantize_8(h[i], top[i]);
          store_8(static_cast<__nv_fp8_e4m3*>(a.y) + row * a.y_stride + 8 * v, h[i]);
          if (args.group_shift >= 0) {
            if ((v & (per_group - 1)) == 0) a.scales[row * args.groups + (v >> args.group_shift)] = scale;
          } else if (v % per_group == 0) {
            a.scales[row * args.groups + v / per_group] = scale;
          }
        }
      }
    }
  }
}

// Any width and alignment: element by element, the row read again for every use.  Each element is read and written by one thread, so the outputs
// may lie on the inputs: what is read again after a store is not needed from there any more.
template <typename T, bool FP8>
__global__ void __launch_bounds__(1024) add_rms_norm_any_kernel(const __grid_constant__ TrisAddRmsNorm a) {
  __shared__ float red[32];
  __shared__ uint32_t red_max[32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  auto sum_at = [&](int i) { return to_float(x[i]) + (res ? to_float(res[i]) : 0.f); };
  float sum = 0.f;
  for (int i = threadIdx.x; i < a.hidden_size; i += blockDim.x) {
    const float h = sum_at(i);
    sum += h * h;
  }
  const float inv = 1.f / sqrtf(block_sum(sum, red) / a.hidden_size + a.eps);
  const int groups = FP8 ? a.hidden_size / a.group_size : 1, width = FP8 ? a.group_size : a.hidden_size;
  for (int q = 0; q < groups; ++q) {
    float div = 1.f;
    if constexpr (FP8) {
      uint32_t top = 0;
      for (int i = q * width + threadIdx.x; i < (q + 1) * width; i += blockDim.x) top = max(top, magnitude(sum_at(i) * inv * to_float(weight[i])));
      __syncthreads();  // red_max of the group before
      const float scale = __uint_as_float(block_max(top, red_max)) / kE4m3Max;
      div = scale == 0.f ? 1.f : scale;
      if (threadIdx.x == 0) a.scales[row * groups + q] = scale;
    }
    for (int i = q * width + threadIdx.x; i < (q + 1) * width; i += blockDim.x) {
      const float h = sum_at(i), y = h * inv * to_float(weight[i]);
      if (a.residual_out) store_float(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + i, h);
      if constexpr (FP8)
        store_float(static_cast<__nv_fp8_e4m3*>(a.y) + row * a.y_stride + i, y / div);
      else
        store_float(static_cast<T*>(a.y) + row * a.y_stride + i, y);
    }
  }
}

template <typename T, bool FP8>
int launch_norm(const TrisAddRmsNorm& a, cudaStream_t stream) {
  const int H = a.hidden_size;
  const bool pdl = programmatic_launch_default();
  const int64_t strides[4] = {a.x_stride, a.residual ? a.residual_stride : 0, a.residual_out ? a.residual_out_stride : 0, a.y_stride};
  bool wide = H % 8 == 0 && H <= 8 * kMaxVectors * most_threads(kMaxVectors);
  for (int64_t s : strides) wide = wide && s % 8 == 0;
  for (const void* p : {a.x, a.residual, a.weight, static_cast<const void*>(a.residual_out), static_cast<const void*>(a.y)}) wide = wide && (!p || aligned_to(p, 16));
  if (!wide) {
    TRIS_CUDA(launch_step(add_rms_norm_any_kernel<T, FP8>, dim3(a.rows), dim3(H >= 1024 ? 1024 : (H + 31) / 32 * 32), 0, stream, pdl, 1, a));
    return TRIS_OK;
  }
  const int vectors = H / 8;
  // few rows: as many threads as vectors, the chain of one row is what counts (100 x 8192: 3.4 us, 4.1 with 256 threads); many: fewer threads with more
  // loads in flight each (2047 x 4096: 10.0 us, 13.8 with a vector a thread, 10.7 with 128 threads)
  const int sms = sm_count();
  int vecs = 1;
  while (vecs < kMaxVectors && (ceil_div(vectors, vecs) > most_threads(vecs) || (a.rows > sms && ceil_div(vectors, vecs) > 256))) vecs *= 2;
  const int threads = (ceil_div(vectors, vecs) + 31) / 32 * 32;
  NormArgs args{a, 1.f / H, FP8 ? H / a.group_size : 1, -1};
  for (int shift = 0; FP8 && shift <= 5; ++shift)
    if (a.group_size == 8 << shift) args.group_shift = shift;
  const size_t smem = FP8 && a.group_size != H && args.group_shift < 0 ? sizeof(float) * vectors : 0;
  auto kernel = vecs == 1 ? add_rms_norm_kernel<T, FP8, 1> : vecs == 2 ? add_rms_norm_kernel<T, FP8, 2> : add_rms_norm_kernel<T, FP8, 4>;
  const int resident = sms * threads_on_sm(vecs) / threads;
  const int turns = ceil_div(a.rows, resident < 1 ? 1 : resident);
  TRIS_CUDA(launch_step(kernel, dim3(ceil_div(a.rows, turns)), dim3(threads), smem, stream, pdl, 1, args));
  return TRIS_OK;
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_add_rms_norm(const TrisAddRmsNorm* args, void* stream) {
  TRIS_REQUIRE(args, TRIS_ERR_INVALID_ARG, "add_rms_norm: null arguments");
  const TrisAddRmsNorm& a = *args;
  TRIS_REQUIRE(a.dtype == TRIS_DTYPE_F16 || a.dtype == TRIS_DTYPE_BF16, TRIS_ERR_INVALID_ARG, "add_rms_norm: rows are fp16 or bf16");
  TRIS_REQUIRE(a.dtype_out == a.dtype || a.dtype_out == TRIS_DTYPE_E4M3, TRIS_ERR_INVALID_ARG, "add_rms_norm: the output has the rows' type or e4m3");
  TRIS_REQUIRE(a.rows >= 0 && a.hidden_size >= 1, TRIS_ERR_INVALID_ARG, "add_rms_norm: negative sizes");
  if (a.rows == 0) return TRIS_OK;
  TRIS_REQUIRE(a.x && a.weight && a.y, TRIS_ERR_INVALID_ARG, "add_rms_norm: null x, weight or y");
  const bool fp8 = a.dtype_out == TRIS_DTYPE_E4M3;
  if (fp8) {
    TRIS_REQUIRE(a.scales, TRIS_ERR_INVALID_ARG, "add_rms_norm: null scales");
    TRIS_REQUIRE(a.group_size == a.hidden_size || (a.group_size > 0 && a.group_size % 16 == 0 && a.hidden_size % a.group_size == 0), TRIS_ERR_INVALID_ARG,
                 "add_rms_norm: groups of %d columns do not divide rows of %d in multiples of 16", a.group_size, a.hidden_size);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == TRIS_DTYPE_F16) return fp8 ? launch_norm<__half, true>(a, s) : launch_norm<__half, false>(a, s);
  return fp8 ? launch_norm<__nv_bfloat16, true>(a, s) : launch_norm<__nv_bfloat16, false>(a, s);
}
