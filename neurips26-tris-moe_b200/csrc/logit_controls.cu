// Penalties for repeated tokens, biases and grammar masks on logits.
//
// A pass over the logits that reads each once and writes it once; which of them a penalty or a bias concerns is looked up in shared memory.  A CTA
// has a slice of one row's vocabulary: it counts the history's tokens that lie in its slice (integer atomics, whose order does not matter), then
// streams over the slice.  Every CTA of a row reads the row's history, which stays in L2: for slices of kSlice logits that is a small part of
// what the slice itself reads and writes, up to histories of some thousand tokens.
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kHasBias = 0x80000000u, kInPrompt = 0x40000000u, kCount = 0x3FFFFFFFu;

struct LogitArgs {
  TrisLogitControls c;
  int slice;      // logits of a CTA, a multiple of 32
  int wide;       // rows of logits and out start on 16-byte boundaries
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logit_controls_kernel(const __grid_constant__ LogitArgs a) {
  extern __shared__ uint32_t words[];  // per logit of the slice: occurrences in the answer, whether in the prompt, whether it has a bias
  pdl_wait();
  pdl_launch_dependents();
  const TrisLogitControls& c = a.c;
  const int row = blockIdx.y, v0 = blockIdx.x * a.slice, n = min(a.slice, c.vocab - v0), tid = threadIdx.x;
  const bool marked = c.tokens || c.bias_ids;
  if (marked) {
    for (int i = tid; i < n; i += kThreads) words[i] = 0;
    __syncthreads();
    if (c.tokens) {
      const int32_t* tok = c.tokens + row * c.tokens_stride;
      const int len = min(max(c.token_lengths[row], 0), c.max_tokens);
      const int prompt = c.prompt_lengths ? c.prompt_lengths[row] : 0;
#pragma unroll 4
      for (int i = tid; i < len; i += kThreads) {
        const uint32_t at = static_cast<uint32_t>(tok[i]) - static_cast<uint32_t>(v0);
        if (tok[i] >= 0 && at < static_cast<uint32_t>(n)) {
          if (i < prompt)
            atomicOr(words + at, kInPrompt);
          else
            atomicAdd(words + at, 1u);
        }
      }
    }
    if (c.bias_ids) {
      for (int i = tid; i < c.num_biases; i += kThreads) {
        const int id = c.bias_ids[row * c.bias_stride + i];
        if (id >= v0 && id - v0 < n) atomicOr(words + (id - v0), kHasBias);
      }
    }
    __syncthreads();
  }
  const float rep = c.repetition ? c.repetition[row] : 1.f, pres = c.presence ? c.presence[row] : 0.f, freq = c.frequency ? c.frequency[row] : 0.f;
  const T* in = static_cast<const T*>(c.logits) + row * c.logits_stride + v0;
  float* out = c.out + row * c.out_stride + v0;
  const int32_t* allowed = c.allowed ? c.allowed + row * c.allowed_stride + v0 / 32 : nullptr;

  auto controlled = [&](float z, int i, uint32_t bits) {
    if (marked) {
      const uint32_t w = words[i];
      if (w) {
        if (w & ~kHasBias) {
          if (c.repetition) z = z > 0.f ? z / rep : z * rep;
          const uint32_t count = w & kCount;
          if (count) z = z - freq * static_cast<float>(count) - pres;
        }
        if (w & kHasBias) {
          float bias = 0.f;
          for (int k = 0; k < c.num_biases; ++k)
            if (c.bias_ids[row * c.bias_stride + k] == v0 + i) bias += c.bias_values[row * c.bias_stride + k];
          z += bias;
        }
      }
    }
    return (bits >> (i & 31)) & 1 ? z : -INFINITY;
  };
  if (a.wide) {
    constexpr int kVec = sizeof(T) == 4 ? 4 : 8;
#pragma unroll 2
    for (int i = tid * kVec; i + kVec <= n; i += kThreads * kVec) {
      float z[kVec];
      if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4*>(in + i);
        z[0] = f.x, z[1] = f.y, z[2] = f.z, z[3] = f.w;
      } else {
        load_8(in + i, z);
      }
      const uint32_t bits = allowed ? allowed[i / 32] : 0xFFFFFFFFu;
#pragma unroll
      for (int k = 0; k < kVec; ++k) z[k] = controlled(z[k], i + k, bits);
#pragma unroll
      for (int k = 0; k < kVec; k += 4) *reinterpret_cast<float4*>(out + i + k) = make_float4(z[k], z[k + 1], z[k + 2], z[k + 3]);
    }
    const int done = n / kVec * kVec;
    if (tid < n - done) out[done + tid] = controlled(to_float(in[done + tid]), done + tid, allowed ? allowed[(done + tid) / 32] : 0xFFFFFFFFu);
  } else {
    for (int i = tid; i < n; i += kThreads) out[i] = controlled(to_float(in[i]), i, allowed ? allowed[i / 32] : 0xFFFFFFFFu);
  }
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_logit_controls(const TrisLogitControls* args, void* stream) {
  TRIS_REQUIRE(args, TRIS_ERR_INVALID_ARG, "logit_controls: null arguments");
  const TrisLogitControls& c = *args;
  TRIS_REQUIRE(c.dtype == TRIS_DTYPE_F16 || c.dtype == TRIS_DTYPE_BF16 || c.dtype == TRIS_DTYPE_F32, TRIS_ERR_INVALID_ARG, "logit_controls: logits are fp16, bf16 or fp32");
  TRIS_REQUIRE(c.rows >= 0 && c.vocab >= 0 && c.max_tokens >= 0 && c.num_biases >= 0, TRIS_ERR_INVALID_ARG, "logit_controls: negative sizes");
  if (c.rows == 0 || c.vocab == 0) return TRIS_OK;
  TRIS_REQUIRE(c.rows <= 65535, TRIS_ERR_UNSUPPORTED, "logit_controls: more than 65535 rows");
  TRIS_REQUIRE(c.max_tokens < (1 << 30), TRIS_ERR_UNSUPPORTED, "logit_controls: histories of 2^30 tokens and more");
  TRIS_REQUIRE(c.logits && c.out, TRIS_ERR_INVALID_ARG, "logit_controls: null logits or out");
  TRIS_REQUIRE(!c.tokens || c.token_lengths, TRIS_ERR_INVALID_ARG, "logit_controls: tokens need token_lengths");
  TRIS_REQUIRE(c.tokens || c.max_tokens == 0 || !(c.repetition || c.presence || c.frequency), TRIS_ERR_INVALID_ARG, "logit_controls: penalties need tokens");
  TRIS_REQUIRE(!c.bias_ids == !c.bias_values, TRIS_ERR_INVALID_ARG, "logit_controls: bias_ids and bias_values go together");
  const int elt = dtype_size(c.dtype);
  LogitArgs a{c, 0, 0};
  if (!(c.repetition || c.presence || c.frequency)) a.c.tokens = nullptr;
  a.wide = aligned_to(c.logits, 16) && aligned_to(c.out, 16) && c.logits_stride * elt % 16 == 0 && c.out_stride % 4 == 0;
  a.slice = 8192;
  while (a.slice > 1024 && static_cast<int64_t>(ceil_div(c.vocab, a.slice)) * c.rows < 148 * 2) a.slice /= 2;
  const size_t smem = a.c.tokens || c.bias_ids ? sizeof(uint32_t) * a.slice : 0;
  const dim3 grid(ceil_div(c.vocab, a.slice), c.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto kernel = c.dtype == TRIS_DTYPE_F16 ? logit_controls_kernel<__half> : c.dtype == TRIS_DTYPE_BF16 ? logit_controls_kernel<__nv_bfloat16> : logit_controls_kernel<float>;
  TRIS_CUDA(launch_kernel(kernel, grid, dim3(kThreads), smem, s, programmatic_launch_default(), 1, a));
  return TRIS_OK;
}
