// Penalties for repeated tokens, biases and grammar masks on logits.
//
// A pass over the logits that reads each once and writes it once; which of them a penalty concerns is looked up in shared memory.  A CTA has a slice
// of one row's vocabulary: it counts the history's tokens that lie in its slice (integer atomics, whose order does not matter) and then changes
// its logits.  Those are few for every thread, and asked for before anything else, as are the first tokens of the history: the three ways to memory
// overlap.  Every CTA of a row reads the row's history, which comes from L2; slices of 4096 logits keep that below what the slice itself takes for
// histories of up to some thousand tokens.  Biases are few: they are added to what the CTA has written, one thread an entry.
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // tokens of the history that a thread asks for at once
constexpr uint32_t kHasBias = 0x80000000u, kInPrompt = 0x40000000u, kCount = 0x3FFFFFFFu;

struct LogitArgs {
  TrisLogitControls c;
  int wide;  // whether four logits can be read, and four results written, at once
};

template <typename T>
__device__ __forceinline__ void load_4(const T* p, float (&z)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    z[0] = f.x, z[1] = f.y, z[2] = f.z, z[3] = f.w;
  } else {
    const uint2 raw = *reinterpret_cast<const uint2*>(p);
    const float2 lo = Pair<T>::unpack(raw.x), hi = Pair<T>::unpack(raw.y);
    z[0] = lo.x, z[1] = lo.y, z[2] = hi.x, z[3] = hi.y;
  }
}

// VECS: groups of four logits that a thread has.
template <typename T, int VECS>
__global__ void __launch_bounds__(kThreads, 5) logit_controls_kernel(const __grid_constant__ LogitArgs a) {
  constexpr int kSlice = kThreads * 4 * VECS;
  __shared__ __align__(16) uint32_t words[kSlice];  // per logit: occurrences in the answer, whether in the prompt, whether it has a bias
  __shared__ int repeated;                          // whether an id has two biases
  const TrisLogitControls& c = a.c;
  const int64_t row = blockIdx.y;
  const int v0 = blockIdx.x * kSlice, n = min(kSlice, c.vocab - v0), tid = threadIdx.x;
  if (c.tokens || c.bias_ids) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) reinterpret_cast<uint4*>(words)[tid + i * kThreads] = make_uint4(0, 0, 0, 0);
    if (tid == 0) repeated = 0;
  }
  pdl_wait();
  pdl_launch_dependents();
  const T* in = static_cast<const T*>(c.logits) + row * c.logits_stride + v0;
  float* out = c.out + row * c.out_stride + v0;
  const int32_t* allowed = c.allowed ? c.allowed + row * c.allowed_stride + v0 / 32 : nullptr;
  const int32_t* tok = c.tokens ? c.tokens + row * c.tokens_stride : nullptr;

  int ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ahead[k] = tok && tid + k * kThreads < c.max_tokens ? tok[tid + k * kThreads] : -1;
  float z[VECS][4];
  uint32_t bits[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = 4 * (tid + i * kThreads);
    bits[i] = allowed && at < n ? allowed[at / 32] >> (at & 31) : 0xFu;
    if (a.wide && at + 4 <= n) {
      load_4(in + at, z[i]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i][k] = at + k < n ? to_float(in[at + k]) : 0.f;
    }
  }

  if (c.tokens || c.bias_ids) {
    const int len = tok ? min(max(c.token_lengths[row], 0), c.max_tokens) : 0;
    const int prompt = c.prompt_lengths ? c.prompt_lengths[row] : 0;
    __syncthreads();
    for (int i0 = tid; i0 < len; i0 += kAhead * kThreads) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k * kThreads;
        const int id = ahead[k];
        if (i < len && id >= v0 && id - v0 < n) {
          if (i < prompt)
            atomicOr(words + (id - v0), kInPrompt);
          else
            atomicAdd(words + (id - v0), 1u);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + (kAhead + k) * kThreads;
        ahead[k] = i < len ? tok[i] : -1;
      }
    }
    for (int i = tid; c.bias_ids && i < c.num_biases; i += kThreads) {
      const int id = c.bias_ids[row * c.bias_stride + i];
      if (id >= v0 && id - v0 < n && (atomicOr(words + (id - v0), kHasBias) & kHasBias)) repeated = 1;
    }
    __syncthreads();
  }

  const float rep = c.repetition ? c.repetition[row] : 1.f, pres = c.presence ? c.presence[row] : 0.f, freq = c.frequency ? c.frequency[row] : 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = 4 * (tid + i * kThreads);
    if (at >= n) break;
    if (tok) {
      const uint4 raw = *reinterpret_cast<const uint4*>(words + at);
      const uint32_t w[4] = {raw.x & ~kHasBias, raw.y & ~kHasBias, raw.z & ~kHasBias, raw.w & ~kHasBias};
      if (w[0] | w[1] | w[2] | w[3]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (w[k]) {
            if (c.repetition) z[i][k] = z[i][k] > 0.f ? z[i][k] / rep : z[i][k] * rep;
            if (w[k] & kCount) z[i][k] = z[i][k] - freq * static_cast<float>(w[k] & kCount) - pres;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (!((bits[i] >> k) & 1)) z[i][k] = -INFINITY;
    if (a.wide && at + 4 <= n) {
      *reinterpret_cast<float4*>(out + at) = make_float4(z[i][0], z[i][1], z[i][2], z[i][3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k < n) out[at + k] = z[i][k];
    }
  }
  if (!c.bias_ids) return;
  __syncthreads();
  for (int i = tid; i < c.num_biases; i += kThreads) {
    const int32_t* ids = c.bias_ids + row * c.bias_stride;
    const float* values = c.bias_values + row * c.bias_stride;
    const int id = ids[i], at = id - v0;
    if (id < v0 || at >= n) continue;
    float bias = values[i];
    if (repeated) {  // the first of an id's entries adds all of them, in their order
      bool first = true;
      for (int k = 0; k < i; ++k) first = first && ids[k] != id;
      if (!first) continue;
      for (int k = i + 1; k < c.num_biases; ++k)
        if (ids[k] == id) bias += values[k];
    }
    if (!allowed || (allowed[at / 32] >> (at & 31)) & 1) out[at] += bias;
  }
}

template <int VECS>
int launch_controls(const LogitArgs& a, cudaStream_t stream) {
  const TrisLogitControls& c = a.c;
  auto kernel = c.dtype == TRIS_DTYPE_F16    ? logit_controls_kernel<__half, VECS>
                : c.dtype == TRIS_DTYPE_BF16 ? logit_controls_kernel<__nv_bfloat16, VECS>
                                             : logit_controls_kernel<float, VECS>;
  TRIS_CUDA(launch_kernel(kernel, dim3(ceil_div(c.vocab, kThreads * 4 * VECS), c.rows), dim3(kThreads), 0, stream, programmatic_launch_default(), 1, a));
  return TRIS_OK;
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
  LogitArgs a{c, 0};
  if (!(c.repetition || c.presence || c.frequency) || c.max_tokens == 0) a.c.tokens = nullptr;
  if (c.num_biases == 0) a.c.bias_ids = nullptr;
  a.wide = aligned_to(c.logits, 4 * elt) && aligned_to(c.out, 16) && c.logits_stride % 4 == 0 && c.out_stride % 4 == 0;
  // slices of 4096 where that still gives every SM some, else of 1024
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return static_cast<int64_t>(ceil_div(c.vocab, 4096)) * c.rows >= 2 * 148 ? launch_controls<4>(a, s) : launch_controls<1>(a, s);
}
