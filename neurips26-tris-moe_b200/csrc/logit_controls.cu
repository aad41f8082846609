// Penalties for repeated tokens, biases and grammar masks on logits.
//
// A pass over the logits that reads each once and writes it once; which of them a penalty or a bias concerns is looked up in shared memory.  A CTA has
// a slice of one row's vocabulary: it counts the history's tokens that lie in its slice (integer atomics, whose order does not matter) and then
// streams over its logits, the next ones always on their way; the first, the mask and the first tokens of the history are asked for together.
// Every CTA of a row reads the row's history, from L2, at some 24 instructions for 32 tokens: with slices of 4096 logits that was half of all work
// (128 rows of 50304 logits, 3000 tokens and 64 biases 22 us), with four slices a row it is 16 us, 8 of them the stream.  Not kept: eight CTAs of a cluster that
// count in one another's shared memory (31 us, two cluster barriers a CTA), a list of the logits concerned in place of the look-up (19 us), tokens of the slice
// collected before they are counted (24 us; all beside 17 us).
#include <float.h>

#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 256;
constexpr int kMostSlice = 12800;
// A word counts the answer's occurrences in its low 16 bits and the prompt's in those above; in histories of more than 32767 tokens, where that could
// overflow, the answer has 30 bits and the prompt's only set a bit.
constexpr uint32_t kHasBias = 0x80000000u, kPrompt = 0x10000u, kLongPrompt = 0x40000000u;


struct LogitArgs {
  TrisLogitControls c;
  int slice;        // logits of a CTA, a multiple of 32
  int wide;         // whether four logits can be read, and four results written, at once
  int wide_tokens;  // whether four tokens can
  int short_history;
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

// VECS: groups of four logits that a thread has at a time.
template <typename T, int VECS>
__global__ void __launch_bounds__(kThreads, 5) logit_controls_kernel(const __grid_constant__ LogitArgs a) {
  extern __shared__ __align__(16) uint32_t words[];  // [slice] per logit: how often answer and prompt have it, and whether it has a bias
  __shared__ int repeated;                           // whether an id has two biases
  const TrisLogitControls& c = a.c;
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x, v0 = blockIdx.x * a.slice, n = min(a.slice, c.vocab - v0);
  const bool fast = a.wide && n % 4 == 0, marked = c.tokens || c.bias_ids;
  pdl_wait();
  pdl_launch_dependents();
  const T* in = static_cast<const T*>(c.logits) + row * c.logits_stride + v0;
  float* out = c.out + row * c.out_stride + v0;
  const int32_t* allowed = c.allowed ? c.allowed + row * c.allowed_stride + v0 / 32 : nullptr;
  const int32_t* tok = c.tokens ? c.tokens + row * c.tokens_stride : nullptr;
  const int32_t* ids = c.bias_ids ? c.bias_ids + row * c.bias_stride : nullptr;
  const float* values = c.bias_ids ? c.bias_values + row * c.bias_stride : nullptr;

  auto tokens_at = [&](int i) {  // four of them, -1 behind the last
    if (a.wide_tokens && i + 4 <= c.max_tokens) return *reinterpret_cast<const int4*>(tok + i);
    return make_int4(i < c.max_tokens ? tok[i] : -1, i + 1 < c.max_tokens ? tok[i + 1] : -1, i + 2 < c.max_tokens ? tok[i + 2] : -1,
                     i + 3 < c.max_tokens ? tok[i + 3] : -1);
  };
  int4 now = make_int4(-1, -1, -1, -1);
  if (tok) now = tokens_at(4 * tid);  // whether or not the history is that long
  const int len = tok ? min(max(c.token_lengths[row], 0), c.max_tokens) : 0;
  const int answer = tok && c.prompt_lengths ? c.prompt_lengths[row] : 0;  // first token that is counted
  const int first_id = ids && tid < c.num_biases ? ids[tid] : -1;
  const float first_value = ids && tid < c.num_biases ? values[tid] : 0.f;
  float z[VECS][4], z_next[VECS][4];
  uint32_t bits[VECS], bits_next[VECS];
  // No branch between the loads, and nothing that waits for one: places behind the slice's end read its last ones.
  auto fetch = [&](int base, float (&z)[VECS][4], uint32_t (&bits)[VECS]) {
    if (fast) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) load_4(in + min(base + 4 * (tid + i * kThreads), n - 4), z[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VECS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) z[i][k] = to_float(in[min(base + 4 * (tid + i * kThreads) + k, n - 1)]);
    }
    if (allowed) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) bits[i] = allowed[min(base + 4 * (tid + i * kThreads), n - 1) / 32];
    }
  };
  fetch(0, z, bits);
  const float rep = c.repetition ? c.repetition[row] : 1.f, pres = c.presence ? c.presence[row] : 0.f, freq = c.frequency ? c.frequency[row] : 0.f;

  if (marked) {
    for (int i = tid; i < a.slice / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) repeated = 0;
    __syncthreads();
    auto mark = [&](int id, int i) {
      const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
      if (at < static_cast<uint32_t>(n)) {
        if (a.short_history || i >= answer)
          atomicAdd(words + at, i >= answer ? 1u : kPrompt);
        else
          atomicOr(words + at, kLongPrompt);
      }
    };
    for (int i = 4 * tid; i < len;) {
      const int next = i + 4 * kThreads;
      int4 then = make_int4(-1, -1, -1, -1);
      if (next < len) then = tokens_at(next);
      if (i + 4 > len) {
        if (i + 1 >= len) now.y = -1;
        if (i + 2 >= len) now.z = -1;
        now.w = -1;
      }
      mark(now.x, i);
      mark(now.y, i + 1);
      mark(now.z, i + 2);
      mark(now.w, i + 3);
      now = then;
      i = next;
    }
    for (int i = tid; ids && i < c.num_biases; i += kThreads) {
      const int id = i == tid ? first_id : ids[i];
      if (id >= v0 && id - v0 < n && (atomicOr(words + (id - v0), kHasBias) & kHasBias)) repeated = 1;
    }
    __syncthreads();
  }

  // z / rep by the reciprocal's two parts (128 rows of 50304 logits without biases: 14.5 us; 15.9 by a division; 13.8 by one part, which is a rounding
  // off).  An infinite z has no second product, a rep of 0 or without end no second part.
  const DivideBy divide(rep);
  const float less_lo = divide.lo == divide.lo ? divide.lo : 0.f;
  auto penalised = [&](float z) {
    const float v = z * divide.lift, second = fminf(v, FLT_MAX) * less_lo;
    return z > 0.f ? fmaf(v, divide.hi, second) : z * rep;
  };
  const uint32_t in_answer = a.short_history ? kPrompt - 1 : kLongPrompt - 1;
  for (int base = 0; base < n; base += 4 * VECS * kThreads) {
    if (base + 4 * VECS * kThreads < n) fetch(base + 4 * VECS * kThreads, z_next, bits_next);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = base + 4 * (tid + i * kThreads);
      if (at >= n) break;
      if (tok) {
        const uint4 raw = *reinterpret_cast<const uint4*>(words + at);
        if ((raw.x | raw.y | raw.z | raw.w) & ~kHasBias) {
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float scaled = penalised(z[i][k]);
            if ((w[k] & ~kHasBias) && c.repetition) z[i][k] = scaled;
            const uint32_t count = w[k] & in_answer;
            const float lower = z[i][k] - freq * static_cast<float>(count) - pres;
            if (count) z[i][k] = lower;
          }
        }
      }
      if (allowed) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (!((bits[i] >> (at & 31)) & (1u << k))) z[i][k] = -INFINITY;
      }
      if (fast) {
        *reinterpret_cast<float4*>(out + at) = make_float4(z[i][0], z[i][1], z[i][2], z[i][3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at + k < n) out[at + k] = z[i][k];
      }
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      bits[i] = bits_next[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i][k] = z_next[i][k];
    }
  }
  if (!ids) return;
  // Biases are few: they are added to what has been written, one thread an entry.
  __syncthreads();
  if (!repeated) {
    for (int i = tid; i < c.num_biases; i += kThreads) {
      const int id = i == tid ? first_id : ids[i], at = id - v0;
      if (id < v0 || at >= n) continue;
      const float bias = i == tid ? first_value : values[i];
      if (!allowed || (allowed[at / 32] >> (at & 31)) & 1) out[at] += bias;
    }
    return;
  }
  // Some ids are there more than once.  The list is taken as many entries at a time as there are threads: of a warp's entries of one id the first adds up all, in
  // their order, and of several warps' the lowest goes first, which the words tell that have done their service.  Time grows with the list's length, not its square.
#pragma unroll 1
  for (int base = 0; base < c.num_biases; base += kThreads) {
    const int i = base + tid, lane = tid & 31;
    const int id = i < c.num_biases ? ids[i] : -1, at = id - v0;
    const bool here = id >= v0 && at < n;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, here ? at : -1);
    const float value = here ? values[i] : 0.f;
    float bias = value;
    if (__any_sync(0xFFFFFFFFu, here && (same & (same - 1)))) {
      for (int k = 1; k < 32; ++k) {
        const float v = __shfl_sync(0xFFFFFFFFu, value, k);
        if (k > lane && ((same >> k) & 1)) bias += v;
      }
    }
    bool pending = here && __ffs(same) - 1 == lane && (!allowed || (allowed[at / 32] >> (at & 31)) & 1);
    while (__syncthreads_or(pending)) {
      if (pending) words[at] = kThreads;
      __syncthreads();
      if (pending) atomicMin(words + at, tid);
      __syncthreads();
      if (pending && words[at] == tid) {
        out[at] += bias;
        pending = false;
      }
    }
  }
}

template <typename T, int VECS>
int launch_controls(LogitArgs& a, int most, cudaStream_t stream) {
  const TrisLogitControls& c = a.c;
  const int slices = ceil_div(c.vocab, most);
  a.slice = (ceil_div(c.vocab, slices) + 31) / 32 * 32;  // even ones
  const size_t smem = c.tokens || c.bias_ids ? 4 * static_cast<size_t>(a.slice) : 0;
  if (int st = allow_shared_memory<logit_controls_kernel<T, VECS>>(4 * kMostSlice)) return st;
  TRIS_CUDA(launch_step(logit_controls_kernel<T, VECS>, dim3(ceil_div(c.vocab, a.slice), c.rows), dim3(kThreads), smem, stream, programmatic_launch_default(), 1, a));
  return TRIS_OK;
}
// Slices of 1024 where larger ones would leave SMs without work: small and large ones take 3.3 and 7.7 us for one row of 50304 logits, 7.1 and 8.2 for 22,
// 9.2 and 8.2 for 32, 15.2 and 9.2 for 64.
template <typename T>
int launch_controls(LogitArgs& a, cudaStream_t stream) {
  const bool few = static_cast<int64_t>(ceil_div(a.c.vocab, 4096)) * a.c.rows < 2 * sm_count();
  return few ? launch_controls<T, 1>(a, 1024, stream) : launch_controls<T, 2>(a, kMostSlice, stream);
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
  TRIS_REQUIRE(c.max_tokens < (1 << 30) && c.vocab < (1 << 30), TRIS_ERR_UNSUPPORTED, "logit_controls: histories or vocabularies of 2^30 tokens and more");
  TRIS_REQUIRE(c.logits && c.out, TRIS_ERR_INVALID_ARG, "logit_controls: null logits or out");
  TRIS_REQUIRE(!c.tokens || c.token_lengths, TRIS_ERR_INVALID_ARG, "logit_controls: tokens need token_lengths");
  TRIS_REQUIRE(c.tokens || c.max_tokens == 0 || !(c.repetition || c.presence || c.frequency), TRIS_ERR_INVALID_ARG, "logit_controls: penalties need tokens");
  TRIS_REQUIRE(!c.bias_ids == !c.bias_values, TRIS_ERR_INVALID_ARG, "logit_controls: bias_ids and bias_values go together");
  const int elt = dtype_size(c.dtype);
  LogitArgs a{c, 0, 0, aligned_to(c.tokens, 16) && c.tokens_stride % 4 == 0, c.max_tokens < 32768};
  if (!(c.repetition || c.presence || c.frequency) || c.max_tokens == 0) a.c.tokens = nullptr;
  if (c.num_biases == 0) a.c.bias_ids = nullptr;
  a.wide = aligned_to(c.logits, 4 * elt) && aligned_to(c.out, 16) && c.logits_stride % 4 == 0 && c.out_stride % 4 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.dtype == TRIS_DTYPE_F16 ? launch_controls<__half>(a, s) : c.dtype == TRIS_DTYPE_BF16 ? launch_controls<__nv_bfloat16>(a, s) : launch_controls<float>(a, s);
}
