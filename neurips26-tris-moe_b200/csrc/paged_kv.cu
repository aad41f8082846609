// New keys and values on their way into a paged cache, rotated by their positions.
//
// A dimension pair (a, b) of a token at position p becomes (a cos - b sin, b cos + a sin) with its frequency's row of the tables: a pass over
// the projection's output that reads every element once and writes it once - queries to rows of their own, keys and values to their slots.
// 8188 tokens of 16/16 heads of 128 (202 MB): 36 us, 5.6 TB/s.  Bound by bytes for prompts, by the chain position -> page -> store for a decode step.
// To e4m3 with scales 32 us (168 MB): pages get the quotients (DivideBy has their cost).
//
// A thread has one unit of two 16-byte chunks - the halves (i, i + rotary / 2) that rotate together - and walks over heads with it, so that its
// eight cosines and sines are read once; two heads are asked for before the first of them is rotated.  How many threads share a token's heads follows
// the number of tokens: all heads at once for a decode step, more of them to a thread where the GPU is full without that.
#include "decode_step.cuh"

namespace tris {

int validate_paged_kv(const TrisPagedKv* c, const char* what) {
  TRIS_REQUIRE(c != nullptr, TRIS_ERR_INVALID_ARG, "%s: null cache", what);
  TRIS_REQUIRE(c->dtype == TRIS_DTYPE_F16 || c->dtype == TRIS_DTYPE_BF16 || c->dtype == TRIS_DTYPE_E4M3, TRIS_ERR_INVALID_ARG, "%s: pages hold fp16, bf16 or e4m3", what);
  TRIS_REQUIRE(c->num_sequences >= 0 && c->table_width >= 0 && c->num_pages >= 0 && c->page_size >= 1 && c->num_kv_heads >= 1 && c->head_dim >= 1,
               TRIS_ERR_INVALID_ARG, "%s: negative or zero sizes", what);
  TRIS_REQUIRE(c->k_pages && c->v_pages, TRIS_ERR_INVALID_ARG, "%s: null pages", what);
  TRIS_REQUIRE(c->block_table || c->num_sequences == 0 || c->table_width == 0, TRIS_ERR_INVALID_ARG, "%s: null block table", what);
  const int elt = dtype_size(c->dtype);
  TRIS_REQUIRE(c->head_dim * elt % 16 == 0 && c->head_dim <= 256, TRIS_ERR_UNSUPPORTED, "%s: a head takes a multiple of 16 bytes and up to 256 dimensions (got %d)", what, c->head_dim);
  const int64_t strides[6] = {c->k_page_stride, c->v_page_stride, c->k_token_stride, c->v_token_stride, c->k_head_stride, c->v_head_stride};
  const int sizes[3] = {c->num_pages, c->page_size, c->num_kv_heads};
  for (int i = 0; i < 6; ++i)  // of a size of 1 the stride is of no account
    TRIS_REQUIRE(sizes[i / 2] <= 1 || (strides[i] >= 0 && strides[i] * elt % 16 == 0), TRIS_ERR_UNSUPPORTED, "%s: strides of the pages must be multiples of 16 bytes", what);
  TRIS_REQUIRE(c->scale_tokens >= 0, TRIS_ERR_INVALID_ARG, "%s: negative scale_tokens", what);
  if (c->scale_tokens) {
    TRIS_REQUIRE(c->dtype == TRIS_DTYPE_E4M3 && c->page_size % c->scale_tokens == 0, TRIS_ERR_INVALID_ARG, "%s: blocks of %d tokens belong to e4m3 pages of a multiple of that (%d)", what,
                 c->scale_tokens, c->page_size);
    TRIS_REQUIRE((c->k_scale && c->v_scale) || c->num_pages == 0, TRIS_ERR_INVALID_ARG, "%s: null scales of blocks", what);
  }
  TRIS_REQUIRE(aligned_to(c->k_pages, 16) && aligned_to(c->v_pages, 16), TRIS_ERR_UNSUPPORTED, "%s: pages must start on a 16-byte boundary", what);
  return TRIS_OK;
}

namespace {

struct AppendArgs {
  TrisPagedKv cache;
  TrisPagedAppend rows;
  int units, head_groups;
};

// VEC elements as they are in memory: one 16-byte access for eight.
template <int VEC, typename T>
struct Chunk {
  T v[VEC];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = p[i];
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_float(v[i]);
  }
};
template <typename T>
struct Chunk<8, T> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack_8<T>(v, f); }
};
template <int VEC, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    store_8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) store_float(p + i, v[i]);
  }
}

// VEC: elements of a chunk, 8 (16-byte accesses) or 2 (rows or tables without that alignment).
template <int VEC, typename T, typename C>
__global__ void __launch_bounds__(128) paged_kv_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedAppend& r = a.rows;
  const TrisPagedKv& c = a.cache;
  const uint32_t idx = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t u = idx % a.units, rest = idx / a.units;
  const uint32_t hg = rest % a.head_groups, t = rest / a.head_groups;
  if (t >= static_cast<uint32_t>(r.num_tokens)) return;
  const int D = c.head_dim, half = r.rotary_dim / 2, hq = r.num_q_heads, hkv = c.num_kv_heads;
  const int64_t pos = r.positions_are_64bit ? reinterpret_cast<const int64_t*>(r.positions)[t] : reinterpret_cast<const int32_t*>(r.positions)[t];
  const int seq = r.sequences ? r.sequences[t] : static_cast<int>(t);

  // this unit's two chunks: they rotate together in the half form; -1 where the head has no second one
  const int chunks = D / VEC, pair_units = r.interleaved ? 0 : half / VEC;
  int c0, c1;
  if (static_cast<int>(u) < pair_units) {
    c0 = u;
    c1 = u + pair_units;
  } else {
    c0 = 2 * u;
    c1 = c0 + 1 < chunks ? c0 + 1 : -1;
  }

  bool padding = pos < 0, fits = false;
  int64_t k_at = 0, v_at = 0;
  if (!padding) {
    bool bad = r.cos && pos >= r.max_positions;
    padding = bad;
    if (!bad) {
      bad = seq < 0 || seq >= c.num_sequences || pos >= static_cast<int64_t>(c.table_width) * c.page_size;
      if (!bad) {
        const int page = c.block_table[seq * c.table_stride + pos / c.page_size];
        bad = page < 0 || page >= c.num_pages;
        const int64_t slot = pos % c.page_size;
        k_at = page * c.k_page_stride + slot * c.k_token_stride;
        v_at = page * c.v_page_stride + slot * c.v_token_stride;
      }
      fits = !bad;
    }
    if (bad && c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
  }

  // cosines and sines: of a pair unit VEC frequencies, of an interleaved chunk VEC / 2 for each of its two
  float cs[VEC], sn[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) cs[i] = 1.f, sn[i] = 0.f;
  if (r.cos && !padding && (static_cast<int>(u) < pair_units || r.interleaved)) {
    const int f0 = r.interleaved ? c0 * (VEC / 2) : c0 * VEC;
    const float *cr = r.cos + pos * half + f0, *sr = r.sin + pos * half + f0;
    constexpr int kStep = VEC == 8 ? 4 : 1;
#pragma unroll
    for (int i = 0; i < VEC; i += kStep) {
      if (f0 + i >= half) break;
      if constexpr (VEC == 8) {
        const float4 x = *reinterpret_cast<const float4*>(cr + i), y = *reinterpret_cast<const float4*>(sr + i);
        cs[i] = x.x, cs[i + 1] = x.y, cs[i + 2] = x.z, cs[i + 3] = x.w;
        sn[i] = y.x, sn[i + 1] = y.y, sn[i + 2] = y.z, sn[i + 3] = y.w;
      } else {
        cs[i] = cr[i], sn[i] = sr[i];
      }
    }
  }

  constexpr int kBatch = 2;  // one: 41 us for 8188 tokens of 48 heads of 128; two: 36; four: 40, six: 38
  const int all = hq + 2 * hkv;
  for (int h0 = hg; h0 < all; h0 += kBatch * a.head_groups) {
    // no branch between the loads: heads behind the last read the last one, a chunk that does not exist is its neighbour
    Chunk<VEC, T> in[kBatch][2];
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int h = min(h0 + n * a.head_groups, all - 1);
      const bool is_q = h < hq, is_k = h < hq + hkv;
      const T* src = static_cast<const T*>(is_q ? r.q : is_k ? r.k : r.v) + t * (is_q ? r.q_token_stride : is_k ? r.k_token_stride : r.v_token_stride) +
                     (h - (is_q ? 0 : is_k ? hq : hq + hkv)) * (is_q ? r.q_head_stride : is_k ? r.k_head_stride : r.v_head_stride);
      in[n][0].load(src + c0 * VEC);
      in[n][1].load(src + (c1 >= 0 ? c1 : c0) * VEC);
    }
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int h = h0 + n * a.head_groups;
      if (h >= all) break;
      const int kind = h < hq ? 0 : h < hq + hkv ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - hq : h - hq - hkv;
      float x[VEC], y[VEC];
      in[n][0].get(x);
      in[n][1].get(y);
      if (padding) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = y[i] = 0.f;
      }
      if (kind < 2) {
        if (static_cast<int>(u) < pair_units) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float p = x[i], q = y[i];
            x[i] = p * cs[i] - q * sn[i];
            y[i] = q * cs[i] + p * sn[i];
          }
        } else if (r.interleaved) {
          // chunks behind the rotated dimensions stay as they are: by a cosine of 1 and a sine of 0 an infinity would spoil its neighbour
          if (c0 * VEC < r.rotary_dim) {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              const float p = x[2 * i], q = x[2 * i + 1];
              x[2 * i] = p * cs[i] - q * sn[i];
              x[2 * i + 1] = q * cs[i] + p * sn[i];
            }
          }
          if (c1 * VEC < r.rotary_dim) {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              const float v = y[2 * i], w = y[2 * i + 1];
              y[2 * i] = v * cs[VEC / 2 + i] - w * sn[VEC / 2 + i];
              y[2 * i + 1] = w * cs[VEC / 2 + i] + v * sn[VEC / 2 + i];
            }
          }
        }
      }
      if (kind == 0 || (kind == 1 && r.k_out)) {
        T* dst = kind == 0 ? static_cast<T*>(r.q_out) + (static_cast<int64_t>(t) * hq + hh) * D : static_cast<T*>(r.k_out) + (static_cast<int64_t>(t) * hkv + hh) * D;
        store_vec<VEC>(dst + c0 * VEC, x);
        if (c1 >= 0) store_vec<VEC>(dst + c1 * VEC, y);
      }
      if (kind > 0 && fits) {
        C* dst = kind == 1 ? static_cast<C*>(c.k_pages) + k_at + hh * c.k_head_stride : static_cast<C*>(c.v_pages) + v_at + hh * c.v_head_stride;
        const float* scales = kind == 1 ? c.k_scale : c.v_scale;
        if (sizeof(C) == 1 && scales) {
          const DivideBy divide(scales[hh]);
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < VEC; ++i) top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(y[i])));
          divide(x, top);
          divide(y, top);
        }
        store_vec<VEC>(dst + c0 * VEC, x);
        if (c1 >= 0) store_vec<VEC>(dst + c1 * VEC, y);
      }
    }
  }
}

template <int VEC, typename T, typename C>
int launch_append(const AppendArgs& a, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(a.units) * a.head_groups * a.rows.num_tokens;
  TRIS_CUDA(launch_step(paged_kv_append_kernel<VEC, T, C>, dim3(static_cast<unsigned>((threads + 127) / 128)), dim3(128), 0, stream,
                          programmatic_launch_default(), 1, a));
  return TRIS_OK;
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_paged_kv_append(const TrisPagedKv* cache, const TrisPagedAppend* rows, void* stream) {
  if (int st = validate_paged_kv(cache, "paged_kv_append")) return st;
  TRIS_REQUIRE(rows, TRIS_ERR_INVALID_ARG, "paged_kv_append: null rows");
  const TrisPagedKv& c = *cache;
  const TrisPagedAppend& r = *rows;
  TRIS_REQUIRE(r.dtype == TRIS_DTYPE_F16 || r.dtype == TRIS_DTYPE_BF16, TRIS_ERR_INVALID_ARG, "paged_kv_append: rows are fp16 or bf16");
  TRIS_REQUIRE(c.dtype == TRIS_DTYPE_E4M3 || c.dtype == r.dtype, TRIS_ERR_INVALID_ARG, "paged_kv_append: pages hold the rows' type or e4m3");
  TRIS_REQUIRE(r.num_tokens >= 0 && r.num_q_heads >= 0, TRIS_ERR_INVALID_ARG, "paged_kv_append: negative sizes");
  TRIS_REQUIRE((r.cos == nullptr) == (r.sin == nullptr), TRIS_ERR_INVALID_ARG, "paged_kv_append: cos and sin go together");
  const int rot = r.cos ? r.rotary_dim : 0;
  TRIS_REQUIRE(rot % 2 == 0 && rot >= 0 && rot <= c.head_dim, TRIS_ERR_INVALID_ARG, "paged_kv_append: rotary_dim must be even and at most head_dim (got %d)", rot);
  if (r.num_tokens == 0) return TRIS_OK;
  TRIS_REQUIRE((r.q && r.q_out) || r.num_q_heads == 0, TRIS_ERR_INVALID_ARG, "paged_kv_append: null q or q_out");
  TRIS_REQUIRE(r.k && r.v && r.positions, TRIS_ERR_INVALID_ARG, "paged_kv_append: null k, v or positions");

  if (c.scale_tokens) return append_block_scaled(c, r, rot, static_cast<cudaStream_t>(stream));
  AppendArgs a{c, r, 0, 1};
  a.rows.rotary_dim = rot;
  // 16-byte accesses need rows that start on such boundaries and chunks of 8 that do not straddle the halves or the rotated part
  bool wide = c.head_dim % 8 == 0 && rot % (r.interleaved ? 8 : 16) == 0 && aligned_to(r.cos, 16) && aligned_to(r.sin, 16) && (!r.q_out || aligned_to(r.q_out, 16)) && (!r.k_out || aligned_to(r.k_out, 16));
  const void* src[3] = {r.num_q_heads ? r.q : nullptr, r.k, r.v};
  const int64_t strides[3][2] = {{r.q_token_stride, r.q_head_stride}, {r.k_token_stride, r.k_head_stride}, {r.v_token_stride, r.v_head_stride}};
  for (int i = 0; i < 3; ++i)
    if (src[i]) wide = wide && aligned_to(src[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0;
  const int vec = wide ? 8 : 2;
  TRIS_REQUIRE(wide || r.interleaved || rot % 4 == 0, TRIS_ERR_UNSUPPORTED, "paged_kv_append: rotary_dim must be a multiple of 4");
  a.units = ceil_div(c.head_dim / vec, 2);
  const int heads = r.num_q_heads + 2 * c.num_kv_heads;
  // threads for two rounds of all SMs, with 640 on each; beyond that a thread takes more heads with its cosines and sines (8188 tokens of 48 heads of
  // 128: 36 us, 45 with half as many threads, 40 with twice and with eight times as many; 2048 tokens 11.1, 14.7, 12.3, 20.7)
  a.head_groups = heads;
  const int64_t enough = 2 * 640 * static_cast<int64_t>(sm_count());
  while (a.head_groups > 1 && static_cast<int64_t>(a.units) * a.head_groups * r.num_tokens > enough) a.head_groups = ceil_div(a.head_groups, 2);
  TRIS_REQUIRE(static_cast<int64_t>(a.units) * a.head_groups * r.num_tokens < (1ll << 31), TRIS_ERR_UNSUPPORTED, "paged_kv_append: too many tokens in one call");
  TRIS_REQUIRE(r.sequences || r.num_tokens <= c.num_sequences, TRIS_ERR_INVALID_ARG, "paged_kv_append: %d tokens without sequences for a block table of %d", r.num_tokens, c.num_sequences);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = r.dtype == TRIS_DTYPE_F16, q8 = c.dtype == TRIS_DTYPE_E4M3;
  if (wide) {
    if (f16) return q8 ? launch_append<8, __half, __nv_fp8_e4m3>(a, s) : launch_append<8, __half, __half>(a, s);
    return q8 ? launch_append<8, __nv_bfloat16, __nv_fp8_e4m3>(a, s) : launch_append<8, __nv_bfloat16, __nv_bfloat16>(a, s);
  }
  if (f16) return q8 ? launch_append<2, __half, __nv_fp8_e4m3>(a, s) : launch_append<2, __half, __half>(a, s);
  return q8 ? launch_append<2, __nv_bfloat16, __nv_fp8_e4m3>(a, s) : launch_append<2, __nv_bfloat16, __nv_bfloat16>(a, s);
}
