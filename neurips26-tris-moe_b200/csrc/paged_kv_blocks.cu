// New keys and values on their way into a paged cache in e4m3 with a scale for each block of tokens and head, rotated by their positions.
//
// A block's scale is the smallest power of two by which its numbers stay within 448.  A token that needs a larger one than its block has gives the block a
// new scale, and the block's tokens ahead of it are read and written once more; between powers of two that shifts exponents, so nothing is lost by it
// (but for what becomes smaller than e4m3 can be), however often it happens.  Bound by bytes for prompts, by the chain position -> page -> scale -> store for
// a decode step.
//
// Tokens that follow one another in a block are a run, and one warp has all of a run for one head's keys or values: it finds the largest
// magnitude, then scales and stores.  Up to kHeld rows for each of its row places stay in registers in between; longer runs are read again, from L1 or L2.
// Whoever has the chunk of tokens in which a run begins has all of it.  Queries are only rotated, head by head.
#include <float.h>

#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kWarps = 4, kHeld = 8;

struct BlockArgs {
  TrisPagedKv cache;
  TrisPagedAppend rows;
  int chunk;        // tokens that a warp looks at: 1 to 32
  int lanes;        // that have a row, eight dimensions each: a power of two
  int wide;         // whether eight elements can be read, and eight results of q_out and k_out written, at once
  int wide_tables;  // whether four cosines can
};

// The biased exponent of the smallest power of two s with top <= 448 s, from 2^-64 to 2^64.
__device__ __forceinline__ float block_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(min(max(e, 127 - 64), 127 + 64)) << 23);
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_kv_append_blocks_kernel(const __grid_constant__ BlockArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedAppend& r = a.rows;
  const TrisPagedKv& c = a.cache;
  const int lane = threadIdx.x & 31, hq = r.num_q_heads, hkv = c.num_kv_heads;
  const int item = blockIdx.y * kWarps + (threadIdx.x >> 5);  // a query head, a head's keys or a head's values
  if (item >= hq + 2 * hkv) return;
  const int kind = item < hq ? 0 : item < hq + hkv ? 1 : 2, head = kind == 0 ? item : kind == 1 ? item - hq : item - hq - hkv;
  const int D = c.head_dim, rot = r.rotary_dim, half = rot / 2, block = c.scale_tokens;
  const int64_t room = static_cast<int64_t>(c.table_width) * c.page_size;
  const int t0 = blockIdx.x * a.chunk, t1 = min(r.num_tokens, t0 + a.chunk);

  // What a lane knows of token t0 + lane: its position (-1: padding, -2: it has no place), its page, and whether it goes on where the token before it is.
  struct Token {
    int pos, page;
    bool follows;
  };
  auto look = [&](int t) {
    Token k{-1, -1, false};
    if (t >= r.num_tokens) return k;
    const int64_t pos = r.positions_are_64bit ? reinterpret_cast<const int64_t*>(r.positions)[t] : reinterpret_cast<const int32_t*>(r.positions)[t];
    const int seq = r.sequences ? r.sequences[t] : t;
    if (pos < 0) return k;
    bool fits = seq >= 0 && seq < c.num_sequences && pos < room;
    const bool turns = !r.cos || pos < r.max_positions;
    if (fits) {
      k.page = c.block_table[seq * c.table_stride + pos / c.page_size];
      fits = k.page >= 0 && k.page < c.num_pages;
    }
    if (!fits || !turns) {
      if (c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
      k.pos = turns ? -2 : -1;  // one without a place is still rotated, as long as the tables have its position
      if (turns) k.page = static_cast<int>(min(pos, static_cast<int64_t>(0x7FFFFFFF)));
      return k;
    }
    k.pos = static_cast<int>(pos);
    if (t > 0 && pos % block) {
      const int64_t before = r.positions_are_64bit ? reinterpret_cast<const int64_t*>(r.positions)[t - 1] : reinterpret_cast<const int32_t*>(r.positions)[t - 1];
      k.follows = before == pos - 1 && r.sequences && r.sequences[t - 1] == seq;
    }
    return k;
  };
  const Token own = look(lane < a.chunk ? t0 + lane : r.num_tokens);

  const int l = lane % a.lanes, place = lane / a.lanes, places = 32 / a.lanes, d0 = 8 * l;
  const bool active = d0 < D;
  const T* src = static_cast<const T*>(kind == 0 ? r.q : kind == 1 ? r.k : r.v) + head * (kind == 0 ? r.q_head_stride : kind == 1 ? r.k_head_stride : r.v_head_stride);
  const int64_t src_stride = kind == 0 ? r.q_token_stride : kind == 1 ? r.k_token_stride : r.v_token_stride;
  auto fetch = [&](int t) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (t < 0 || !active) return raw;
    const T* p = src + t * src_stride + d0;
    if (a.wide) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint16_t*>(p + 2 * i) | (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 2 * i + 1)) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // Eight dimensions of token t at position pos (t < 0: none), rotated where they are queries or keys.  By a whole warp.
  const bool halves = !r.interleaved && half % 8 == 0;  // the other element of each pair is in one other lane, at the same place
  auto turned = [&](const uint4& raw, int t, int pos, float (&v)[8]) {
    unpack_8<T>(raw, v);
    if (kind == 2 || rot == 0) return;
    float other[8];
    if (halves) {
      const int from = d0 < half ? lane + half / 8 : d0 < rot ? lane - half / 8 : lane;
      const uint4 pair = make_uint4(__shfl_sync(0xFFFFFFFFu, raw.x, from), __shfl_sync(0xFFFFFFFFu, raw.y, from), __shfl_sync(0xFFFFFFFFu, raw.z, from), __shfl_sync(0xFFFFFFFFu, raw.w, from));
      unpack_8<T>(pair, other);
    }
    if (t < 0 || !active || d0 >= rot) return;
    const float *cr = r.cos + static_cast<int64_t>(pos) * half, *sr = r.sin + static_cast<int64_t>(pos) * half;
    if (halves) {
      const int f0 = d0 < half ? d0 : d0 - half;
      float cs[8], sn[8];
      if (a.wide_tables) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 x = *reinterpret_cast<const float4*>(cr + f0 + i), y = *reinterpret_cast<const float4*>(sr + f0 + i);
          cs[i] = x.x, cs[i + 1] = x.y, cs[i + 2] = x.z, cs[i + 3] = x.w;
          sn[i] = y.x, sn[i + 1] = y.y, sn[i + 2] = y.z, sn[i + 3] = y.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = cr[f0 + i], sn[i] = sr[f0 + i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d0 < half ? v[i] * cs[i] - other[i] * sn[i] : v[i] * cs[i] + other[i] * sn[i];
    } else if (r.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if (d0 + i >= rot) break;
        const float x = v[i], y = v[i + 1], cs = cr[(d0 + i) / 2], sn = sr[(d0 + i) / 2];
        v[i] = x * cs - y * sn;
        v[i + 1] = y * cs + x * sn;
      }
    } else {
      const T* p = src + t * src_stride;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        if (d >= rot) break;
        v[i] = d < half ? v[i] * cr[d] - to_float(p[d + half]) * sr[d] : v[i] * cr[d - half] + to_float(p[d - half]) * sr[d - half];
      }
    }
  };
  auto put_row = [&](void* out, int64_t row, const float (&v)[8]) {  // of q_out or k_out
    if (!active) return;
    T* p = static_cast<T*>(out) + row * D + d0;
    if (a.wide) {
      store_8(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) store_float(p + i, v[i]);
    }
  };

  // Rows that are rotated and go out as they are: queries, and keys that the caller asks for.
  void* out = kind == 0 ? r.q_out : kind == 1 ? r.k_out : nullptr;
  if (out) {
    const int heads = kind == 0 ? hq : hkv;
#pragma unroll 1
    for (int base = t0; base < t1; base += 4 * places) {
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = base + i * places + place;
        raw[i] = fetch(t < t1 ? t : -1);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = base + i * places + place, from = t < t1 ? t - t0 : 0;
        int pos = __shfl_sync(0xFFFFFFFFu, own.pos, from);
        const int without = __shfl_sync(0xFFFFFFFFu, own.page, from);
        if (pos == -2) pos = without;
        float v[8];
        turned(raw[i], t < t1 && pos >= 0 ? t : -1, pos, v);
        if (pos < 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = 0.f;
        }
        if (t < t1) put_row(out, static_cast<int64_t>(t) * heads + head, v);
      }
    }
  }
  if (kind == 0) return;

  uint8_t* pages = static_cast<uint8_t*>(kind == 1 ? c.k_pages : c.v_pages) + head * (kind == 1 ? c.k_head_stride : c.v_head_stride);
  const int64_t page_stride = kind == 1 ? c.k_page_stride : c.v_page_stride, token_stride = kind == 1 ? c.k_token_stride : c.v_token_stride;
  float* scales = const_cast<float*>(kind == 1 ? c.k_scale : c.v_scale);
  const uint32_t placed = __ballot_sync(0xFFFFFFFFu, own.pos >= 0), follows = __ballot_sync(0xFFFFFFFFu, own.follows);
#pragma unroll 1
  for (uint32_t runs = placed & ~follows; runs; runs &= runs - 1) {
    const int lead = __ffs(runs) - 1;
    const int pos0 = __shfl_sync(0xFFFFFFFFu, own.pos, lead), page = __shfl_sync(0xFFFFFFFFu, own.page, lead), first = t0 + lead;
    // its length: tokens that follow, in this chunk and behind it
    const uint32_t behind = lead == 31 ? 0 : ~follows >> (lead + 1);  // (bits behind the chunk's last token are 0 in follows)
    int length = behind ? __ffs(behind) : 32 - lead;
    if (first + length == t1) {
      for (;;) {
        const uint32_t more = ~__ballot_sync(0xFFFFFFFFu, look(first + length + lane).follows);
        length += more ? __ffs(more) - 1 : 32;
        if (more) break;
      }
    }
    const int slot0 = pos0 % c.page_size, ahead = slot0 % block;  // tokens of the block ahead of the run
    length = min(length, block - ahead);
    float* scale_at = scales + (static_cast<int64_t>(page) * (c.page_size / block) + slot0 / block) * hkv + head;
    const float held = ahead ? *scale_at : 0.f;
    uint8_t* rows = pages + page * page_stride;

    uint4 raw[kHeld];
    float top = 0.f;
    bool all_finite = true;
    const int steps = (length + places - 1) / places;
    auto fetch_steps = [&](int base) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int k = (base + i) * places + place;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (base + i < steps) raw[i] = fetch(k < length ? first + k : -1);
      }
    };
#pragma unroll 1
    for (int base = 0; base < steps; base += kHeld) {
      fetch_steps(base);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (base + i >= steps) break;
        const int k = (base + i) * places + place;
        float v[8];
        turned(raw[i], k < length ? first + k : -1, pos0 + k, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = fabsf(v[e]);
          if (m <= FLT_MAX) top = fmaxf(top, m);
          else all_finite = false;
        }
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const float need = block_scale(top), old = held > 0.f && held <= FLT_MAX ? held : 0.f, scale = fmaxf(need, old);
    if (ahead && old < scale) {  // what the block holds already
      const float by = old / scale;
      for (int k = place; k < ahead; k += places) {
        if (!active) continue;
        uint2* at = reinterpret_cast<uint2*>(rows + (slot0 - ahead + k) * token_stride + d0);
        const uint2 was = *at;
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((i < 2 ? was.x : was.y) >> (16 * (i & 1))), __NV_E4M3);
          const float2 f = __half22float2(__half2(two));
          v[2 * i] = f.x * by, v[2 * i + 1] = f.y * by;
        }
        *at = make_uint2(e4m3_pack4(v[0], v[1], v[2], v[3]), e4m3_pack4(v[4], v[5], v[6], v[7]));
      }
    }
    const DivideBy divide(scale);
#pragma unroll 1
    for (int base = 0; base < steps; base += kHeld) {
      if (steps > kHeld) fetch_steps(base);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (base + i >= steps) break;
        const int k = (base + i) * places + place;
        float v[8];
        turned(raw[i], k < length ? first + k : -1, pos0 + k, v);
        divide(v, all_finite ? top : INFINITY);
        if (k < length && active) store_8(reinterpret_cast<__nv_fp8_e4m3*>(rows + (slot0 + k) * token_stride + d0), v);
      }
    }
    if (lane == 0 && scale != held) *scale_at = scale;
  }
}

template <typename T>
int launch_blocks(const BlockArgs& a, cudaStream_t stream) {
  const int items = a.rows.num_q_heads + 2 * a.cache.num_kv_heads;
  TRIS_CUDA(launch_step(paged_kv_append_blocks_kernel<T>, dim3(ceil_div(a.rows.num_tokens, a.chunk), ceil_div(items, kWarps)), dim3(kWarps * 32), 0, stream,
                        programmatic_launch_default(), 1, a));
  return TRIS_OK;
}

}  // namespace

// Arguments have been checked (tris_paged_kv_append).
int append_block_scaled(const TrisPagedKv& c, const TrisPagedAppend& r, int rotary_dim, cudaStream_t stream) {
  BlockArgs a{c, r};
  a.rows.rotary_dim = rotary_dim;
  a.lanes = 2;
  while (8 * a.lanes < c.head_dim) a.lanes *= 2;
  a.wide = (!r.q_out || aligned_to(r.q_out, 16)) && (!r.k_out || aligned_to(r.k_out, 16));
  const void* src[3] = {r.num_q_heads ? r.q : nullptr, r.k, r.v};
  const int64_t strides[3][2] = {{r.q_token_stride, r.q_head_stride}, {r.k_token_stride, r.k_head_stride}, {r.v_token_stride, r.v_head_stride}};
  for (int i = 0; i < 3; ++i)
    if (src[i]) a.wide = a.wide && aligned_to(src[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0;
  a.wide_tables = aligned_to(r.cos, 16) && aligned_to(r.sin, 16) && rotary_dim / 2 % 4 == 0;
  // a token to a warp where there are few (a decode step), 16 where there are many
  const int64_t items = r.num_q_heads + 2 * c.num_kv_heads;
  a.chunk = r.num_tokens * items <= 64 * static_cast<int64_t>(sm_count()) ? 1 : 16;
  TRIS_REQUIRE(items <= 65535 * kWarps, TRIS_ERR_UNSUPPORTED, "paged_kv_append: too many heads");
  return r.dtype == TRIS_DTYPE_F16 ? launch_blocks<__half>(a, stream) : launch_blocks<__nv_bfloat16>(a, stream);
}

}  // namespace tris
