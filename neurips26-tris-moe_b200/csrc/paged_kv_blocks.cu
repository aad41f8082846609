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
  int shares;       // CTAs that share a chunk's heads
  int page_shift;   // log2(page_size), or -1
  int block_mask;   // scale_tokens - 1 where that is a power of two, or -1
  int page_scales;  // scales of a page and head
  int lanes;        // that have a row, eight dimensions each: a power of two
};

// Which pairs of dimensions rotate together, and whether eight elements and four cosines can be read, and eight results written, at once: (i, i + half) with
// half a multiple of 8, so that the other element is in another lane at the same place; (2 i, 2 i + 1); and whatever else there is.
enum class Form { kHalves, kPairs, kAny };

// The biased exponent of the smallest power of two s with top <= 448 s, from 2^-64 to 2^64.
__device__ __forceinline__ float block_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(min(max(e, 127 - 64), 127 + 64)) << 23);
}

// A warp has some of the heads' rows (queries, keys, values) of one chunk of tokens, and what it needs of the next head is on its way while it does one.  Raw rows
// wait in shared memory, where a lane finds what it has asked for itself; in registers they would cost half of the warps that are resident.
template <typename T, Form F>
__global__ void __launch_bounds__(kWarps * 32, 4) paged_kv_append_blocks_kernel(const __grid_constant__ BlockArgs a) {
  __shared__ uint4 staged[kWarps][2][kHeld][32];
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedAppend& r = a.rows;
  const TrisPagedKv& c = a.cache;
  const int lane = threadIdx.x & 31, hq = r.num_q_heads, hkv = c.num_kv_heads, items = hq + 2 * hkv;
  const int first_item = blockIdx.y * kWarps + (threadIdx.x >> 5), item_step = gridDim.y * kWarps;
  if (first_item >= items) return;
  const int D = c.head_dim, rot = r.rotary_dim, half = rot / 2, block = c.scale_tokens;
  const int64_t room = static_cast<int64_t>(c.table_width) * c.page_size;
  const int t0 = blockIdx.x * a.chunk, t1 = min(r.num_tokens, t0 + a.chunk);

  auto position = [&](int t) -> int64_t { return r.positions_are_64bit ? reinterpret_cast<const int64_t*>(r.positions)[t] : reinterpret_cast<const int32_t*>(r.positions)[t]; };
  auto page_of = [&](int pos) { return a.page_shift >= 0 ? pos >> a.page_shift : pos / c.page_size; };
  auto in_block = [&](int pos) { return a.block_mask >= 0 ? pos & a.block_mask : pos % block; };  // pages are whole blocks
  // Whether token t, which has a place at `pos`, goes on where the token before it in the call is.
  auto follows_at = [&](int t, int64_t pos) {
    return t > 0 && r.sequences && in_block(static_cast<int>(pos)) && position(t - 1) == pos - 1 && r.sequences[t - 1] == r.sequences[t];
  };
  // What a lane knows of token t0 + lane: its position (-1: padding, -2: it has no place), its page, and whether it follows.
  struct Token {
    int pos, page;
    bool follows;
  };
  auto look = [&](int t) {
    Token k{-1, -1, false};
    const int64_t pos = position(t);
    const int seq = r.sequences ? r.sequences[t] : t;
    if (pos < 0) return k;
    bool fits = seq >= 0 && seq < c.num_sequences && pos < room;
    const bool turns = !r.cos || pos < r.max_positions;
    if (fits) {
      k.page = c.block_table[seq * c.table_stride + page_of(static_cast<int>(pos))];
      fits = k.page >= 0 && k.page < c.num_pages;
    }
    if (!fits || !turns) {
      if (c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
      k.pos = turns ? -2 : -1;  // one without a place is still rotated, as long as the tables have its position
      if (turns) k.page = static_cast<int>(min(pos, static_cast<int64_t>(0x7FFFFFFF)));
      return k;
    }
    k.pos = static_cast<int>(pos);
    k.follows = follows_at(t, pos);
    return k;
  };

  const int l = lane % a.lanes, place = lane / a.lanes, places = 32 / a.lanes, d0 = 8 * l;
  const bool active = d0 < D;
  struct Source {
    const T* rows;
    int64_t stride;
    int kind, head;  // 0: queries, 1: keys, 2: values
  };
  auto source = [&](int item) {
    const int kind = item < hq ? 0 : item < hq + hkv ? 1 : 2, head = item - (kind == 0 ? 0 : kind == 1 ? hq : hq + hkv);
    const T* base = static_cast<const T*>(kind == 0 ? r.q : kind == 1 ? r.k : r.v);
    return Source{base + head * (kind == 0 ? r.q_head_stride : kind == 1 ? r.k_head_stride : r.v_head_stride), kind == 0 ? r.q_token_stride : kind == 1 ? r.k_token_stride : r.v_token_stride, kind, head};
  };
  // Rows [from, to) of a source, as many as a buffer holds; a lane has row from + i * places + place at step i.
  auto ask = [&](int buffer, const Source& src, int from, int to) {
    uint4* dst = &staged[threadIdx.x >> 5][buffer][0][lane];
    const T* p = src.rows + static_cast<int64_t>(from + place) * src.stride + d0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (from + i * places >= to) break;
      const bool there = active && from + i * places + place < to;
      if constexpr (F != Form::kAny) {
        cp_async_16(dst + i * 32, there ? p + i * places * src.stride : src.rows, there);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
        const uint16_t* e = reinterpret_cast<const uint16_t*>(p + i * places * src.stride);
        for (int k = 0; there && k < 4; ++k) w[k] = e[2 * k] | (static_cast<uint32_t>(e[2 * k + 1]) << 16);
        dst[i * 32] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    cp_async_commit();
  };
  // Step i's eight dimensions of token t at position pos, rotated; zeros where the buffer has no row (t and pos are those of another one then).  By a whole warp.
  const bool turns_here = active && d0 < rot;
  const int partner = !turns_here ? lane : d0 < half ? lane + half / 8 : lane - half / 8, f0 = F == Form::kPairs ? d0 / 2 : d0 < half ? d0 : d0 - half;
  const uint32_t flip = d0 < half ? 0x80008000u : 0;  // a cos - b sin, b cos + a sin
  auto turned = [&](const Source& src, int buffer, int i, int t, int pos, float (&v)[8]) {
    const uint4 raw = staged[threadIdx.x >> 5][buffer][i][lane];
    unpack_8<T>(raw, v);
    if (rot == 0) return;
    uint4 pair;
    if constexpr (F == Form::kHalves)
      pair = make_uint4(__shfl_sync(0xFFFFFFFFu, raw.x, partner) ^ flip, __shfl_sync(0xFFFFFFFFu, raw.y, partner) ^ flip, __shfl_sync(0xFFFFFFFFu, raw.z, partner) ^ flip,
                        __shfl_sync(0xFFFFFFFFu, raw.w, partner) ^ flip);
    if (!turns_here) return;
    const int64_t table = static_cast<int64_t>(pos) * half + f0;
    if constexpr (F == Form::kHalves) {
      float other[8];
      unpack_8<T>(pair, other);
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        const float4 x = *reinterpret_cast<const float4*>(r.cos + table + k), y = *reinterpret_cast<const float4*>(r.sin + table + k);
        v[k] = fmaf(v[k], x.x, other[k] * y.x);
        v[k + 1] = fmaf(v[k + 1], x.y, other[k + 1] * y.y);
        v[k + 2] = fmaf(v[k + 2], x.z, other[k + 2] * y.z);
        v[k + 3] = fmaf(v[k + 3], x.w, other[k + 3] * y.w);
      }
    } else if constexpr (F == Form::kPairs) {
      const float4 x = *reinterpret_cast<const float4*>(r.cos + table), y = *reinterpret_cast<const float4*>(r.sin + table);
      const float cs[4] = {x.x, x.y, x.z, x.w}, sn[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float p = v[2 * k], q = v[2 * k + 1];
        v[2 * k] = p * cs[k] - q * sn[k];
        v[2 * k + 1] = q * cs[k] + p * sn[k];
      }
    } else {
      const T* p = src.rows + t * src.stride;
      const float *cr = r.cos + static_cast<int64_t>(pos) * half, *sr = r.sin + static_cast<int64_t>(pos) * half;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int d = d0 + k;
        if (d >= rot) break;
        const bool up = r.interleaved ? d & 1 : d >= half;
        const int f = r.interleaved ? d / 2 : up ? d - half : d, with = r.interleaved ? d ^ 1 : up ? d - half : d + half;
        const float x = to_float(p[with]) * sr[f];
        v[k] = v[k] * cr[f] + (up ? x : -x);
      }
    }
  };
  auto put_row = [&](void* out, int64_t row, const float (&v)[8]) {  // of q_out or k_out
    if (!active) return;
    T* p = static_cast<T*>(out) + row * D + d0;
    if constexpr (F != Form::kAny) {
      store_8(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) store_float(p + i, v[i]);
    }
  };

  // Rows that are rotated and go out as they are: queries, and keys that the caller asks for.
  const int goes_out = r.k_out ? hq + hkv : hq;
  const int window = kHeld * places;  // rows of a buffer
  if (first_item < goes_out) ask(0, source(first_item), t0, min(t1, t0 + window));
  Token own{-1, -1, false};
  if (t0 + lane < t1) own = look(t0 + lane);
  int buffer = 0;
#pragma unroll 1
  for (int item = first_item; item < goes_out; item += item_step) {
    const Source src = source(item);
#pragma unroll 1
    for (int from = t0; from < t1; from += window) {
      if (from + window < t1) ask(buffer ^ 1, src, from + window, min(t1, from + 2 * window));
      else if (item + item_step < goes_out) ask(buffer ^ 1, source(item + item_step), t0, min(t1, t0 + window));
      else cp_async_commit();
      cp_async_wait<1>();
#pragma unroll 2
      for (int i = 0; i < kHeld; ++i) {
        if (from + i * places >= t1) break;
        const int t = min(from + i * places + place, t1 - 1);
        const int pos = __shfl_sync(0xFFFFFFFFu, own.pos == -2 ? own.page : own.pos, t - t0);
        float v[8];
        turned(src, buffer, i, t, max(pos, 0), v);
        if (pos < 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.f;
        }
        if (from + i * places + place < t1) put_row(src.kind == 0 ? r.q_out : r.k_out, static_cast<int64_t>(t) * (src.kind == 0 ? hq : hkv) + src.head, v);
      }
      buffer ^= 1;
    }
  }
  // Keys and values.
  const int first_cached = first_item + (first_item < hq ? (hq - first_item + item_step - 1) / item_step * item_step : 0);
  if (first_cached >= items) return;
  const uint32_t placed = __ballot_sync(0xFFFFFFFFu, own.pos >= 0), follows = __ballot_sync(0xFFFFFFFFu, own.follows);
#pragma unroll 1
  for (uint32_t runs = placed & ~follows; runs; runs &= runs - 1) {
    const int lead = __ffs(runs) - 1;
    const int pos0 = __shfl_sync(0xFFFFFFFFu, own.pos, lead), page = __shfl_sync(0xFFFFFFFFu, own.page, lead), first = t0 + lead;
    // its length: tokens that follow, in this chunk and behind it
    const uint32_t behind = lead == 31 ? 0 : ~follows >> (lead + 1);  // (bits behind the chunk's last token are 0 in follows)
    int length = behind ? __ffs(behind) : 32 - lead;
    const int slot0 = pos0 - page_of(pos0) * c.page_size, ahead = in_block(pos0);  // tokens of the block ahead of the run
    const int room_left = block - ahead, most = min(room_left, r.num_tokens - first);
    if (first + length == t1) {
      while (length < most) {
        // the block's next tokens have places where its first one has, but for the rotation's tables
        const int t = first + length + lane, pos = pos0 + length + lane;
        const bool on = length + lane < most && position(t) == pos && (!r.cos || pos < r.max_positions) && follows_at(t, pos);
        const uint32_t more = ~__ballot_sync(0xFFFFFFFFu, on);
        length += more ? __ffs(more) - 1 : 32;
        if (more) break;
      }
    }
    length = min(length, most);
    const int64_t scale_index = (static_cast<int64_t>(page) * a.page_scales + (slot0 - ahead) / block) * hkv;
    const bool whole = length <= window;  // a buffer holds the run
    auto rows_from = [&](int k) { return min(first + length, first + k + window); };
    ask(buffer, source(first_cached), first, rows_from(0));
#pragma unroll 1
    for (int item = first_cached; item < items; item += item_step) {
      const Source src = source(item);
      const bool keys = src.kind == 1;
      float* scale_at = const_cast<float*>(keys ? c.k_scale : c.v_scale) + scale_index + src.head;
      const float held = ahead ? *scale_at : 0.f;
      // Step i of the rows from `base` on.
      float v[kHeld][8];
      auto row_of = [&](int base, int i) { return min(base + i * places + place, length - 1); };
      auto load_window = [&](int base) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          if (base + i * places >= length) break;
          if (keys) turned(src, buffer, i, first + row_of(base, i), pos0 + row_of(base, i), v[i]);
          else unpack_8<T>(staged[threadIdx.x >> 5][buffer][i][lane], v[i]);
        }
      };
      // The largest magnitude, of finite numbers alone where there are others, too.
      auto largest = [&](int base, float top, bool finite) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          if (base + i * places >= length) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, !finite || fabsf(v[i][e]) <= FLT_MAX ? fabsf(v[i][e]) : 0.f);
        }
        return top;
      };
      auto of_all = [&](float top) {
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        return top;
      };
      float top = 0.f;
      if (whole) {
        if (item + item_step < items) ask(buffer ^ 1, source(item + item_step), first, rows_from(0));
        else cp_async_commit();
        cp_async_wait<1>();
        load_window(0);
        top = of_all(largest(0, 0.f, false));
        if (top == INFINITY) top = of_all(largest(0, 0.f, true));
      } else {
#pragma unroll 1
        for (int base = 0; base < length; base += window) {
          if (base) ask(buffer, src, first + base, rows_from(base));
          cp_async_wait<0>();
          load_window(base);
          top = largest(base, top, true);
        }
        top = of_all(top);
      }
      const float need = block_scale(top), old = held > 0.f && held <= FLT_MAX ? held : 0.f, scale = fmaxf(need, old);
      uint8_t* rows = static_cast<uint8_t*>(keys ? c.k_pages : c.v_pages) + src.head * (keys ? c.k_head_stride : c.v_head_stride) + page * (keys ? c.k_page_stride : c.v_page_stride) + d0;
      const int64_t token_stride = keys ? c.k_token_stride : c.v_token_stride;
      if (ahead && old < scale) {  // what the block holds already
        const float by = old / scale;
#pragma unroll 4
        for (int k = place; k < ahead; k += places) {
          if (!active) continue;
          uint2* at = reinterpret_cast<uint2*>(rows + (slot0 - ahead + k) * token_stride);
          const uint2 was = *at;
          float f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((i < 2 ? was.x : was.y) >> (16 * (i & 1))), __NV_E4M3);
            const float2 pair = __half22float2(__half2(two));
            f[2 * i] = pair.x * by, f[2 * i + 1] = pair.y * by;
          }
          *at = make_uint2(e4m3_pack4(f[0], f[1], f[2], f[3]), e4m3_pack4(f[4], f[5], f[6], f[7]));
        }
      }
      // x / scale: by a power of two, which a scale is unless the caller has put in another, the product with its reciprocal
      const uint32_t scale_bits = __float_as_uint(scale);
      const bool shifts = (scale_bits & 0x7FFFFFu) == 0;
      const float up = __uint_as_float((254u << 23) - scale_bits);
#pragma unroll 1
      for (int base = 0; base < length; base += window) {
        if (!whole) {
          ask(buffer, src, first + base, rows_from(base));
          cp_async_wait<0>();
          load_window(base);
        }
        if (!shifts) {
          const DivideBy divide(scale);
#pragma unroll
          for (int i = 0; i < kHeld; ++i) {
            if (base + i * places >= length) break;
            divide(v[i], INFINITY);
          }
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const int k = base + i * places + place;
          if (base + i * places >= length) break;
          if (shifts) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= up;
          }
          if (k < length && active) store_8(reinterpret_cast<__nv_fp8_e4m3*>(rows + (slot0 + k) * token_stride), v[i]);
        }
      }
      if (lane == 0 && scale != held) *scale_at = scale;
      if (whole) buffer ^= 1;
      else if (item + item_step < items) ask(buffer, source(item + item_step), first, rows_from(0));
    }
  }
}

template <typename T, Form F>
int launch_blocks(const BlockArgs& a, cudaStream_t stream) {
  TRIS_CUDA(launch_step(paged_kv_append_blocks_kernel<T, F>, dim3(ceil_div(a.rows.num_tokens, a.chunk), a.shares), dim3(kWarps * 32), 0, stream, programmatic_launch_default(), 1, a));
  return TRIS_OK;
}

template <typename T>
int launch_blocks(const BlockArgs& a, Form form, cudaStream_t stream) {
  return form == Form::kHalves ? launch_blocks<T, Form::kHalves>(a, stream) : form == Form::kPairs ? launch_blocks<T, Form::kPairs>(a, stream) : launch_blocks<T, Form::kAny>(a, stream);
}

}  // namespace

// Arguments have been checked (tris_paged_kv_append).
int append_block_scaled(const TrisPagedKv& c, const TrisPagedAppend& r, int rotary_dim, cudaStream_t stream) {
  TRIS_REQUIRE(r.sequences || r.num_tokens <= c.num_sequences, TRIS_ERR_INVALID_ARG, "paged_kv_append: %d tokens without sequences for a block table of %d", r.num_tokens, c.num_sequences);
  BlockArgs a{c, r};
  a.rows.rotary_dim = rotary_dim;
  a.page_shift = a.block_mask = -1;
  for (int i = 0; i < 31; ++i) {
    if (c.page_size == 1 << i) a.page_shift = i;
    if (c.scale_tokens == 1 << i) a.block_mask = c.scale_tokens - 1;
  }
  a.page_scales = c.page_size / c.scale_tokens;
  a.lanes = 2;
  while (8 * a.lanes < c.head_dim) a.lanes *= 2;
  bool wide = (!r.q_out || aligned_to(r.q_out, 16)) && (!r.k_out || aligned_to(r.k_out, 16)) && aligned_to(r.cos, 16) && aligned_to(r.sin, 16);
  const void* src[3] = {r.num_q_heads ? r.q : nullptr, r.k, r.v};
  const int64_t strides[3][2] = {{r.q_token_stride, r.q_head_stride}, {r.k_token_stride, r.k_head_stride}, {r.v_token_stride, r.v_head_stride}};
  for (int i = 0; i < 3; ++i)
    if (src[i]) wide = wide && aligned_to(src[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0;
  const Form form = wide && rotary_dim % (r.interleaved ? 8 : 16) == 0 ? (r.interleaved ? Form::kPairs : Form::kHalves) : Form::kAny;
  // a token to a warp where there are few (a decode step), 32 where there are many
  const int64_t items = r.num_q_heads + 2 * c.num_kv_heads;
  a.chunk = r.num_tokens * items <= 64 * static_cast<int64_t>(sm_count()) ? 1 : 32;
  // and as many CTAs to a chunk as a warp has kHeads heads
  constexpr int kHeads = 2;
  a.shares = ceil_div(static_cast<int>(items), kWarps * (a.chunk == 1 ? 1 : kHeads));
  TRIS_REQUIRE(items <= 65535 * kWarps, TRIS_ERR_UNSUPPORTED, "paged_kv_append: too many heads");
  return r.dtype == TRIS_DTYPE_F16 ? launch_blocks<__half>(a, form, stream) : launch_blocks<__nv_bfloat16>(a, form, stream);
}

}  // namespace tris
