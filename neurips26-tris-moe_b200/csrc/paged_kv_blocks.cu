// New keys and values on their way into a paged cache in e4m3 with a scale for each block of tokens and head, rotated by their positions.
//
// A block's scale is the smallest power of two by which its numbers stay within 448.  A token that needs a larger one than its block has gives the block a
// new scale, and the block's tokens ahead of it are read and written once more; between powers of two that shifts exponents, so nothing is lost by it
// (but for what becomes smaller than e4m3 can be), however often it happens.  Bound by bytes for prompts, by the chain position -> page -> scale -> store for
// a decode step.
//
// Tokens that follow one another in a block are a run.  A CTA has the rows of some neighbouring tokens, whole runs that begin among its 16 tokens, and some heads: a thread has the same 16 dimensions
// of its row for one head after the other - two chunks of eight that rotate together - so that its cosines and sines are read once.  A head is rotated, its rows' largest
// magnitudes meet in shared memory, and while they do the next head's are on their way.  A run longer than a CTA's rows is read twice, the second time from L2.
//
// 32/8 heads of 128 in bf16, blocks of 16 tokens, replayed: one token 5.1 us, 64 sequences' 5.7 (half of the slots free: 6.0), a prompt of 512 tokens 6.9, of 2048 14, 4 of 2047 55 to 60 (165 MB, 2.8 TB/s:
// 270 instructions for the 16 dimensions that a lane reads, at 20 warps an SM and 45 % of the issue slots, so latency holds the rest back).  Blocks of more than 16 tokens take a CTA a run, one window after the
// other: 4 of 2047 tokens of 16/16 heads 58 us with blocks of 16, 120, 137 and 246 with 32, 64 and 128.  A decode step of 64 sequences whose blocks all get a larger scale, with some 8 tokens to bring along, takes 20 us.  Two heads at a time, 8.2 for one token and 59 for 4 of 2047; a warp for each run and head, which had the
// rows' cosines to read for every head, 75.
#include <float.h>

#include "block_runs.cuh"
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kWindow = 16;  // rows of a CTA

struct BlockArgs {
  TrisPagedKv cache;
  TrisPagedAppend rows;
  int lanes;        // that have a row, 16 dimensions each: a power of two from 2 to 16
  int page_shift;   // log2(page_size), or -1
  int block_mask;   // scale_tokens - 1 where that is a power of two, or -1
  int page_scales;  // scales of a page and head
};

// Which pairs of dimensions rotate together, and whether eight elements and four cosines can be read, and eight results written, at once: (i, i + half) with
// half a multiple of 8; (2 i, 2 i + 1); and whatever else there is.
enum class Form { kHalves, kPairs, kAny };

// The smallest power of two s with top <= 448 s, from 2^-64 to 2^64.
__device__ __forceinline__ float block_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(min(max(e, 127 - 64), 127 + 64)) << 23);
}

// grid (windows of tokens, shares of the heads), kWindow * L threads.
// L: lanes that have a row, 16 dimensions each.
template <typename T, Form F, int L>
__global__ void __launch_bounds__(kWindow * L, L == 16 ? 3 : L == 8 ? 6 : 12) paged_kv_append_blocks_kernel(const __grid_constant__ BlockArgs a) {
  __shared__ __align__(16) float tops[2][kWindow];  // largest magnitude of every row; two turns
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedAppend& r = a.rows;
  const TrisPagedKv& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 31, row = tid / L, u = tid % L;
  constexpr int R = kWindow;
  const int hq = r.num_q_heads, hkv = c.num_kv_heads, D = c.head_dim, rot = r.rotary_dim, half = rot / 2, block = c.scale_tokens;
  const int64_t room = min(static_cast<int64_t>(c.table_width) * c.page_size, static_cast<int64_t>(0x7FFFFFFF));  // positions are 32-bit numbers from here on
  const bool active = 16 * u < D;
  // this thread's two chunks of eight dimensions
  const bool pairs_up = F == Form::kHalves && u < half / 8;
  const int c0 = pairs_up ? u : 2 * u, c1 = pairs_up ? u + half / 8 : 2 * u + 1;

  auto position = [&](int t) -> int64_t { return r.positions_are_64bit ? reinterpret_cast<const int64_t*>(r.positions)[t] : reinterpret_cast<const int32_t*>(r.positions)[t]; };
  auto in_block = [&](int pos) { return a.block_mask >= 0 ? pos & a.block_mask : pos % block; };  // pages are whole blocks
  auto outside = [&](int64_t pos) { return pos < 0 || pos >= room; };
  // Which of 32 tokens, of which a window has 16, begin runs: those that do not go on, inside a block, where the token before them in the call is.  And which of these are refused, as
  // the call's tokens ahead of them, padding aside, are in the same block: two runs of one block would both bring it to a new scale.
  uint32_t refused = 0;
  auto beginnings = [&](int w) {
    const int t = w + lane;
    bool begins = true, again = false, hidden = false, valid = false;
    int seq = 0, at_block = 0;  // of a token that has a place: its sequence and its block's first position
    if (t < r.num_tokens && t > 0 && r.sequences) {
      const int64_t pos = position(t), before = position(t - 1);
      seq = r.sequences[t];
      const bool same = r.sequences[t - 1] == seq;
      if (!outside(pos)) {
        const int at = in_block(static_cast<int>(pos));
        valid = true;
        at_block = static_cast<int>(pos) - at;
        begins = at == 0 || before != pos - 1 || !same;
        hidden = at && outside(before);
        again = begins && same && !outside(before) && before - in_block(static_cast<int>(before)) == at_block;
      }
    }
    if (__any_sync(0xFFFFFFFFu, hidden)) {  // tokens inside a block behind padding: what is ahead of that, among these 32 or, for the first of them, wherever it is
      const uint32_t ahead = __ballot_sync(0xFFFFFFFFu, valid) & ((1u << lane) - 1);
      const int from = ahead ? highest_bit(ahead) : 0;
      const int ahead_seq = __shfl_sync(0xFFFFFFFFu, seq, from), ahead_block = __shfl_sync(0xFFFFFFFFu, at_block, from);  // (by all lanes, whatever is compared)
      if (hidden && ahead) again = ahead_seq == seq && ahead_block == at_block;
      const uint32_t ask = __ballot_sync(0xFFFFFFFFu, hidden && !ahead);  // one at most
      if (ask) {
        const int whose = lowest_bit(ask), want_seq = __shfl_sync(0xFFFFFFFFu, seq, whose), want_block = __shfl_sync(0xFFFFFFFFu, at_block, whose);
        uint32_t found = 0;
#pragma unroll 1
        for (int t0 = w + whose - 2; !found; t0 -= 32) {
          const int other = t0 - lane;
          const int64_t pos = other >= 0 ? position(other) : 0;
          found = __ballot_sync(0xFFFFFFFFu, other < 0 || !outside(pos));
          const bool here = found && lane == lowest_bit(found) && other >= 0 && r.sequences[other] == want_seq && pos - in_block(static_cast<int>(pos)) == want_block;
          if (__any_sync(0xFFFFFFFFu, here) && lane == whose) again = true;
        }
      }
    }
    refused = __ballot_sync(0xFFFFFFFFu, again);
    return __ballot_sync(0xFFFFFFFFu, begins);
  };

  // What a thread knows of its row's token.
  int t = 0, pos = 0, page = 0;
  bool placed = false, turns = false;  // whether it goes to the cache, and out as something else than zeros
  float cs[8], sn[8];
  auto enter = [&](int token, bool there, bool again) {
    t = token;
    placed = turns = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
    if (!there) return;
    const int64_t p = position(t);
    const int seq = r.sequences ? r.sequences[t] : t;
    turns = p >= 0 && (!r.cos || p < r.max_positions);
    pos = static_cast<int>(min(p, static_cast<int64_t>(0x7FFFFFFF)));
    if (turns && rot && active && (F == Form::kHalves ? pairs_up : F == Form::kPairs)) {
      const int64_t table = p * half;
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // kHalves: the eight frequencies of both chunks; kPairs: four of each
        const int f = F == Form::kHalves ? 8 * c0 + 4 * k : 4 * (c0 + k);
        if (f >= half) break;
        const float4 x = *reinterpret_cast<const float4*>(r.cos + table + f), y = *reinterpret_cast<const float4*>(r.sin + table + f);
        cs[4 * k] = x.x, cs[4 * k + 1] = x.y, cs[4 * k + 2] = x.z, cs[4 * k + 3] = x.w;
        sn[4 * k] = y.x, sn[4 * k + 1] = y.y, sn[4 * k + 2] = y.z, sn[4 * k + 3] = y.w;
      }
    }
    if (p < 0) return;
    bool fits = seq >= 0 && seq < c.num_sequences && p < room;
    if (fits) {
      page = c.block_table[seq * c.table_stride + (a.page_shift >= 0 ? pos >> a.page_shift : pos / c.page_size)];
      fits = page >= 0 && page < c.num_pages;
    }
    placed = fits && turns && !again;
    if (!placed && c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
  };

  struct Source {
    const T* row;    // this thread's, of some head
    int64_t stride;  // to the next head
  };
  auto source = [&](int kind, int head) {  // 0: queries, 1: keys, 2: values
    const int64_t stride = kind == 0 ? r.q_head_stride : kind == 1 ? r.k_head_stride : r.v_head_stride;
    return Source{static_cast<const T*>(kind == 0 ? r.q : kind == 1 ? r.k : r.v) + t * (kind == 0 ? r.q_token_stride : kind == 1 ? r.k_token_stride : r.v_token_stride) + head * stride, stride};
  };
  auto fetch = [&](const T* p, uint4 (&raw)[2]) {
    raw[0] = raw[1] = make_uint4(0, 0, 0, 0);
    if (!turns || !active) return;
    if constexpr (F != Form::kAny) {
      raw[0] = *reinterpret_cast<const uint4*>(p + 8 * c0);
      raw[1] = *reinterpret_cast<const uint4*>(p + 8 * c1);
    } else {
      const uint16_t* e = reinterpret_cast<const uint16_t*>(p) + 16 * u;
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = e[2 * k] | (static_cast<uint32_t>(e[2 * k + 1]) << 16);
      raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
      raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  };
  auto rotate = [&](const T* p, float (&x)[8], float (&y)[8]) {
    if (!rot) return;
    if constexpr (F == Form::kHalves) {
      if (pairs_up) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float p = x[k], q = y[k];
          x[k] = p * cs[k] - q * sn[k];
          y[k] = q * cs[k] + p * sn[k];
        }
      }
    } else if constexpr (F == Form::kPairs) {
      // (dimensions behind the rotated ones stay as they are: by a cosine of 1 and a sine of 0 an infinity would spoil its neighbour)
      if (8 * c0 < rot) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = x[2 * k], q = x[2 * k + 1];
          x[2 * k] = p * cs[k] - q * sn[k];
          x[2 * k + 1] = q * cs[k] + p * sn[k];
        }
      }
      if (8 * c1 < rot) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = y[2 * k], q = y[2 * k + 1];
          y[2 * k] = p * cs[4 + k] - q * sn[4 + k];
          y[2 * k + 1] = q * cs[4 + k] + p * sn[4 + k];
        }
      }
    } else {
      if (!turns || !active) return;
      const float *cr = r.cos + static_cast<int64_t>(pos) * half, *sr = r.sin + static_cast<int64_t>(pos) * half;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int d = 16 * u + k;
        if (d >= rot) break;
        const bool up = r.interleaved ? d & 1 : d >= half;
        const int f = r.interleaved ? d / 2 : up ? d - half : d, with = r.interleaved ? d ^ 1 : up ? d - half : d + half;
        const float other = to_float(p[with]) * sr[f];
        float& v = k < 8 ? x[k & 7] : y[k & 7];
        v = v * cr[f] + (up ? other : -other);
      }
    }
  };
  auto put_row = [&](void* out, int heads, int head, const float (&x)[8], const float (&y)[8]) {  // of q_out or k_out
    if (!active) return;
    T* p = static_cast<T*>(out) + (static_cast<int64_t>(t) * heads + head) * D;
    if constexpr (F != Form::kAny) {
      store_8(p + 8 * c0, x);
      store_8(p + 8 * c1, y);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        store_float(p + 16 * u + k, x[k]);
        store_float(p + 16 * u + 8 + k, y[k]);
      }
    }
  };
  auto row_top = [&](const float (&x)[8], const float (&y)[8], bool finite) {  // over the row's lanes
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      top = fmaxf(top, !finite || fabsf(x[k]) <= FLT_MAX ? fabsf(x[k]) : 0.f);
      top = fmaxf(top, !finite || fabsf(y[k]) <= FLT_MAX ? fabsf(y[k]) : 0.f);
    }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    return top;
  };
  // Where a block of a head's keys or values lies: its first token's row, and its scale; both for the next head, too.
  struct Place {
    uint8_t* row;
    float* scale;
    int64_t token_stride, head_stride;
  };
  auto place_of = [&](bool keys, int head) {  // of the block that this thread's row is in
    const int slot = a.page_shift >= 0 ? pos & (c.page_size - 1) : pos % c.page_size, at = in_block(slot);
    Place to;
    to.token_stride = keys ? c.k_token_stride : c.v_token_stride;
    to.head_stride = keys ? c.k_head_stride : c.v_head_stride;
    to.row = static_cast<uint8_t*>(keys ? c.k_pages : c.v_pages) + page * (keys ? c.k_page_stride : c.v_page_stride) + (slot - at) * to.token_stride + head * to.head_stride;
    to.scale = const_cast<float*>(keys ? c.k_scale : c.v_scale) + (static_cast<int64_t>(page) * a.page_scales + (slot - at) / block) * hkv + head;
    return to;
  };
  // The block's tokens ahead of the run are brought to its new scale, by the run's rows in turn.
  auto bring_along = [&](uint8_t* rows, int64_t stride, int ahead, int from, int step, float by) {
#pragma unroll 1
    for (int k = from; k < ahead; k += step) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        uint2* at = reinterpret_cast<uint2*>(rows + k * stride + 8 * (h ? c1 : c0));
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
  };
  auto known = [](float held) { return held > 0.f && held <= FLT_MAX ? held : 0.f; };
  auto store_row = [&](uint8_t* p, float scale, float (&x)[8], float (&y)[8]) {
    // x / scale: by a power of two, which a scale is unless the caller has put in another, the product with its reciprocal
    const uint32_t bits = __float_as_uint(scale);
    if ((bits & 0x7FFFFFu) == 0) {
      const float up = __uint_as_float((254u << 23) - bits);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= up, y[k] *= up;
    } else {
      const DivideBy divide(scale);
      divide(x, INFINITY);
      divide(y, INFINITY);
    }
    store_8(reinterpret_cast<__nv_fp8_e4m3*>(p + 8 * c0), x);
    store_8(reinterpret_cast<__nv_fp8_e4m3*>(p + 8 * c1), y);
  };

  const int share = blockIdx.y, shares = gridDim.y;
  auto queries = [&](bool there) {
    if (share >= hq) return;
    Source src = source(0, share);
    uint4 next[2];
    fetch(src.row, next);
#pragma unroll 1
    for (int h = share; h < hq; h += shares) {
      float x[8], y[8];
      unpack_8<T>(next[0], x);
      unpack_8<T>(next[1], y);
      const T* now = src.row;
      src.row += shares * src.stride;
      if (h + shares < hq) fetch(src.row, next);
      rotate(now, x, y);
      if (there) put_row(r.q_out, hq, h, x, y);
    }
  };

  const int end = min((static_cast<int>(blockIdx.x) + 1) * R, r.num_tokens);
  int w = blockIdx.x * R, turn = 0;
  uint32_t starts = beginnings(w);
  if (!(starts & ((1u << R) - 1))) return;  // all of these tokens belong to a run that begins ahead of them
  w += lowest_bit(starts);
  refused >>= lowest_bit(starts);
  starts >>= lowest_bit(starts);
#pragma unroll 1
  while (w < end) {
    const int count = tokens_of_whole_runs(starts, end - w, R);
    if (count) {
      const int first = highest_bit(starts & ((2u << row) - 1));  // of this row's run
      const int last = min(row + __ffs(starts >> (row + 1)), count);  // behind it; a run begins at row `count`
      const bool there = row < count && w + row < r.num_tokens;
      enter(min(w + row, r.num_tokens - 1), there, (refused >> first) & 1);
      queries(there);
      const int ahead = in_block(pos) - (row - first);  // tokens of the block ahead of the run
      const bool whole = first == 0 && last == R;
      const int sharers = r.cos ? min(last - first, r.max_positions - (pos - (row - first))) : last - first;  // rows of the run that have a place
#pragma unroll 1
      for (int kind = 1; kind <= 2 && share < hkv; ++kind) {
        Source src = source(kind, share);
        Place to = place_of(kind == 1, share);
        const int64_t own_row = in_block(pos) * to.token_stride;
        uint4 next[2];
        fetch(src.row, next);
#pragma unroll 1
        for (int h = share; h < hkv; h += shares, turn ^= 1) {
          float x[8], y[8];
          unpack_8<T>(next[0], x);
          unpack_8<T>(next[1], y);
          if (kind == 1) rotate(src.row, x, y);
          const float held = placed && ahead > 0 ? *to.scale : 0.f;
          const float top = row_top(x, y, false);
          if (u == 0) tops[turn][row] = placed ? top : 0.f;
          src.row += shares * src.stride;
          if (h + shares < hkv) fetch(src.row, next);
          if (__syncthreads_or(placed && top == INFINITY)) {  // rare: the largest of the finite ones alone
            const float finite = row_top(x, y, true);
            if (u == 0) tops[turn][row] = placed ? finite : 0.f;
            __syncthreads();
          }
          float all = 0.f;
          if (whole) {
#pragma unroll
            for (int n = 0; n < R; n += 4) {
              const float4 m = *reinterpret_cast<const float4*>(&tops[turn][n]);
              all = fmaxf(fmaxf(fmaxf(all, m.x), fmaxf(m.y, m.z)), m.w);
            }
          } else {
            for (int n = first; n < last; ++n) all = fmaxf(all, tops[turn][n]);
          }
          if (kind == 1 && r.k_out && there) put_row(r.k_out, hkv, h, x, y);
          if (placed && active) {
            const float old = known(held), scale = fmaxf(block_scale(all), old);
            if (ahead > 0 && old < scale) bring_along(to.row, to.token_stride, ahead, row - first, sharers, old / scale);
            store_row(to.row + own_row, scale, x, y);
            if (row == first && u == 0 && scale != held) *to.scale = scale;
          }
          to.row += shares * to.head_stride;
          to.scale += shares;
        }
      }
      w += count;
    } else {
      // one run, longer than a window: its length first
      const bool again = refused & 1;
      int length = R;
      for (;;) {
        const uint32_t more = beginnings(w + length);
        length += more ? __ffs(more) - 1 : 32;
        if (more) break;
      }
      for (int at = 0; at < length; at += R) {
        enter(w + min(at + row, length - 1), at + row < length, again);
        queries(at + row < length);
      }
#pragma unroll 1
      for (int item = blockIdx.y; item < 2 * hkv; item += gridDim.y, turn ^= 1) {  // one head at a time
        const bool keys = item < hkv;
        const int head = keys ? item : item - hkv;
        float most = 0.f, scale = 0.f;
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
          for (int at = 0; at < length; at += R) {
            const bool there = at + row < length;
            enter(w + min(at + row, length - 1), there, again);
            uint4 raw[2];
            float x[8], y[8];
            const T* from = source(keys ? 1 : 2, head).row;
            fetch(from, raw);
            unpack_8<T>(raw[0], x);
            unpack_8<T>(raw[1], y);
            if (keys) rotate(from, x, y);
            if (pass == 0) {
              const float top = row_top(x, y, true);
              if (placed) most = fmaxf(most, top);
            } else {
              if (keys && r.k_out && there) put_row(r.k_out, hkv, head, x, y);
              if (placed && active) {
                const Place to = place_of(keys, head);
                store_row(to.row + in_block(pos) * to.token_stride, scale, x, y);
              }
            }
          }
          if (pass == 1) break;
          enter(w, true, again);  // the run's first token, for all
          if (u == 0) tops[turn][row] = most;
          __syncthreads();
          float all = 0.f, held = 0.f;
          for (int n = 0; n < R; ++n) all = fmaxf(all, tops[turn][n]);
          if (placed) {
            const int ahead = in_block(pos);
            const Place to = place_of(keys, head);
            held = ahead ? *to.scale : 0.f;
            const float old = known(held);
            scale = fmaxf(block_scale(all), old);
            if (active && ahead && old < scale) bring_along(to.row, to.token_stride, ahead, row, R, old / scale);
          }
          __syncthreads();  // all have read the scale that is written now
          if (placed && tid == 0 && scale != held) *place_of(keys, head).scale = scale;
        }
      }
      w += length;
    }
    if (w < end) starts = beginnings(w);
  }
}

template <typename T, Form F>
int launch_blocks(const BlockArgs& a, cudaStream_t stream) {
  const int heads = a.rows.num_q_heads > a.cache.num_kv_heads ? a.rows.num_q_heads : a.cache.num_kv_heads;
  // CTAs that share a window's heads: one for each head where there are few windows, else until a thread has kWalk heads of queries, keys and values each.  us, the first and the
  // second: one token 5.0 and 5.6, 512 tokens 6.8 and 7.1, 1024 10.0 and 8.4, 8188 77 and 60.  (A walk of 2 heads 62 for 8188, of 8 heads 64.)
  constexpr int kWalk = 4;
  const int64_t windows = (static_cast<int64_t>(a.rows.num_tokens) + kWindow - 1) / kWindow;
  const int shares = windows * heads <= 8 * static_cast<int64_t>(sm_count()) ? heads : ceil_div(heads, kWalk);
  TRIS_REQUIRE(shares <= 65535, TRIS_ERR_UNSUPPORTED, "paged_kv_append: too many heads");
  auto kernel = a.lanes == 2 ? paged_kv_append_blocks_kernel<T, F, 2> : a.lanes == 4 ? paged_kv_append_blocks_kernel<T, F, 4> : a.lanes == 8 ? paged_kv_append_blocks_kernel<T, F, 8>
                                                                                                                                              : paged_kv_append_blocks_kernel<T, F, 16>;
  TRIS_CUDA(launch_step(kernel, dim3(static_cast<unsigned>(windows), shares), dim3(kWindow * a.lanes), 0, stream, programmatic_launch_default(), 1, a));
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
  TRIS_REQUIRE(r.num_tokens <= 1 << 30, TRIS_ERR_UNSUPPORTED, "paged_kv_append: too many tokens in one call");
  TRIS_REQUIRE(c.k_scale != c.v_scale || c.num_pages == 0, TRIS_ERR_INVALID_ARG, "paged_kv_append: keys and values with the same scales of blocks");
  BlockArgs a{c, r};
  a.rows.rotary_dim = rotary_dim;
  a.page_shift = a.block_mask = -1;
  for (int i = 0; i < 31; ++i) {
    if (c.page_size == 1 << i) a.page_shift = i;
    if (c.scale_tokens == 1 << i) a.block_mask = c.scale_tokens - 1;
  }
  a.page_scales = c.page_size / c.scale_tokens;
  a.lanes = 2;
  while (16 * a.lanes < c.head_dim) a.lanes *= 2;
  bool wide = (!r.q_out || aligned_to(r.q_out, 16)) && (!r.k_out || aligned_to(r.k_out, 16)) && aligned_to(r.cos, 16) && aligned_to(r.sin, 16);
  const void* src[3] = {r.num_q_heads ? r.q : nullptr, r.k, r.v};
  const int64_t strides[3][2] = {{r.q_token_stride, r.q_head_stride}, {r.k_token_stride, r.k_head_stride}, {r.v_token_stride, r.v_head_stride}};
  for (int i = 0; i < 3; ++i)
    if (src[i]) wide = wide && aligned_to(src[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0;
  const Form form = wide && rotary_dim % (r.interleaved ? 8 : 16) == 0 ? (r.interleaved ? Form::kPairs : Form::kHalves) : Form::kAny;
  return r.dtype == TRIS_DTYPE_F16 ? launch_blocks<__half>(a, form, stream) : launch_blocks<__nv_bfloat16>(a, form, stream);
}

}  // namespace tris
