// Attention of one new token per sequence over a paged cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = scale * q . k_t, m the largest s so far: one pass over keys and values, in which the
// sums are scaled down whenever m grows.  Two such partial results (m, l, o) of different tokens join by the same rule, so a sequence can be cut
// anywhere.  Every cached byte is read once and used for as many query heads as share it: bound by bytes.
//
// Work.  The tokens of every (sequence, key/value head) are cut into blocks of 16, all blocks are numbered through, and each warp of the grid
// takes an equal run of them, whatever sequences it crosses: lengths may differ by any factor, change from one replay of a graph to the next,
// and a single long sequence still occupies every SM.  A warp that has all of a sequence's blocks writes its result; others write partial
// results to the workspace (at most two a warp), which the second kernel joins in the order of the tokens.
//
// One warp's step.  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16: the cached rows are the 16-row operand and the query heads of a group the
// 8 columns, so that a step of 16 tokens costs two MMAs per 16 dimensions with up to 8 heads (with the heads as rows it would cost four, half
// of them zeros).  No operand goes through a transposing load: the order of dimensions inside a product is free as long as both operands have the
// same, so a lane's 16 bytes of a key row are its fragments as they are; of four value rows a lane has the same 8 dimensions, whose pairs of
// tokens are put together by PRMT.  A lane therefore reads from shared memory exactly what it has itself copied there (cp.async): the ring
// of a warp needs no barrier, and serves as a queue of loads in flight instead of registers.
#include <type_traits>

#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kBlock = 16;  // tokens of a step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  TrisPagedKv cache;
  TrisPagedAttention query;
  int group;        // query heads of a key/value head
  int row_tiles;    // tiles of kHeads query heads it takes
  int tile_heads;   // heads of a tile that exist at most
  int page_shift;   // log2(page_size), or -1
  int min_run;      // blocks a warp takes at least
  int workers;      // warps of the grid
  float* part_o;    // [2 * workers][tile_heads][head_dim]
  float* part_ml;   // [2 * workers][tile_heads][2]
};

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_m16n8k16(c, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two e4m3 values as fp16, exact.
__device__ __forceinline__ uint32_t e4m3_to_h2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

struct Span {
  int lo, hi;  // tokens [lo, hi)
  __device__ __forceinline__ int blocks() const { return (hi - lo + kBlock - 1) / kBlock; }
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  const int64_t room = static_cast<int64_t>(a.cache.table_width) * a.cache.page_size;
  const int n = a.query.lengths[b];
  const int hi = n < 0 ? 0 : n > room ? static_cast<int>(room) : n;
  return {a.query.window > 0 && hi > a.query.window ? hi - a.query.window : 0, hi};
}

// Blocks ahead of sequence `stop` (all lanes get the sum); the number of sequences is small and the lengths stay in L1.
__device__ __forceinline__ int64_t blocks_before(const AttnArgs& a, int stop, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < stop; b += 32) sum += span_of(a, b).blocks();
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  return sum * a.cache.num_kv_heads * a.row_tiles;
}
__device__ __forceinline__ int64_t run_length(const AttnArgs& a, int64_t total) {
  const int64_t even = (total + a.workers - 1) / a.workers;
  return even > a.min_run ? even : a.min_run;
}

// Where a warp is in the numbering: block `blk` of `span`, head item `item` (head * row_tiles + tile) of sequence b.
struct Cursor {
  int b, item, blk;
  Span span;
  int blocks;
  __device__ __forceinline__ void enter(const AttnArgs& a, int seq) {
    b = seq;
    item = blk = 0;
    do {
      span = span_of(a, b);
      blocks = span.blocks();
    } while (blocks == 0 && ++b < a.cache.num_sequences);
  }
  __device__ __forceinline__ void next(const AttnArgs& a) {
    if (++blk < blocks) return;
    blk = 0;
    if (++item < a.cache.num_kv_heads * a.row_tiles) return;
    item = 0;
    if (b + 1 < a.cache.num_sequences) enter(a, b + 1);
  }
};

// T: type of q and out.  FP8: e4m3 pages, multiplied as fp16.  DP: head_dim rounded up to 64, 128 or 256.  NT: tiles of 8 query heads.
template <typename T, bool FP8, int DP, int NT>
struct Shape {
  static constexpr int kElems = FP8 ? 16 : 8;                          // of a 16-byte chunk
  static constexpr int kKeyChunks = DP / kElems / 4;                   // of a key row that a lane has
  static constexpr int kValueChunks = DP / kElems / 8 ? DP / kElems / 8 : 1;
  static constexpr int kSlots = 2 * kKeyChunks + 4 * kValueChunks;     // 16-byte pieces of a lane and step
  static constexpr int kStageBytes = kSlots * 512;
  static constexpr int kWarps = kStageBytes >= 16384 ? 4 : 8;
  static constexpr int kStages = 24576 / kStageBytes > 6 ? 6 : (kWarps == 4 ? 49152 : 24576) / kStageBytes;
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  static constexpr int kSteps = DP / 16;                               // K = 16 steps of S
  static constexpr int kDimTiles = kValueChunks * kElems / 2;          // 16-dimension tiles of O
  static constexpr int kHeads = 8 * NT;
};

template <typename T, bool FP8, int DP, int NT>
__global__ void __launch_bounds__(Shape<T, FP8, DP, NT>::kWarps * 32, 1) paged_attention_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<T, FP8, DP, NT>;
  using M = std::conditional_t<FP8, __half, T>;  // type of the products
  constexpr int kElt = FP8 ? 1 : 2;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const TrisPagedKv& c = a.cache;
  pdl_wait();
  pdl_launch_dependents();

  const int worker = warp * gridDim.x + blockIdx.x;  // few blocks: on as many SMs as there are
  const int D = c.head_dim;
  const int per_seq = c.num_kv_heads * a.row_tiles;
  const int64_t total = blocks_before(a, c.num_sequences, lane);
  const int64_t run = run_length(a, total);
  const int64_t first = worker * run;
  if (first >= total) return;
  const int count = static_cast<int>(min(run, total - first));

  Cursor use;
  {  // the sequence that holds block `first`
    int64_t before = 0;
    for (int b0 = 0;; b0 += 32) {
      const int b = b0 + lane;
      const int64_t mine = b < c.num_sequences ? static_cast<int64_t>(span_of(a, b).blocks()) * per_seq : 0;
      int64_t upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += v;
      }
      const uint32_t beyond = __ballot_sync(0xFFFFFFFFu, before + upto > first);
      if (beyond) {
        const int l = __ffs(beyond) - 1;
        const int64_t start = before + __shfl_sync(0xFFFFFFFFu, upto - mine, l);
        use.enter(a, b0 + l);
        use.item = static_cast<int>((first - start) / use.blocks);
        use.blk = static_cast<int>((first - start) % use.blocks);
        break;
      }
      before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }
  bool owns_start = use.blk == 0;  // whether the current item begins in this run

  Cursor load = use;
  int left = count;  // blocks that are not asked for yet
  // Lane l < 16: page of token l of the block that is asked for next.
  auto page_of = [&](const Cursor& cur) {
    const int tok = cur.span.lo + cur.blk * kBlock + (lane & 15);
    if (tok >= cur.span.hi) return -1;
    const int at = a.page_shift >= 0 ? tok >> a.page_shift : tok / c.page_size;
    const int page = c.block_table[cur.b * c.table_stride + at];
    if (page >= 0 && page < c.num_pages) return page;
    if (c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
    return -1;
  };
  int page = page_of(load);
  uint8_t* ring = smem + warp * (S::kStages * S::kStageBytes) + lane * 16;
  auto issue = [&](int stage) {
    if (left > 0) {
      const int tok = load.span.lo + load.blk * kBlock + (lane & 15);
      const int in_page = a.page_shift >= 0 ? tok & (c.page_size - 1) : tok % c.page_size;
      const int head = load.item / a.row_tiles;
      const int64_t k_off = page < 0 ? -1 : (page * c.k_page_stride + in_page * c.k_token_stride + head * c.k_head_stride) * kElt;
      const int64_t v_off = page < 0 ? -1 : (page * c.v_page_stride + in_page * c.v_token_stride + head * c.v_head_stride) * kElt;
      uint8_t* dst = ring + stage * S::kStageBytes;
#pragma unroll
      for (int r = 0; r < 2; ++r) {  // keys g and g + 8: chunks 4 j + t
        const int64_t off = __shfl_sync(0xFFFFFFFFu, k_off, g + 8 * r);
        const uint8_t* src = static_cast<const uint8_t*>(c.k_pages) + (off < 0 ? 0 : off);
#pragma unroll
        for (int j = 0; j < S::kKeyChunks; ++j) {
          const bool ok = off >= 0 && (4 * j + t) * S::kElems < D;
          cp_async_16(dst + (r * S::kKeyChunks + j) * 512, ok ? src + (4 * j + t) * 16 : static_cast<const uint8_t*>(c.k_pages), ok);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // values 2 t, 2 t + 1, 2 t + 8, 2 t + 9: chunks 8 j + g
        const int64_t off = __shfl_sync(0xFFFFFFFFu, v_off, 2 * t + (r & 1) + 8 * (r >> 1));
        const uint8_t* src = static_cast<const uint8_t*>(c.v_pages) + (off < 0 ? 0 : off);
#pragma unroll
        for (int j = 0; j < S::kValueChunks; ++j) {
          const bool ok = off >= 0 && (8 * j + g) * S::kElems < D;
          cp_async_16(dst + (2 * S::kKeyChunks + r * S::kValueChunks + j) * 512, ok ? src + (8 * j + g) * 16 : static_cast<const uint8_t*>(c.v_pages), ok);
        }
      }
      if (--left > 0) {
        load.next(a);
        page = page_of(load);
      }
    }
    cp_async_commit();  // empty groups keep the count of groups in step
  };
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) issue(s);

  uint32_t qf[NT][S::kSteps][2];
  float scale[NT][2];  // of heads 2 t and 2 t + 1 of a tile, to base 2
  float m[NT][2], l[NT][2], acc[S::kDimTiles][NT][4];
  const TrisPagedAttention& query = a.query;

  auto load_query = [&] {
    const int head = use.item / a.row_tiles, tile = use.item % a.row_tiles;
    const float base = query.softmax_scale * kLog2e * (FP8 && c.k_scale ? c.k_scale[head] : 1.f);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = tile * S::kHeads + 8 * n + g;
      const T* src = static_cast<const T*>(query.q) + use.b * query.q_token_stride + (static_cast<int64_t>(head) * a.group + row) * query.q_head_stride;
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < S::kKeyChunks; ++j) {
#pragma unroll
        for (int w = 0; w < S::kElems / 2; ++w) {
          const int d = (4 * j + t) * S::kElems + 2 * w;
          uint32_t v = 0;
          if (row < a.group && d < D) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(src + d);
            v = p[0] | (static_cast<uint32_t>(p[1]) << 16);
          }
          if constexpr (FP8 && !std::is_same_v<T, __half>) {
            const float2 f = Pair<T>::unpack(v);
            top = max_nan(top, max_nan(fabsf(f.x), fabsf(f.y)));
          }
          qf[n][j * (S::kElems / 4) + w / 2][w & 1] = v;
        }
      }
      float up = 1.f;  // bf16 queries against fp16 keys: a power of two brings a row's largest element to [1, 2)
      if constexpr (FP8 && !std::is_same_v<T, __half>) {
        top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const int e = top > 0.f && top < INFINITY ? max(ilogbf(top), -100) : 0;
        up = ldexpf(1.f, e);
        const float down = ldexpf(1.f, -e);
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = Pair<T>::unpack(qf[n][s][i]);
            qf[n][s][i] = Pair<__half>::pack(f.x * down, f.y * down);
          }
      }
      scale[n][0] = base * __shfl_sync(0xFFFFFFFFu, up, 8 * t);
      scale[n][1] = base * __shfl_sync(0xFFFFFFFFu, up, 8 * t + 4);
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < S::kDimTiles; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][n][k] = 0.f;
    }
  };

  auto finish_item = [&](bool owns_end) {
    const int head = use.item / a.row_tiles, tile = use.item % a.row_tiles;
    const bool whole = owns_start && owns_end;
    const int64_t slot = 2 * static_cast<int64_t>(worker) + (owns_start ? 1 : 0);
    const float v_scale = FP8 && c.v_scale ? c.v_scale[head] : 1.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[n][h];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        const int in_tile = 8 * n + 2 * t + h, row = tile * S::kHeads + in_tile;
        if (row >= a.group) continue;
        const int64_t out_row = static_cast<int64_t>(use.b) * query.num_q_heads + head * a.group + row;
        const float inv = whole ? (sum == 0.f ? 0.f : v_scale / sum) : v_scale;
#pragma unroll
        for (int j = 0; j < S::kValueChunks; ++j) {
          const int d0 = (8 * j + g) * S::kElems;
          if (d0 >= D) continue;
#pragma unroll
          for (int q = 0; q < S::kElems / 8; ++q) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[2 * i] = acc[j * (S::kElems / 2) + 4 * q + i][n][h] * inv;
              v[2 * i + 1] = acc[j * (S::kElems / 2) + 4 * q + i][n][2 + h] * inv;
            }
            if (whole) {
              store_8(static_cast<T*>(query.out) + out_row * D + d0 + 8 * q, v);
            } else {
              float4* dst = reinterpret_cast<float4*>(a.part_o + (slot * a.tile_heads + in_tile) * D + d0 + 8 * q);
              dst[0] = make_float4(v[0], v[1], v[2], v[3]);
              dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
        }
        if (g == 0) {
          if (!whole)
            *reinterpret_cast<float2*>(a.part_ml + (slot * a.tile_heads + in_tile) * 2) = make_float2(m[n][h], sum);
          else if (query.lse)
            query.lse[out_row] = sum == 0.f ? -INFINITY : (m[n][h] + log2f(sum)) * kLn2;
        }
      }
  };

  load_query();
  for (int i = 0; i < count; ++i) {
    cp_async_wait<S::kStages - 2>();
    const uint8_t* src = ring + (i % S::kStages) * S::kStageBytes;

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int j = 0; j < S::kKeyChunks; ++j) {
      const uint4 ka = *reinterpret_cast<const uint4*>(src + j * 512), kb = *reinterpret_cast<const uint4*>(src + (S::kKeyChunks + j) * 512);
      const uint32_t x[4] = {ka.x, ka.y, ka.z, ka.w}, y[4] = {kb.x, kb.y, kb.z, kb.w};
      if constexpr (FP8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = e4m3_to_h2(x[w] & 0xFFFF), a2 = e4m3_to_h2(x[w] >> 16), a1 = e4m3_to_h2(y[w] & 0xFFFF), a3 = e4m3_to_h2(y[w] >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<M>(s[n], a0, a1, a2, a3, qf[n][4 * j + w][0], qf[n][4 * j + w][1]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<M>(s[n], x[2 * w], y[2 * w], x[2 * w + 1], y[2 * w + 1], qf[n][2 * j + w][0], qf[n][2 * j + w][1]);
      }
    }

    // tokens g and g + 8 of heads 2 t and 2 t + 1
    const int tok = use.span.lo + use.blk * kBlock + g;
    const bool in0 = tok < use.span.hi, in1 = tok + 8 < use.span.hi;
    uint32_t p[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float old[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[n][h] = in0 ? s[n][h] * scale[n][h] : -INFINITY;
        s[n][2 + h] = in1 ? s[n][2 + h] * scale[n][h] : -INFINITY;
        float top = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        const float now = fmaxf(m[n][h], top);
        const float base = now == -INFINITY ? 0.f : now;  // nothing but -inf so far: weights of 0
        old[h] = exp2f(m[n][h] - base);
        m[n][h] = now;
        s[n][h] = exp2f(s[n][h] - base);
        s[n][2 + h] = exp2f(s[n][2 + h] - base);
        l[n][h] = l[n][h] * old[h] + s[n][h] + s[n][2 + h];
      }
      // the weights as the 8-column operand: pairs of tokens of one head.  Rounded to the values' type, as 16-bit operands are: 2^-9 (bf16) or
      // 2^-12 (fp16) of a weight, independent from token to token; the sum l is of the weights before that
      p[n][0] = transpose_8x8(Pair<M>::pack(s[n][0], s[n][1]));
      p[n][1] = transpose_8x8(Pair<M>::pack(s[n][2], s[n][3]));
#pragma unroll
      for (int k = 0; k < S::kDimTiles; ++k) {
        acc[k][n][0] *= old[0];
        acc[k][n][1] *= old[1];
        acc[k][n][2] *= old[0];
        acc[k][n][3] *= old[1];
      }
    }

    const uint8_t* vals = src + 2 * S::kKeyChunks * 512;
#pragma unroll
    for (int j = 0; j < S::kValueChunks; ++j) {
      uint32_t v[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint4 raw = *reinterpret_cast<const uint4*>(vals + (r * S::kValueChunks + j) * 512);
        v[r][0] = raw.x, v[r][1] = raw.y, v[r][2] = raw.z, v[r][3] = raw.w;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
#pragma unroll
        for (int e = 0; e < (FP8 ? 2 : 1); ++e) {
          uint32_t x[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = FP8 ? e4m3_to_h2(e ? v[r][w] >> 16 : v[r][w] & 0xFFFF) : v[r][w];
          const uint32_t a0 = prmt(x[0], x[1], 0x5410), a1 = prmt(x[0], x[1], 0x7632), a2 = prmt(x[2], x[3], 0x5410), a3 = prmt(x[2], x[3], 0x7632);
          const int tile = FP8 ? j * 8 + 2 * w + e : j * 4 + w;
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<M>(acc[tile][n], a0, a1, a2, a3, p[n][0], p[n][1]);
        }
      }
    }
    issue((i + S::kStages - 1) % S::kStages);

    const bool last = i + 1 == count;
    if (last || use.blk + 1 == use.blocks) {
      finish_item(use.blk + 1 == use.blocks);
      if (!last) {
        use.next(a);
        owns_start = true;
        load_query();
      }
    } else {
      ++use.blk;
    }
  }
  cp_async_wait<0>();
}

// Joins the partial results of one query head of one sequence; zeros where there was nothing to attend to.
constexpr int kJoinThreads = 128;
constexpr int kMaxWorkers = 4096;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ AttnArgs a, int tile_rows) {
  __shared__ float weight[kMaxWorkers];
  __shared__ float red[kJoinThreads / 32][2];
  __shared__ float4 sums[kJoinThreads];
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedKv& c = a.cache;
  const TrisPagedAttention& query = a.query;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y, q_head = blockIdx.x, head = q_head / a.group, row = q_head % a.group;
  const int tile = row / tile_rows, in_tile = row % tile_rows, D = c.head_dim, D4 = D / 4;
  const int64_t out_row = static_cast<int64_t>(b) * query.num_q_heads + q_head;
  const Span span = span_of(a, b);
  const int blocks = span.blocks();
  T* out = static_cast<T*>(query.out) + out_row * D;
  if (query.lengths[b] > span.hi && c.status_dev && q_head == 0 && tid == 0) *c.status_dev = TRIS_ERR_CORRUPT;
  if (blocks == 0) {
    for (int d = tid; d < D; d += kJoinThreads) store_float(out + d, 0.f);
    if (query.lse && tid == 0) query.lse[out_row] = -INFINITY;
    return;
  }
  const int64_t run = run_length(a, blocks_before(a, c.num_sequences, lane));
  const int64_t start = blocks_before(a, b, lane) + static_cast<int64_t>(head * a.row_tiles + tile) * blocks;
  const int w0 = static_cast<int>(start / run), n = static_cast<int>((start + blocks - 1) / run) - w0 + 1;
  if (n == 1) return;  // one warp had all of it
  auto slot = [&](int i) { return (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * a.tile_heads + in_tile; };

  float top = -INFINITY;
  for (int i = tid; i < n; i += kJoinThreads) top = fmaxf(top, a.part_ml[slot(i) * 2]);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  if (lane == 0) red[warp][0] = top;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[w][0]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int i = tid; i < n; i += kJoinThreads) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + slot(i) * 2);
    const float w = exp2f(ml.x - base);
    weight[i] = w;
    sum += w * ml.y;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if (lane == 0) red[warp][1] = sum;
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[w][1];

  // a group of D / 4 threads per partial result; the groups' sums are added in their order
  const int groups = kJoinThreads / D4, grp = tid / D4, col = tid % D4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < groups) {
#pragma unroll 8
    for (int i = grp; i < n; i += groups) {
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + slot(i) * D + 4 * col);
      const float w = weight[i];
      o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
    }
    sums[tid] = o;
  }
  __syncthreads();
  if (tid < D4) {
    for (int k = 1; k < groups; ++k) {
      const float4 v = sums[k * D4 + tid];
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 packed = make_uint2(Pair<T>::pack(o.x * inv, o.y * inv), Pair<T>::pack(o.z * inv, o.w * inv));
    *reinterpret_cast<uint2*>(out + 4 * tid) = packed;
  }
  if (query.lse && tid == 0) query.lse[out_row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

int sm_count() {
  static int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!count[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    count[dev] = n;
  }
  return count[dev];
}

// Tiles of 8 query heads that share a key/value head's pass.  With heads of 256 dimensions the accumulators of two do not fit the registers.
int head_tiles(int group, int head_dim) { return group > 8 && head_dim <= 128 ? 2 : 1; }

size_t part_floats(int workers, int tile_heads, int head_dim) { return 2 * static_cast<size_t>(workers) * tile_heads * (head_dim + 2); }

template <typename T, bool FP8, int DP, int NT>
int launch_attention(AttnArgs& a, cudaStream_t stream) {
  using S = Shape<T, FP8, DP, NT>;
  auto kernel = paged_attention_kernel<T, FP8, DP, NT>;
  TRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
  const TrisPagedKv& c = a.cache;
  const int sms = sm_count();
  TRIS_REQUIRE(sms > 0 && sms * S::kWarps <= kMaxWorkers, TRIS_ERR_CUDA, "paged_decode_attention: no device");
  a.min_run = 1;
  a.workers = sms * S::kWarps;
  a.part_ml = static_cast<float*>(a.query.workspace);
  a.part_o = a.part_ml + 4 * static_cast<size_t>(a.workers) * a.tile_heads;
  const int64_t need = part_floats(a.workers, a.tile_heads, c.head_dim) * 4;
  TRIS_REQUIRE(a.query.workspace && a.query.workspace_bytes >= need, TRIS_ERR_WORKSPACE, "paged_decode_attention: workspace of %lld bytes needed, got %lld",
               static_cast<long long>(need), static_cast<long long>(a.query.workspace_bytes));
  TRIS_CUDA(launch_kernel(kernel, dim3(sms), dim3(S::kWarps * 32), S::kSmem, stream, programmatic_launch_default(), 1, a));
  TRIS_CUDA(launch_kernel(paged_attention_join_kernel<T>, dim3(a.query.num_q_heads, c.num_sequences), dim3(kJoinThreads), 0, stream, true, 1, a, S::kHeads));
  return TRIS_OK;
}
template <typename T, bool FP8>
int launch_shape(AttnArgs& a, cudaStream_t stream) {
  const int d = a.cache.head_dim;
  if (head_tiles(a.group, d) == 2) return d <= 64 ? launch_attention<T, FP8, 64, 2>(a, stream) : launch_attention<T, FP8, 128, 2>(a, stream);
  return d <= 64 ? launch_attention<T, FP8, 64, 1>(a, stream) : d <= 128 ? launch_attention<T, FP8, 128, 1>(a, stream) : launch_attention<T, FP8, 256, 1>(a, stream);
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" size_t tris_paged_decode_attention_workspace_bytes(const TrisPagedKv* cache, int32_t num_q_heads) {
  if (validate_paged_kv(cache, "paged_decode_attention")) return 0;
  if (num_q_heads < 1 || num_q_heads % cache->num_kv_heads) return 0;
  const int group = num_q_heads / cache->num_kv_heads, heads = 8 * head_tiles(group, cache->head_dim);
  const int sms = sm_count();
  return sms > 0 ? part_floats(sms * 8, group < heads ? group : heads, cache->head_dim) * 4 : 0;
}

extern "C" int tris_paged_decode_attention(const TrisPagedKv* cache, const TrisPagedAttention* query, void* stream) {
  if (int st = validate_paged_kv(cache, "paged_decode_attention")) return st;
  TRIS_REQUIRE(query, TRIS_ERR_INVALID_ARG, "paged_decode_attention: null query");
  const TrisPagedKv& c = *cache;
  const TrisPagedAttention& q = *query;
  TRIS_REQUIRE(q.dtype == TRIS_DTYPE_F16 || q.dtype == TRIS_DTYPE_BF16, TRIS_ERR_INVALID_ARG, "paged_decode_attention: queries are fp16 or bf16");
  TRIS_REQUIRE(c.dtype == TRIS_DTYPE_E4M3 || c.dtype == q.dtype, TRIS_ERR_INVALID_ARG, "paged_decode_attention: pages hold the queries' type or e4m3");
  TRIS_REQUIRE(q.num_q_heads >= 1 && q.num_q_heads % c.num_kv_heads == 0, TRIS_ERR_INVALID_ARG, "paged_decode_attention: %d query heads do not share %d key/value heads evenly",
               q.num_q_heads, c.num_kv_heads);
  TRIS_REQUIRE(q.window >= 0, TRIS_ERR_INVALID_ARG, "paged_decode_attention: negative window");
  if (c.num_sequences == 0) return TRIS_OK;
  TRIS_REQUIRE(c.num_sequences <= 65535, TRIS_ERR_UNSUPPORTED, "paged_decode_attention: more than 65535 sequences");
  TRIS_REQUIRE(q.q && q.out && q.lengths, TRIS_ERR_INVALID_ARG, "paged_decode_attention: null q, out or lengths");
  TRIS_REQUIRE(aligned_to(q.out, 16) && aligned_to(q.workspace, 16), TRIS_ERR_INVALID_ARG, "paged_decode_attention: out and workspace must be 16-byte aligned");

  AttnArgs a{};
  a.cache = c;
  a.query = q;
  a.group = q.num_q_heads / c.num_kv_heads;
  const int heads = 8 * head_tiles(a.group, c.head_dim);
  a.row_tiles = ceil_div(a.group, heads);
  a.tile_heads = a.group < heads ? a.group : heads;
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page_size == 1 << s) a.page_shift = s;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool q8 = c.dtype == TRIS_DTYPE_E4M3;
  if (q.dtype == TRIS_DTYPE_F16) return q8 ? launch_shape<__half, true>(a, s) : launch_shape<__half, false>(a, s);
  return q8 ? launch_shape<__nv_bfloat16, true>(a, s) : launch_shape<__nv_bfloat16, false>(a, s);
}
