// Attention of one new token per sequence over a paged cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = scale * q . k_t, m the largest s so far: one pass over keys and values, in which the
// sums are scaled down whenever m grows.  Two such partial results (m, l, o) of different tokens join by the same rule, so a sequence can be cut
// anywhere.  Every cached byte is read once and used for as many query heads as share it: bound by bytes where there are many (64 sequences of 1 to
// 16384 tokens, 32/8 heads of 128 in bf16, 1.8 GB: 290 us, 6.2 TB/s; one of 131071 in fp16 96 us, 5.6), by the chain length - page - rows - join
// where there are few (513 tokens of 16 heads 8 us).  16 sequences of 4096 in 8 bits (heads of 256, 66 MB) take 22 us: of a CTA's 37 800 cycles the eight
// steps of a warp take 21 500, nine tenths of the rate of a copy, the reads ahead of them, which depend on one another, 6 600, and the joins 9 700.
// Scales of blocks (SB) cost a step two more loads; a key's scale is multiplied into its score, a value's into its token's weight - its power of two into the exponent, which
// the largest s counts in, so that neither weights nor sums leave their range:
// 64 sequences of 1 to 16384 tokens of 32/8 heads of 128 in 8 bits with a scale for 32 tokens, 0.9 GB, 182 us.
//
// Work.  Short sequences: a cluster of CTAs has one key/value head of one sequence and cuts its tokens evenly (cluster_size has the rule).
// Long ones: the tokens of every (sequence, key/value head) are cut into blocks of 16, all blocks are numbered through, and each warp of the grid
// takes an equal run of them, whatever sequences it crosses: lengths may differ by any factor, change from one replay of a graph to the next,
// and a single long sequence still occupies every SM.  A warp that has all of an item's blocks writes its result; others leave partial
// results that are joined in the order of the tokens: first those of a CTA's warps in shared memory, then those of a cluster's CTAs over distributed
// shared memory or, of numbered blocks, by a second kernel from the workspace (at most two a CTA).
//
// One warp's step.  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16: the cached rows are the 16-row operand and the query heads of a group the
// 8 columns, so that a step of 16 tokens costs three MMAs per 16 dimensions with up to 8 heads - one for the scores, two for the two parts of a
// weight - (with the heads as rows it would cost six, half of them zeros).  No operand goes through a transposing load: the order of dimensions
// inside a product is free as long as both operands have the same, so a lane's 16 bytes of a key row are its fragments as they are; of four value
// rows a lane has the same 8 dimensions, whose pairs of tokens are put together by PRMT.  A step's MMAs take a seventh of the time its bytes take (heads of 128: 24 at two cycles of an SM, 8 KB at 23 bytes a
// cycle), so nothing waits for the tensor pipe; tcgen05 tiles have 128 rows and their second operand in shared memory.  Each warp has a ring of its
// own in shared memory, filled by cp.async, and meets no other warp before it is done.
#include <type_traits>

#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kBlock = 16;  // tokens of a step
constexpr int kWarps = 4;   // of a CTA (W); 2 for many very short sequences
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  TrisPagedKv cache;
  TrisPagedAttention query;
  int group;        // query heads of a key/value head
  int row_tiles;    // tiles of kHeads query heads it takes
  int tile_heads;   // heads of a tile that exist at most
  int page_shift;   // log2(page_size), or -1
  int page_blocks;  // whether a block of 16 tokens never crosses a page
  int wide_query;   // whether q's heads start on 16-byte boundaries
  int cluster;      // CTAs that share one item (a sequence's key/value head), or 0: the work is numbered through and cut evenly
  int ctas;         // of the first kernel
  int resident;     // of them, at one time
  int rows_together;  // whether a head's rows in a page are side by side
  int scale_shift;    // log2 of the tokens of a scale, or -1
  int page_scales;    // scales of a page and head
  float* part_o;    // [2 * ctas][tile_heads][head_dim]
  float* part_ml;   // [2 * ctas][tile_heads][2]
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
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return h;
}
__device__ __forceinline__ void cp_async_16_at(uint32_t dst, const void* src, int bytes) {  // bytes: 16, or 0 for zeros
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_4_at(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 2^x; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two weights as sums of two 16-bit numbers: off by 2^-16 (bf16) or 2^-21 (fp16) of a weight, where one number is off by 2^-9 or 2^-12 - as much as the
// result's own rounding, but for results in bf16 over 8-bit pages, whose weights are single fp16 numbers.  (One number and two, us: 32 x 512-768 34.8 and 35.3,
// 1 x 131071 94.3 and 94.5, 64 x 1-16384 287.5 and 288.0, 8 x 8192 of fp16 queries over 8 bits 53.1 and 55.4; 64 x 1-16384 of bf16 over 8 bits 153.4, with two 162.)
// Neither number is zero or negative, so that an infinite value gives an infinity and not NaN: the first is rounded from a little less than the weight.
// (In fp16 that ends with weights of 2^-23, 2^-30 of the largest, whose first number is zero.)
template <typename M>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& most, uint32_t& rest) {
  if constexpr (std::is_same_v<M, __half>) {
    constexpr float kLess = 1.f - 0x1p-10f, kTiny = -0x1p-23f;
    most = Pair<M>::pack(fmaxf(fmaf(a, kLess, kTiny), 0.f), fmaxf(fmaf(b, kLess, kTiny), 0.f));
    const float2 f = Pair<M>::unpack(most);
    rest = Pair<M>::pack(a - f.x, b - f.y);
  } else {
    constexpr float kLess = 1.f - 0x1p-12f;
    const uint32_t x = __float_as_uint(a * kLess), y = __float_as_uint(b * kLess);
    most = prmt(x, y, 0x7632);  // rounded towards zero
    rest = Pair<M>::pack(a - __uint_as_float(x & 0xFFFF0000u), b - __uint_as_float(y & 0xFFFF0000u));
  }
}

constexpr int kMostCluster = 8;

// Tokens [lo, hi) of a sequence; its blocks begin at multiples of kBlock.
struct Span {
  int lo, hi;
  __device__ __forceinline__ int first() const { return lo / kBlock; }
  __device__ __forceinline__ int blocks() const { return hi > lo ? (hi - 1) / kBlock - lo / kBlock + 1 : 0; }
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  const int64_t room = static_cast<int64_t>(a.cache.table_width) * a.cache.page_size;
  const int n = a.query.lengths[b];
  const int hi = n < 0 ? 0 : n > room ? static_cast<int>(room) : n;
  return {a.query.window > 0 && hi > a.query.window ? hi - a.query.window : 0, hi};
}

// Blocks of sequences [32 i, 32 i + 32) up to and with each lane's own, times the items of a sequence.  (Block numbers fit 32 bits: the host sees to it.)
__device__ __forceinline__ int scan_blocks(const AttnArgs& a, int i, int lane, int& mine) {
  const int b = 32 * i + lane;
  mine = b < a.cache.num_sequences ? span_of(a, b).blocks() * (a.cache.num_kv_heads * a.row_tiles) : 0;
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += v;
  }
  return upto;
}
// All blocks, and those ahead of sequence `stop`.
__device__ __forceinline__ int count_blocks(const AttnArgs& a, int stop, int lane, int& before) {
  int total = 0;
  before = 0;
  for (int i = 0; 32 * i < a.cache.num_sequences; ++i) {
    int mine;
    const int upto = scan_blocks(a, i, lane, mine);
    if (stop / 32 == i) before = total + __shfl_sync(0xFFFFFFFFu, upto - mine, stop % 32);
    total += __shfl_sync(0xFFFFFFFFu, upto, 31);
  }
  return total;
}
// Blocks that each warp takes.  The grid has as many CTAs as are resident twice over, so that an SM that is done early takes another one; where that
// would leave a warp fewer than kMinRun blocks, half of them do the work.
constexpr int kMinRun = 64;
__device__ __forceinline__ int run_length(const AttnArgs& a, int total) {
  const unsigned workers = static_cast<unsigned>(a.ctas) * kWarps;
  const unsigned run = (static_cast<unsigned>(total) + workers - 1) / workers;
  if (run >= kMinRun || a.resident >= a.ctas) return run;
  const unsigned fewer = static_cast<unsigned>(a.resident) * kWarps;
  return (static_cast<unsigned>(total) + fewer - 1) / fewer;
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
  __device__ __forceinline__ int token() const { return (span.first() + blk) * kBlock; }
};

// T: type of q and out.  FP8: e4m3 pages, multiplied as fp16.  SB: their scales belong to blocks of tokens and heads, not to heads.  DP: head_dim rounded up to 64, 128 or 256.  NT: tiles of 8 query heads.
// CTAs on an SM, of which some compute while others start or end.  Pages in 8 bits are bound by instructions that wait for one another, so as many as
// the registers allow (13 x 49925 tokens of heads of 64: 44 us with three or four, 64 with two); in 16 bits two with a deep ring (32 x 512-768 of heads
// of 128: 34 us, 41 with three and two stages), and one where a step takes 16 KB.
constexpr int ctas_per_sm(int dp, bool fp8, int nt) {
  if (dp == 64) return fp8 && nt == 1 ? 4 : 3;
  if (dp == 128) return fp8 && nt == 1 ? 3 : 2;
  return fp8 ? 2 : 1;
}
template <typename T, bool FP8, bool SB, int DP, int NT, int W>
struct Shape {
  static constexpr int kElems = FP8 ? 16 : 8;                          // of a 16-byte chunk
  static constexpr int kKeyChunks = DP / kElems / 4;                   // of a key row that a lane has
  static constexpr int kValueElems = FP8 && DP == 64 ? 8 : kElems;     // of a value row that a lane has at a time: eight lanes have the row
  static constexpr int kValueChunks = DP / kValueElems / 8;
  static constexpr int kRowBytes = DP * (FP8 ? 1 : 2);
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kCopyRows = kRowChunks > 32 ? 1 : 32 / kRowChunks;  // rows that 32 lanes copy at once, 16 bytes each
  static constexpr int kTile = kBlock * kRowBytes;                     // 16 rows of keys or of values
  static constexpr int kScales = 2 * kTile;                            // where a stage has its 16 tokens' scales, of keys and of values
  static constexpr int kStageBytes = kScales + (SB ? 2 * kBlock * 4 : 0);
  // Chunk that holds a row's chunk in shared memory, XORed: eight lanes that read together - keys: rows of both parities, four neighbouring
  // chunks; values: rows 2 t, two neighbouring chunks - find eight different 16-byte columns.  (64-byte rows: two lanes a column for values, of which
  // a lane has 8 bytes.)
  static __device__ __forceinline__ constexpr int key_swizzle(int row) { return kRowChunks >= 8 ? (row & 1) << 2 : 0; }
  static __device__ __forceinline__ constexpr int value_swizzle(int row) { return kRowChunks >= 8 ? ((row >> 1) & 3) << 1 : ((row >> 1) & 1) << 1; }
  static constexpr int kSteps = DP / 16;                               // K = 16 steps of S
  static constexpr int kDimTiles = kValueChunks * kValueElems / 2;        // 16-dimension tiles of O
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPieceBytes = kHeads * (DP + 2) * 4;
  static constexpr int kCtasPerSm = ctas_per_sm(DP, FP8, NT) * (kWarps / W);
  static constexpr int kStagesThatFit = ((228 / kCtasPerSm - 1) * 1024 - 256 - (W == kWarps ? W * kPieceBytes : 0)) / (W * kStageBytes);
  static constexpr int kStages = kStagesThatFit > 6 ? 6 : kStagesThatFit;
  static constexpr int kRing = W * kStages * kStageBytes;
  static constexpr int kMostSmem = kRing + (W == kWarps ? W * kPieceBytes : 0);
  static_assert(kStages >= 2 && kPieceBytes <= kStages * kStageBytes, "ring");
};
// A piece of that many heads; all of them start on 16-byte boundaries.
__host__ __device__ __forceinline__ int piece_bytes(int heads, int head_dim) { return (heads * (head_dim + 2) * 4 + 15) / 16 * 16; }
constexpr float kLowest = -3.402823466e38f;  // m before any score

// A warp's partial result of an item that another warp shares, left in shared memory: o [tile_heads][head_dim], then (m, l) of every head.
struct Piece {
  int b, item;
  int starts, ends;  // whether the item's first and last block are in it
  int used;
};

template <typename T, bool FP8, bool SB, int DP, int NT, int W>
__global__ void __launch_bounds__(W * 32, Shape<T, FP8, SB, DP, NT, W>::kCtasPerSm) paged_attention_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<T, FP8, SB, DP, NT, W>;
  using M = std::conditional_t<FP8, __half, T>;  // type of the products
  constexpr int kElt = FP8 ? 1 : 2;
  // Range of the weights, to base 2.  bf16 ones are not lifted: they lose nothing below 1, and values may go up to the end of 32 bits themselves.
  constexpr float kLift = std::is_same_v<M, __half> ? 7.f : 0.f, kMostWeight = kLift + 8.f;
  // Two 16-bit numbers of a weight, so that a result is rounded once.  (bf16 queries over 8-bit pages with a scale for each head have one, good to 2^-12 of each weight.  With scales of
  // blocks one took, replayed, 171 us for 64 sequences of 1 to 16384 tokens of 32/8 heads of 128, 32.2 for 32 of 700 of 16/16 and 8.2 for one of 513; two 182, 33.6 and 8.2.)
  constexpr bool kTwoParts = !FP8 || SB || std::is_same_v<T, __half>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Piece pieces[2 * W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const TrisPagedKv& c = a.cache;
  const TrisPagedAttention& query = a.query;
  const int D = c.head_dim;
  pdl_wait();
  pdl_launch_dependents();

  // This warp's run: its part of the CTA's (cluster's) one item, or of the numbering, with the sequence that holds its first block.
  Cursor use{};
  int count = 0, shares = 1;  // shares: CTAs of the cluster that have a part
  if (W < kWarps || a.cluster) {
    use.b = blockIdx.y;
    use.item = blockIdx.x;
    // the block table's row comes to L2 while the length is on its way
    if (warp == 0 && lane * 32 < c.table_width) asm volatile("prefetch.global.L2 [%0];" ::"l"(c.block_table + use.b * c.table_stride + lane * 32));
    use.span = span_of(a, use.b);
    use.blocks = use.span.blocks();
    if (query.lengths[use.b] != use.span.hi && c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
    const int run = (use.blocks + a.cluster * W - 1) / (a.cluster * W);
    use.blk = (blockIdx.z * W + warp) * run;
    count = max(0, min(run, use.blocks - use.blk));
    shares = run ? (use.blocks + W * run - 1) / (W * run) : 0;
    if (use.blocks <= 1 && (blockIdx.z > 0 || use.blocks == 0)) {  // one block is its warp's alone; nothing at all gives zeros
      if (use.blocks == 0 && blockIdx.z == 0) {
        const int head = use.item / a.row_tiles, row0 = use.item % a.row_tiles * S::kHeads, rows = min(S::kHeads, a.group - row0);
        const int64_t out_row = static_cast<int64_t>(use.b) * query.num_q_heads + head * a.group + row0;
        for (int i = threadIdx.x; i < rows * D; i += W * 32) store_float(static_cast<T*>(query.out) + out_row * D + i, 0.f);
        for (int i = threadIdx.x; query.lse && i < rows; i += W * 32) query.lse[out_row + i] = -INFINITY;
      }
      return;  // the whole cluster: none of its CTAs has a piece
    }
  } else if constexpr (W == kWarps) {
    int mine, upto = scan_blocks(a, 0, lane, mine);
    int total = __shfl_sync(0xFFFFFFFFu, upto, 31);
    for (int i = 1; 32 * i < c.num_sequences; ++i) {
      int own;
      total += __shfl_sync(0xFFFFFFFFu, scan_blocks(a, i, lane, own), 31);
    }
    const int run = run_length(a, total);
    if (static_cast<int64_t>(blockIdx.x) * kWarps * run >= total) return;
    const int64_t first_block = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * run;
    const int first = static_cast<int>(first_block);
    count = first_block < total ? min(run, total - first) : 0;
    if (count) {
      int before = 0;
      for (int i = 0;; ++i) {
        if (i) upto = scan_blocks(a, i, lane, mine);
        const uint32_t beyond = __ballot_sync(0xFFFFFFFFu, before + upto > first);
        if (beyond) {
          const int l = __ffs(beyond) - 1;
          const int ahead = first - before - __shfl_sync(0xFFFFFFFFu, upto - mine, l);
          use.enter(a, 32 * i + l);
          use.item = static_cast<unsigned>(ahead) / static_cast<unsigned>(use.blocks);
          use.blk = ahead - use.item * use.blocks;
          break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
      }
    }
  }
  if (lane < 2) pieces[2 * warp + lane].used = 0;
  __syncwarp();
  bool owns_start = use.blk == 0;  // whether the current item begins in this run

  uint32_t qf[NT][S::kSteps][2];
  float scale[NT][2];  // of heads 2 t and 2 t + 1 of a tile, to base 2
  float m[NT][2], l[NT][2], acc[S::kDimTiles][NT][4];
  auto fetch_query = [&] {
    const int head = use.item / a.row_tiles, tile = use.item % a.row_tiles;
    scale[0][0] = FP8 && !SB && c.k_scale ? c.k_scale[head] : 1.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = tile * S::kHeads + 8 * n + g;
      const T* src = static_cast<const T*>(query.q) + use.b * query.q_token_stride + (static_cast<int64_t>(head) * a.group + row) * query.q_head_stride;
      const bool there = row < a.group;
      if (a.wide_query) {
#pragma unroll
        for (int j = 0; j < S::kKeyChunks; ++j)
#pragma unroll
          for (int w = 0; w < S::kElems / 2; w += 4) {
            const int d = (4 * j + t) * S::kElems + 2 * w;
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (there && d < D) raw = *reinterpret_cast<const uint4*>(src + d);
            const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[n][j * (S::kElems / 4) + (w + i) / 2][i & 1] = v[i];
          }
      } else {
#pragma unroll
        for (int j = 0; j < S::kKeyChunks; ++j)
#pragma unroll
          for (int w = 0; w < S::kElems / 2; ++w) {
            const int d = (4 * j + t) * S::kElems + 2 * w;
            const uint16_t* at = reinterpret_cast<const uint16_t*>(src + d);
            qf[n][j * (S::kElems / 4) + w / 2][w & 1] = there && d < D ? at[0] | (static_cast<uint32_t>(at[1]) << 16) : 0;
          }
      }
    }
  };
  auto start_item = [&] {
    const float base = query.softmax_scale * kLog2e * scale[0][0];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float up = 1.f;
      if constexpr (FP8 && !std::is_same_v<T, __half>) {
        // bf16 queries against fp16 keys: a power of two brings a row's largest element to [2^14, 2^15), so that elements down to 2^-31 of it keep all
        // their bits; sums are in 32 bits and keys at most 448.  The magnitudes' bits order like the numbers.
        constexpr uint32_t kRaise = 14;
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) top = __vmaxu2(top, qf[n][s][i] & 0x7FFF7FFFu);
        top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const uint32_t e = min(max(max(top & 0xFFFFu, top >> 16) >> 7, 27u), 253u);  // biased exponent; zeros, infinities and NaN stay what they are
        up = __uint_as_float((e - kRaise) << 23);
        const float down = __uint_as_float((254 - e + kRaise) << 23);
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
      m[n][0] = m[n][1] = kLowest;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < S::kDimTiles; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][n][k] = 0.f;
    }
  };

  if (count) fetch_query();  // on its way while the first blocks are asked for

  Cursor load = use;
  int left = count;  // blocks that are not asked for yet
  // Page of token `lane & 15` of the block that is asked for next; of the block itself where blocks do not cross pages.
  auto page_of = [&](const Cursor& cur) {
    int tok = cur.token();
    if (!a.page_blocks) {
      tok += lane & 15;
      if (tok < cur.span.lo || tok >= cur.span.hi) return -1;
    }
    const int at = a.page_shift >= 0 ? tok >> a.page_shift : tok / c.page_size;
    const int page = c.block_table[cur.b * c.table_stride + at];
    if (page >= 0 && page < c.num_pages) return page;
    if (c.status_dev) *c.status_dev = TRIS_ERR_CORRUPT;
    return -1;
  };
  int page = left > 0 ? page_of(load) : -1;
  uint8_t* ring = smem + warp * (S::kStages * S::kStageBytes);
  const uint32_t ring_at = smem_u32(ring);
  const uint8_t *k_pages = static_cast<const uint8_t*>(c.k_pages), *v_pages = static_cast<const uint8_t*>(c.v_pages);
  const int64_t k_row = c.k_token_stride * kElt, v_row = c.v_token_stride * kElt;
  // A copy takes 512 bytes of neighbouring rows, lane after lane.  (Lanes that copy what they need themselves - values: four rows, 128 bytes
  // each, neighbouring lanes in different rows - reach 3.9 TB/s where this reaches 7.0.)
  constexpr int kCopies = S::kTile / 512;
  const int copy_row = lane / S::kRowChunks, copy_chunk = lane % S::kRowChunks;
  const uint32_t k_to = copy_row * S::kRowBytes + ((copy_chunk ^ S::key_swizzle(copy_row)) << 4);
  const uint32_t v_to = copy_row * S::kRowBytes + ((copy_chunk ^ S::value_swizzle(copy_row)) << 4);

  auto issue = [&](int stage) {
    if (left > 0) {
      const int tok0 = load.token(), head = load.item / a.row_tiles;
      const uint32_t dst = ring_at + stage * S::kStageBytes;
      if (a.rows_together && page >= 0 && tok0 >= load.span.lo && tok0 + kBlock <= load.span.hi) {
        // a whole block of one page, side by side in memory: addresses are one base and constants (32 x 512-768: 34.6 us, 36.9 without)
        const int64_t in_page = a.page_shift >= 0 ? tok0 & (c.page_size - 1) : tok0 % c.page_size;
        const uint8_t* k = k_pages + (page * c.k_page_stride + head * c.k_head_stride) * kElt + in_page * S::kRowBytes + lane * 16;
        const uint8_t* v = v_pages + (page * c.v_page_stride + head * c.v_head_stride) * kElt + in_page * S::kRowBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) cp_async_16_at(dst + (k_to ^ (S::key_swizzle(i * S::kCopyRows) << 4)) + i * 512, k + i * 512, 16);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) cp_async_16_at(dst + (v_to ^ (S::value_swizzle(i * S::kCopyRows) << 4)) + S::kTile + i * 512, v + i * 512, 16);
      } else {
        const int tok = tok0 + (lane & 15);
        const bool there = page >= 0 && tok >= load.span.lo && tok < load.span.hi;
        const int in_page = a.page_shift >= 0 ? tok & (c.page_size - 1) : tok % c.page_size;
        const int64_t k_off = there ? (page * c.k_page_stride + head * c.k_head_stride) * kElt + in_page * k_row : -1;
        const int64_t v_off = there ? (page * c.v_page_stride + head * c.v_head_stride) * kElt + in_page * v_row : -1;
        const bool in_row = copy_chunk * S::kElems < D;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int64_t off = __shfl_sync(0xFFFFFFFFu, k_off, i * S::kCopyRows + copy_row);
          const bool ok = off >= 0 && in_row;
          cp_async_16_at(dst + (k_to ^ (S::key_swizzle(i * S::kCopyRows) << 4)) + i * 512, ok ? k_pages + off + copy_chunk * 16 : k_pages, ok ? 16 : 0);
        }
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int64_t off = __shfl_sync(0xFFFFFFFFu, v_off, i * S::kCopyRows + copy_row);
          const bool ok = off >= 0 && in_row;
          cp_async_16_at(dst + (v_to ^ (S::value_swizzle(i * S::kCopyRows) << 4)) + S::kTile + i * 512, ok ? v_pages + off + copy_chunk * 16 : v_pages, ok ? 16 : 0);
        }
      }
      if constexpr (SB) {
        // each lane brings the scale of one token: keys' in the first half, values' in the other
        const int tok = tok0 + (lane & 15);
        const bool there = page >= 0 && tok >= load.span.lo && tok < load.span.hi;
        const int in_page = a.page_shift >= 0 ? tok & (c.page_size - 1) : tok % c.page_size;
        const int block = a.scale_shift >= 0 ? in_page >> a.scale_shift : in_page / c.scale_tokens;
        const float* src = (lane < 16 ? c.k_scale : c.v_scale) + (there ? (static_cast<int64_t>(page) * a.page_scales + block) * c.num_kv_heads + head : 0);
        cp_async_4_at(dst + S::kScales + 4 * lane, src, there ? 4 : 0);
      }
      if (--left > 0) {
        load.next(a);
        page = page_of(load);
      }
    }
    cp_async_commit();  // empty groups keep the count of groups in step
  };
  // where this lane's fragments are in a stage: keys g and g + 8, chunks 4 j + t; values 2 t, 2 t + 1, 2 t + 8, 2 t + 9, chunks 8 j + g
  const uint32_t k_from = g * S::kRowBytes + ((t ^ S::key_swizzle(g)) << 4);
  const uint32_t v_from = S::kTile + 2 * t * S::kRowBytes +
                          (S::kValueElems == S::kElems ? (g ^ S::value_swizzle(2 * t)) << 4 : (((g >> 1) ^ S::value_swizzle(2 * t)) << 4) + 8 * (g & 1));

  // The result of an item that this warp has had alone goes out; otherwise its piece is left for the other warps' (to != nullptr).
  auto write_item = [&](float* to) {
    const int head = use.item / a.row_tiles, tile = use.item % a.row_tiles;
    const float v_scale = FP8 && !SB && c.v_scale ? c.v_scale[head] : 1.f;
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
        const float inv = to ? v_scale : sum == 0.f ? 0.f : v_scale / sum;
#pragma unroll
        for (int j = 0; j < S::kValueChunks; ++j) {
          const int d0 = (8 * j + g) * S::kValueElems;
          if (d0 >= D) continue;
#pragma unroll
          for (int q = 0; q < S::kValueElems / 8; ++q) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[2 * i] = acc[j * (S::kValueElems / 2) + 4 * q + i][n][h] * inv;
              v[2 * i + 1] = acc[j * (S::kValueElems / 2) + 4 * q + i][n][2 + h] * inv;
            }
            if (to) {
              float4* dst = reinterpret_cast<float4*>(to + in_tile * D + d0 + 8 * q);
              dst[0] = make_float4(v[0], v[1], v[2], v[3]);
              dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
              store_8(static_cast<T*>(query.out) + out_row * D + d0 + 8 * q, v);
            }
          }
        }
        if (g == 0) {
          if (to)
            *reinterpret_cast<float2*>(to + a.tile_heads * D + 2 * in_tile) = make_float2(m[n][h], sum);
          else if (query.lse)
            query.lse[out_row] = sum == 0.f ? -INFINITY : (m[n][h] + log2f(sum)) * kLn2;
        }
      }
  };
  // Two pieces at most: of the item that another warp began (slot 0), and, with the warp's last block, of one that another warp ends (slot 1).
  // The second one takes the ring's place, all of which has been read by then.
  auto piece_at = [&](int slot) {
    uint8_t* at = slot & 1 || W < kWarps ? smem + (slot >> 1) * (S::kStages * S::kStageBytes) : smem + S::kRing + (slot >> 1) * piece_bytes(a.tile_heads, D);
    return reinterpret_cast<float*>(at);
  };
  // Lanes 0 to 7 have the (m, l) of partial results: the largest m, the weight of each, and the weighted sum of the l.
  auto weight_of = [](float2 ml, float& top, float& sum) {
    top = ml.x;
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
    const float weight = exp2_fast(ml.x - top);
    sum = weight * ml.y;
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, k);
    top = __shfl_sync(0xFFFFFFFFu, top, 0);
    sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
    return weight;
  };
  static_assert(2 * W <= 8 && kMostCluster <= 8, "weight_of");
  auto store_result = [&](int b, int q_head, int d, float top, float sum, float4 o) {
    const int64_t out_row = static_cast<int64_t>(b) * query.num_q_heads + q_head;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(static_cast<T*>(query.out) + out_row * D + d) = make_uint2(Pair<T>::pack(o.x * inv, o.y * inv), Pair<T>::pack(o.z * inv, o.w * inv));
    if (d == 0 && query.lse) query.lse[out_row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  };

  bool fresh = true;  // an item begins
  // The first turns only ask for blocks; every later one does its block and asks for another in the place of the one before.  (Code that runs once
  // a CTA comes from far away: it is written once, and in loops.)
  int stage = 0, place = 0;
#pragma unroll 1
  for (int i = count ? 1 - S::kStages : 0; i < count; ++i) {
    if (i < 0) {
      issue(place++);
      continue;
    }
    if (fresh) start_item();
    fresh = false;
    cp_async_wait<S::kStages - 2>();
    __syncwarp();  // all lanes' copies are there, and all lanes are done with the stage that is filled next
    const uint8_t* src = ring + stage * S::kStageBytes;

    float s[NT][4], s_odd[NT][4];  // two sums: an MMA waits 20 cycles for the one before it
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = s_odd[n][k] = 0.f;
#pragma unroll
    for (int j = 0; j < S::kKeyChunks; ++j) {
      const uint8_t* keys = src + (k_from ^ ((j & 1) << 6)) + ((j & ~1) << 6);
      const uint4 ka = *reinterpret_cast<const uint4*>(keys), kb = *reinterpret_cast<const uint4*>(keys + 8 * S::kRowBytes);
      const uint32_t x[4] = {ka.x, ka.y, ka.z, ka.w}, y[4] = {kb.x, kb.y, kb.z, kb.w};
      if constexpr (FP8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = e4m3_to_h2(x[w] & 0xFFFF), a2 = e4m3_to_h2(x[w] >> 16), a1 = e4m3_to_h2(y[w] & 0xFFFF), a3 = e4m3_to_h2(y[w] >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<M>(w & 1 ? s_odd[n] : s[n], a0, a1, a2, a3, qf[n][4 * j + w][0], qf[n][4 * j + w][1]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<M>(w ? s_odd[n] : s[n], x[2 * w], y[2 * w], x[2 * w + 1], y[2 * w + 1], qf[n][2 * j + w][0], qf[n][2 * j + w][1]);
      }
    }

    // Tokens g and g + 8 of heads 2 t and 2 t + 1.  Weights are 2^(s - m); m is the largest score so far less kLift when it moves, and moves only when
    // a score exceeds it by more than kMostWeight, which is rare after the first blocks.  Of fp16 the largest weight is so between 2^7 and
    // 2^15 (the type ends below 2^16), and weights down to 2^-21 of it have all of its bits; sums in 32 bits are as exact at any scale.
    // With scales of blocks a token's weight in the sum over the values has its value scale in it, 2^e * f with f in [1/2, 1): m follows s + e, so that it is that
    // weight which keeps its bits, whatever the scales of other blocks are; the sum l is of 2^(s - m).
    float key_scale[2] = {1.f, 1.f}, value_part[2] = {1.f, 1.f}, lift[2] = {0.f, 0.f};
    if constexpr (SB) {
      const float* scales = reinterpret_cast<const float*>(src + S::kScales);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        key_scale[h] = scales[g + 8 * h];
        const uint32_t bits = __float_as_uint(fminf(fmaxf(scales[kBlock + g + 8 * h], 0x1p-64f), 0x1p64f));
        lift[h] = static_cast<float>(static_cast<int>(bits >> 23) - 126);
        value_part[h] = __uint_as_float((bits & 0x7FFFFFu) | (126u << 23));
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[n][k] = (s[n][k] + s_odd[n][k]) * scale[n][k & 1];
        if constexpr (SB) s[n][k] = fmaf(s[n][k], key_scale[k >> 1], lift[k >> 1]);
      }
    const int tok = use.token();
    if (tok < use.span.lo || tok + kBlock > use.span.hi) {
      const bool in0 = tok + g >= use.span.lo && tok + g < use.span.hi, in1 = tok + g + 8 >= use.span.lo && tok + g + 8 < use.span.hi;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (!in0) s[n][0] = s[n][1] = -INFINITY;
        if (!in1) s[n][2] = s[n][3] = -INFINITY;
      }
    }
    float x[NT][4];
    bool above = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[n][k] = s[n][k] - m[n][k & 1];
        above |= x[n][k] > kMostWeight;
      }
    if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float old[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
          top = fmaxf(m[n][h], top - kLift);
          old[h] = exp2_fast(m[n][h] - top);
          m[n][h] = top;
          l[n][h] *= old[h];
          x[n][h] = s[n][h] - top;
          x[n][2 + h] = s[n][2 + h] - top;
        }
#pragma unroll
        for (int k = 0; k < S::kDimTiles; ++k) {
          acc[k][n][0] *= old[0];
          acc[k][n][1] *= old[1];
          acc[k][n][2] *= old[0];
          acc[k][n][3] *= old[1];
        }
      }
    }
    // The weights as the 8-column operand: pairs of tokens of one head, each weight a 16-bit number or the sum of two (two_parts), whose products with the
    // values add up in the same accumulators.  The sum l is of the weights as they are.
    uint32_t p[NT][2], rest[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (SB) {
        float plain[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          plain[k] = exp2_fast(x[n][k] - lift[k >> 1]);
          x[n][k] = exp2_fast(x[n][k]) * value_part[k >> 1];
        }
        l[n][0] += plain[0] + plain[2];
        l[n][1] += plain[1] + plain[3];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[n][k] = exp2_fast(x[n][k]);
        l[n][0] += x[n][0] + x[n][2];
        l[n][1] += x[n][1] + x[n][3];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if constexpr (kTwoParts) {
          two_parts<M>(x[n][2 * k], x[n][2 * k + 1], p[n][k], rest[n][k]);
          rest[n][k] = transpose_8x8(rest[n][k]);
        } else {
          p[n][k] = Pair<M>::pack(x[n][2 * k], x[n][2 * k + 1]);
        }
        p[n][k] = transpose_8x8(p[n][k]);
      }
    }

    const uint8_t* vals = src + v_from;
#pragma unroll
    for (int j = 0; j < S::kValueChunks; ++j) {
      uint32_t v[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint8_t* at = vals + ((r & 1) + 8 * (r >> 1)) * S::kRowBytes + j * 128;
        if constexpr (S::kValueElems == S::kElems) {
          const uint4 raw = *reinterpret_cast<const uint4*>(at);
          v[r][0] = raw.x, v[r][1] = raw.y, v[r][2] = raw.z, v[r][3] = raw.w;
        } else {
          const uint2 raw = *reinterpret_cast<const uint2*>(at);
          v[r][0] = raw.x, v[r][1] = raw.y;
        }
      }
#pragma unroll
      for (int w = 0; w < 4 * S::kValueElems / S::kElems; ++w) {
        if constexpr (FP8) {
          // bytes of two tokens side by side first, then two values at a time: {token 0, token 1} of dimensions 4 w + i
          const uint32_t lo0 = prmt(v[0][w], v[1][w], 0x5140), hi0 = prmt(v[0][w], v[1][w], 0x7362);
          const uint32_t lo1 = prmt(v[2][w], v[3][w], 0x5140), hi1 = prmt(v[2][w], v[3][w], 0x7362);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t u0 = e ? hi0 : lo0, u1 = e ? hi1 : lo1;
            const uint32_t a0 = e4m3_to_h2(u0 & 0xFFFF), a1 = e4m3_to_h2(u0 >> 16), a2 = e4m3_to_h2(u1 & 0xFFFF), a3 = e4m3_to_h2(u1 >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16x8x16<M>(acc[j * (S::kValueElems / 2) + 2 * w + e][n], a0, a1, a2, a3, p[n][0], p[n][1]);
              if constexpr (kTwoParts) mma_16x8x16<M>(acc[j * (S::kValueElems / 2) + 2 * w + e][n], a0, a1, a2, a3, rest[n][0], rest[n][1]);
            }
          }
        } else {
          const uint32_t a0 = prmt(v[0][w], v[1][w], 0x5410), a1 = prmt(v[0][w], v[1][w], 0x7632);
          const uint32_t a2 = prmt(v[2][w], v[3][w], 0x5410), a3 = prmt(v[2][w], v[3][w], 0x7632);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16x8x16<M>(acc[j * 4 + w][n], a0, a1, a2, a3, p[n][0], p[n][1]);
            if constexpr (kTwoParts) mma_16x8x16<M>(acc[j * 4 + w][n], a0, a1, a2, a3, rest[n][0], rest[n][1]);
          }
        }
      }
    }
    issue(place);
    if (++place == S::kStages) place = 0;
    if (++stage == S::kStages) stage = 0;

    const bool last = i + 1 == count, ends = use.blk + 1 == use.blocks;
    if (last || ends) {
      float* to = nullptr;
      if (!(owns_start && ends)) {
        const int slot = 2 * warp + (owns_start ? 1 : 0);
        to = piece_at(slot);
        if (lane == 0) pieces[slot] = {use.b, use.item, owns_start, ends, 1};
        __syncwarp();
      }
      write_item(to);
      if (!last) {
        use.next(a);
        owns_start = fresh = true;
        fetch_query();
      }
    } else {
      ++use.blk;
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // Neighbouring warps' pieces of one item are joined here; what other CTAs share goes to the workspace, or is left for the cluster.
  const uint32_t used = __ballot_sync(0xFFFFFFFFu, lane < 2 * W && pieces[lane & (2 * W - 1)].used);
  const uint32_t last_ones = used & __ballot_sync(0xFFFFFFFFu, pieces[lane & (2 * W - 1)].ends);
#pragma unroll 1
  for (uint32_t rest = used; rest;) {
    const int s0 = __ffs(rest) - 1;
    const uint32_t ends = last_ones & rest;
    const uint32_t group = ends ? rest & (ends ^ (ends - 1)) : rest;  // up to the first piece that ends an item
    rest &= ~group;
    const Piece item = pieces[s0];
    const bool whole = item.starts && ends;
    const int head = item.item / a.row_tiles, tile = item.item % a.row_tiles;
    const int heads = min(S::kHeads, a.group - tile * S::kHeads);
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (item.starts ? 1 : 0);
    float* to_o = W < kWarps || a.cluster ? piece_at(3) : a.part_o + slot * a.tile_heads * D;
    float* to_ml = W < kWarps || a.cluster ? piece_at(3) + a.tile_heads * D : a.part_ml + slot * a.tile_heads * 2;
    // a warp takes 128 dimensions of a head at a time
#pragma unroll 1
    for (int unit = warp; unit < heads * ((D + 127) / 128); unit += W) {
      const int h = D > 128 ? unit >> 1 : unit, d = (D > 128 ? (unit & 1) * 128 : 0) + 4 * lane;
      // lane k has the weight of piece k
      float2 ml = make_float2(kLowest, 0.f);
      if ((group >> lane) & 1) ml = *reinterpret_cast<const float2*>(piece_at(lane) + a.tile_heads * D + 2 * h);
      float top, sum;
      const float weight = weight_of(ml, top, sum);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 2 * W; ++k) {
        if (!((group >> k) & 1)) continue;
        const float4 v = *reinterpret_cast<const float4*>(piece_at(k) + h * D + min(d, D - 4));
        const float w = __shfl_sync(0xFFFFFFFFu, weight, k);
        o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
      }
      if (d >= D) continue;
      if (whole) {
        store_result(item.b, head * a.group + tile * S::kHeads + h, d, top, sum, o);
      } else {
        *reinterpret_cast<float4*>(to_o + h * D + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(to_ml + h * 2) = make_float2(top, sum);
      }
    }
  }

  if (W < kWarps || a.cluster < 2 || shares < 2) return;  // all CTAs of a cluster agree on that
  // The cluster's CTAs have left what they have of the item in the part of their rings that the item's second warp had; each joins some of it.
  cluster_sync();
  const int head = use.item / a.row_tiles, tile = use.item % a.row_tiles, heads = min(S::kHeads, a.group - tile * S::kHeads);
  const uint32_t local = smem_u32(piece_at(3));
#pragma unroll 1
  for (int unit = blockIdx.z * W + warp; unit < heads * ((D + 127) / 128); unit += a.cluster * W) {
    const int h = D > 128 ? unit >> 1 : unit, d = (D > 128 ? (unit & 1) * 128 : 0) + 4 * lane, at = (h * D + min(d, D - 4)) * 4;
    // lane r has the weight of CTA r
    float2 ml = load_cluster_2(in_cta(local, min(lane, shares - 1)) + (a.tile_heads * D + 2 * h) * 4);
    if (lane >= shares) ml = make_float2(kLowest, 0.f);
    float top, sum;
    const float weight = weight_of(ml, top, sum);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int r = 0; r < shares; ++r) {
      const float4 v = load_cluster_4(in_cta(local, r) + at);
      const float w = __shfl_sync(0xFFFFFFFFu, weight, r);
      o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
    }
    if (d < D) store_result(use.b, head * a.group + tile * S::kHeads + h, d, top, sum, o);
  }
  cluster_sync();  // nobody leaves while another reads its shared memory
}

// Joins the partial results of one query head of one sequence; zeros where there was nothing to attend to.
constexpr int kJoinWarps = 4, kJoinThreads = 32 * kJoinWarps;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ AttnArgs a, int tile_rows) {
  __shared__ float2 stats[kJoinThreads];
  __shared__ float4 sums[kJoinThreads];
  pdl_wait();
  pdl_launch_dependents();
  const TrisPagedKv& c = a.cache;
  const TrisPagedAttention& query = a.query;
  const int tid = threadIdx.x, lane = tid & 31;
  const int b = blockIdx.y, q_head = blockIdx.x, head = q_head / a.group, row = q_head % a.group;
  const int tile = row / tile_rows, in_tile = row % tile_rows, D = c.head_dim, D4 = D / 4;
  const int64_t out_row = static_cast<int64_t>(b) * query.num_q_heads + q_head;
  int before;
  const int total = count_blocks(a, b, lane, before);
  const Span span = span_of(a, b);
  const int blocks = span.blocks();
  T* out = static_cast<T*>(query.out) + out_row * D;
  if (query.lengths[b] != span.hi && c.status_dev && q_head == 0 && tid == 0) *c.status_dev = TRIS_ERR_CORRUPT;
  if (blocks == 0) {
    for (int d = tid; d < D; d += kJoinThreads) store_float(out + d, 0.f);
    if (query.lse && tid == 0) query.lse[out_row] = -INFINITY;
    return;
  }
  const unsigned run = run_length(a, total) * kWarps;  // of a CTA
  const unsigned start = before + (head * a.row_tiles + tile) * blocks;
  const int w0 = start / run, n = (start + blocks - 1) / run - w0 + 1;
  if (n == 1) return;  // one CTA had all of it
  auto slot = [&](int i) { return (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * a.tile_heads + in_tile; };

  // A group of D / 4 threads takes every groups-th partial result, kBatch of them at a time so that their loads are in flight together;
  // the groups' results are joined in their order.
  constexpr int kBatch = 8;
  const int groups = kJoinThreads / D4, grp = tid / D4, col = tid - grp * D4;
  float top = kLowest, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, float2 ml, float4 v) {
    sum += w * ml.y;
    o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
  };
  auto rescale = [&](float to) {
    const float w = exp2_fast(top - to);
    sum *= w;
    o.x *= w, o.y *= w, o.z *= w, o.w *= w;
    top = to;
  };
  if (grp < groups) {
    for (int i0 = grp; i0 < n; i0 += kBatch * groups) {
      float2 ml[kBatch];
      float4 v[kBatch];
      float to = top;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * groups;
        ml[k] = make_float2(kLowest, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n) {
          ml[k] = *reinterpret_cast<const float2*>(a.part_ml + slot(i) * 2);
          v[k] = *reinterpret_cast<const float4*>(a.part_o + slot(i) * D + 4 * col);
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) to = fmaxf(to, ml[k].x);
      rescale(to);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) add(exp2_fast(ml[k].x - top), ml[k], v[k]);
    }
    sums[tid] = o;
    stats[tid] = make_float2(top, sum);
  }
  __syncthreads();
  if (tid >= D4) return;
  const int used = n < groups ? n : groups;
  float to = top;
  for (int k = 1; k < used; ++k) to = fmaxf(to, stats[k * D4].x);
  rescale(to);
  for (int k = 1; k < used; ++k) {
    const float2 ml = stats[k * D4];
    add(exp2_fast(ml.x - top), ml, sums[k * D4 + tid]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(out + 4 * tid) = make_uint2(Pair<T>::pack(o.x * inv, o.y * inv), Pair<T>::pack(o.z * inv, o.w * inv));
  if (query.lse && tid == 0) query.lse[out_row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// CTAs of the first kernel: twice as many as are resident, but no more than there can be shares of one block for their warps.
int attention_ctas(int resident, int64_t blocks) {
  const int64_t ctas = (blocks + kWarps - 1) / kWarps;
  return static_cast<int>(ctas < 1 ? 1 : ctas < 2 * resident ? ctas : 2 * resident);
}
int64_t most_blocks(const TrisPagedKv& c, int row_tiles) {
  return static_cast<int64_t>(c.num_sequences) * c.num_kv_heads * row_tiles * ((static_cast<int64_t>(c.table_width) * c.page_size + kBlock - 1) / kBlock + 1);
}
// CTAs that share an item, as many as still run at the same time for all items, up to kMostCluster; 0: the work is numbered through.  One launch instead
// of two and no numbering are worth 1 to 3 us (flat and clusters, us: 20 x 1 token 6.1 / 4.3, 1 x 513 8.7 / 7.4, 16 x 4096 in 8 bits 25.5 / 22.3), and
// many short sequences gain more (32 x 512-768 37.6 / 34.7, 64 x 1-1024 44.6 / 34.9).  But a cluster's longest sequence ends last, and SMs without an
// item stay idle: 1 x 8192 13.4 / 20.0, 1 x 4096 10.7 / 12.5, 64 x 1-2048 59.1 / 60.3, 64 x 1-3000 79 / 84, 64 x 1-16384 293 / 299.  Where the items take many
// rounds their ends even out: 128 x 1-4096 197 / 183, 128 x 1-8192 354 / 355, 200 x 1-8192 560 / 540.  So a warp may have up to kMostShare blocks
// of the longest sequence that the table (or the window) has room for, times the rounds, or the part of one, that the items take.
// The host knows that room, not the lengths: short sequences in a table for 8192 tokens or 131072 are numbered (tight and wide tables, us: 1 x 513
// 8.0 / 9.0, 8 x 513 11.8 / 14.6, 32 x 512-768 35.5 / 36.9).
constexpr int kMostShare = 24, kLeastShare = 4;
int cluster_size(const TrisPagedKv& c, int row_tiles, int window, int resident) {
  const int64_t items = static_cast<int64_t>(c.num_sequences) * c.num_kv_heads * row_tiles;
  int64_t tokens = static_cast<int64_t>(c.table_width) * c.page_size;
  if (window > 0 && window < tokens) tokens = static_cast<int64_t>(window) + kBlock;
  int size = kMostCluster;
  while (size > 1 && items * size > resident) size /= 2;
  int64_t share = kMostShare * items * size / resident;
  if (share < kLeastShare) share = kLeastShare;
  return tokens <= share * kBlock * kWarps * size ? size : 0;
}
// More items than CTAs that run at one time, of at most kShort tokens: start and end of a CTA are all there is, and CTAs of two warps, of which twice
// as many run, halve the rounds.  Four and two warps, us: 42 x 16 tokens of 8 heads 7.3 / 4.5, 128 x 64 19.6 / 14.1, 64 x 256 18.4 / 17.0; 64 x 512 27.0 / 29.3, and
// for 42 x 128 in 8 bits, all of whose CTAs run, 7.5 / 8.5.
constexpr int kShort = 256;
bool two_warps(const TrisPagedKv& c, int row_tiles, int window, int resident) {
  const int64_t items = static_cast<int64_t>(c.num_sequences) * c.num_kv_heads * row_tiles;
  return items > resident && (static_cast<int64_t>(c.table_width) * c.page_size <= kShort || (window > 0 && window <= kShort - kBlock));
}
int resident_ctas(int head_dim, bool fp8, int tiles) { return sm_count() * ctas_per_sm(head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256, fp8, tiles); }
// Tiles of 8 query heads that share a key/value head's pass: two where a group has more than 8 - with heads of 256 dimensions the accumulators of two
// do not fit the registers -, but where even so every tile has a cluster of its own of the largest size, one: the pages are read twice, by two
// clusters, and what a warp does alone at its end is halved (group of 16, 8 x 1000 tokens 11.5 / 9.4 us, 32 x 1000 15.1 / 15.9, 128 x 1000 32 / 40).
int head_tiles(const TrisPagedKv& c, int group, int window) {
  if (group <= 8 || c.head_dim > 128) return 1;
  const int singles = ceil_div(group, 8), resident = resident_ctas(c.head_dim, c.dtype == TRIS_DTYPE_E4M3, 1);
  const bool room = static_cast<int64_t>(c.num_sequences) * c.num_kv_heads * singles * kMostCluster <= resident;
  return room && cluster_size(c, singles, window, resident) ? 1 : 2;
}
size_t part_floats(int ctas, int tile_heads, int head_dim) { return 2 * static_cast<size_t>(ctas) * tile_heads * (head_dim + 2); }

template <typename T, bool FP8, bool SB, int DP, int NT>
int launch_attention(AttnArgs& a, cudaStream_t stream) {
  using S = Shape<T, FP8, SB, DP, NT, kWarps>;
  auto kernel = paged_attention_kernel<T, FP8, SB, DP, NT, kWarps>;
  const TrisPagedKv& c = a.cache;
  if (int st = allow_shared_memory<paged_attention_kernel<T, FP8, SB, DP, NT, kWarps>>(S::kMostSmem)) return st;
  TRIS_REQUIRE(sm_count() > 0, TRIS_ERR_CUDA, "paged_decode_attention: no device");
  a.resident = resident_ctas(c.head_dim, FP8, NT);
  a.rows_together = a.page_blocks && c.head_dim == DP && c.k_token_stride == DP && c.v_token_stride == DP;
  const bool pdl = programmatic_launch_default();
  a.cluster = cluster_size(c, a.row_tiles, a.query.window, a.resident);
  const dim3 items(c.num_kv_heads * a.row_tiles, c.num_sequences, a.cluster);
  if (a.cluster == 1 && two_warps(c, a.row_tiles, a.query.window, a.resident)) {
    using P = Shape<T, FP8, SB, DP, NT, 2>;
    if (int st = allow_shared_memory<paged_attention_kernel<T, FP8, SB, DP, NT, 2>>(P::kMostSmem)) return st;
    TRIS_CUDA(launch_step(paged_attention_kernel<T, FP8, SB, DP, NT, 2>, items, dim3(64), P::kMostSmem, stream, pdl, 1, a));
    return TRIS_OK;
  }
  if (a.cluster) {
    TRIS_CUDA(launch_step(kernel, items, dim3(kWarps * 32), S::kRing + kWarps * piece_bytes(a.tile_heads, c.head_dim), stream, pdl, a.cluster, a));
    return TRIS_OK;
  }
  a.ctas = attention_ctas(a.resident, most_blocks(c, a.row_tiles));
  a.part_ml = static_cast<float*>(a.query.workspace);
  a.part_o = a.part_ml + 4 * static_cast<size_t>(a.ctas) * a.tile_heads;
  const int64_t need = part_floats(a.ctas, a.tile_heads, c.head_dim) * 4;
  TRIS_REQUIRE(a.query.workspace && a.query.workspace_bytes >= need, TRIS_ERR_WORKSPACE, "paged_decode_attention: workspace of %lld bytes needed, got %lld",
               static_cast<long long>(need), static_cast<long long>(a.query.workspace_bytes));
  TRIS_CUDA(launch_step(kernel, dim3(a.ctas), dim3(kWarps * 32), S::kRing + kWarps * piece_bytes(a.tile_heads, c.head_dim), stream, pdl, 1, a));
  TRIS_CUDA(launch_step(paged_attention_join_kernel<T>, dim3(a.query.num_q_heads, c.num_sequences), dim3(kJoinThreads), 0, stream, true, 1, a, S::kHeads));
  return TRIS_OK;
}
template <typename T, bool FP8, bool SB>
int launch_shape(AttnArgs& a, int tiles, cudaStream_t stream) {
  const int d = a.cache.head_dim;
  if (tiles == 2) return d <= 64 ? launch_attention<T, FP8, SB, 64, 2>(a, stream) : launch_attention<T, FP8, SB, 128, 2>(a, stream);
  return d <= 64 ? launch_attention<T, FP8, SB, 64, 1>(a, stream) : d <= 128 ? launch_attention<T, FP8, SB, 128, 1>(a, stream) : launch_attention<T, FP8, SB, 256, 1>(a, stream);
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" size_t tris_paged_decode_attention_workspace_bytes(const TrisPagedKv* cache, int32_t num_q_heads, int32_t window) {
  if (validate_paged_kv(cache, "paged_decode_attention")) return 0;
  if (num_q_heads < 1 || num_q_heads % cache->num_kv_heads || window < 0 || sm_count() == 0) return 0;
  const int group = num_q_heads / cache->num_kv_heads, tiles = head_tiles(*cache, group, window), heads = 8 * tiles, row_tiles = ceil_div(group, heads);
  const int resident = resident_ctas(cache->head_dim, cache->dtype == TRIS_DTYPE_E4M3, tiles);
  if (cluster_size(*cache, row_tiles, window, resident)) return 0;
  return part_floats(attention_ctas(resident, most_blocks(*cache, row_tiles)), group < heads ? group : heads, cache->head_dim) * 4;
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
  const int tiles = head_tiles(c, a.group, q.window), heads = 8 * tiles;
  a.row_tiles = ceil_div(a.group, heads);
  a.tile_heads = a.group < heads ? a.group : heads;
  a.page_blocks = c.page_size % kBlock == 0;
  a.wide_query = aligned_to(q.q, 16) && q.q_token_stride % 8 == 0 && q.q_head_stride % 8 == 0;
  TRIS_REQUIRE(static_cast<int64_t>(c.table_width) * c.page_size < (1ll << 31) - kBlock && most_blocks(c, a.row_tiles) < (1ll << 31), TRIS_ERR_UNSUPPORTED,
               "paged_decode_attention: a block table for more than 2^31 blocks of %d tokens (all sequences and heads)", kBlock);
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page_size == 1 << s) a.page_shift = s;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool q8 = c.dtype == TRIS_DTYPE_E4M3;
  a.scale_shift = -1;
  if (c.scale_tokens) {
    a.page_scales = c.page_size / c.scale_tokens;
    for (int i = 0; i < 31; ++i)
      if (c.scale_tokens == 1 << i) a.scale_shift = i;
    return q.dtype == TRIS_DTYPE_F16 ? launch_shape<__half, true, true>(a, tiles, s) : launch_shape<__nv_bfloat16, true, true>(a, tiles, s);
  }
  if (q.dtype == TRIS_DTYPE_F16) return q8 ? launch_shape<__half, true, false>(a, tiles, s) : launch_shape<__half, false, false>(a, tiles, s);
  return q8 ? launch_shape<__nv_bfloat16, true, false>(a, tiles, s) : launch_shape<__nv_bfloat16, false, false>(a, tiles, s);
}
