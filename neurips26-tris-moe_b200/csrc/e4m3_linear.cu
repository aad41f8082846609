// Products of e4m3 rows with e4m3 weights, a scale for each row and 128 columns of x and for each 128 x 128 block of the weights.
//
// y[t, n] = sum_g xs[t, g] ws[n / 128, g] sum_{k in g} x[t, k] w[n, k] + bias[n].  The inner sums are products of 128 columns on the tensor cores
// (tcgen05.mma, kind::f8f6f4, fp32 accumulators in TMEM); the scales differ from one group to the next, so every group's tile leaves TMEM and is added
// to 32-bit sums in registers, times its scale.  TMEM tiles take turns: one is filled while another is read.
//
// Roles: one warp asks for operands (TMA, a ring of stages), one issues the MMAs, and one or two groups of four warps add up.
//   rows few (kFeatures): the 128 lanes of a tile are features, its columns rows of x, so that a tile wastes nothing on rows that do not exist; a thread has
//   one feature, and the rows' scales come from shared memory.  Bound by the weights' bytes; the groups are cut among the CTAs of a cluster, whose sums
//   are joined in the order of the CTAs over distributed shared memory.
//   rows many (kRows): the lanes are rows of x, the columns features.  A thread has one row and its scales, four groups of them at a time.
//   rows many, tiles enough (kPair): two CTAs of a cluster have one tile of 256 rows x 256 features, each 128 of its rows in TMEM and 128 of either operand in shared
//   memory, which the MMAs of both read.  The way from L2 brings an SM some 50 bytes a cycle: a group of a tile of 128 x 256 is 48 KB for 512 cycles of the tensor core,
//   half a pair's tile 32 KB.  The tile's halves are multiplied, read and given back by themselves, a half for each group of warps.
// 8192 rows of 4096 to 14336 features in bf16: 0.9 million cycles: 560 to 585 us in a loop (563 at 1590 MHz, 576 at 1560, which the power limit leaves), 470 to 515 after a pause (1.65 to 2.0 PFLOP/s;
// beside 471 us tiles of 128 x 128 took 640 and of 128 x 256 without pairs 570), of which loads and products alone take 332; the rest is the sums: 128 columns of a thread leave TMEM in four loads that wait, some 1000 cycles a group with what is around
// them, at two warps a scheduler.  Tried, us beside 471: four groups of warps 520, 16 columns a load 512, packed sums 540, more registers for the sums by setmaxnreg 484.
// 64 rows of 4096 to 32000 in fp32: 30 us, 131 MB of weights; streaming them alone takes 24.  One row of 2048 to 6144: 6.1 us, a chain of launch, loads, products and join.
#include <type_traits>

#include "decode_step.cuh"
#include "umma.cuh"

namespace tris {

// Row-major rows of `cols` bytes, `stride` bytes apart; one copy = 128 columns of box_rows rows, 128-byte-swizzled, zeros past the matrix (tc_gemm.cu).
bool encode_bytes_map(CUtensorMap* map, const void* base, int rows, int cols, int64_t stride, int box_rows);
// The same of outputs, elt bytes each: 128 bytes of 128 rows, nothing is written past the matrix.
bool encode_output_map(CUtensorMap* map, const void* base, int rows, int cols, int elt, int64_t stride);

namespace {

constexpr int kGroup = 128;  // columns of a scale, and bytes of a swizzled line
constexpr int kLanes = 128;  // rows of a tile's first operand

enum class Mode { kFeatures, kRows, kPair };

struct LinearArgs {
  TrisE4m3Linear a;
  int groups;       // of K
  int per_cta;      // of them, that a CTA adds up
  int row_tiles, feature_tiles;
  int store_map;    // whether outputs go out by tensor copies
  int wide_scales;  // whether four scales of a row can be read at once
};
struct LinearMaps {
  CUtensorMap lanes, columns, out;
};

// BN: columns of a tile.  WGS: groups of four warps that add up, each BN / WGS columns.
template <int BN, int WGS, Mode M>
struct LinearShape {
  static constexpr bool kSwap = M == Mode::kFeatures, kPair = M == Mode::kPair;
  static constexpr int kLoaded = kPair ? BN / 2 : BN;  // rows of the second operand that a CTA loads
  static constexpr int kStageBytes = (kLanes + kLoaded) * kGroup;
  static constexpr int kCtasPerSm = kSwap ? 2 : 1;
  static constexpr int kOutBytes = kSwap ? 0 : WGS * kLanes * 128;       // 128 bytes of every row, for each group of warps
  static constexpr int kScaleBytes = kSwap ? 0 : WGS * (kLanes + 4) * 32;  // twice four groups' scales, for each thread and warp
  static constexpr int kStagesThatFit = ((kCtasPerSm == 1 ? 227 : 113) * 1024 - 1024 - 1280 - kOutBytes - kScaleBytes) / kStageBytes;  // less the boundary's part and what else there is
  static constexpr int kStages = kStagesThatFit > 8 ? 8 : kStagesThatFit;
  static constexpr int kWarps = 4 * WGS, kThreads = 32 * (kWarps + 2);
  static constexpr int kColumns = BN / WGS;  // of a thread
  static constexpr int kTiles = BN == 256 ? 2 : 4;  // in TMEM, that take turns
  static constexpr int kHalves = kPair ? WGS : 1;    // of a tile that are multiplied, read and given back by themselves
  static constexpr int kHalf = BN / kHalves;
  static constexpr int kTmem = kTiles * BN;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + kOutBytes + kScaleBytes + 1024;
  static_assert(!kPair || (kHalf == kColumns && kHalf == kGroup), "a group of warps has a half, and one block's scale");
  static constexpr int kPitch = kSwap ? kLanes : kLanes + 1;  // of a column of sums, for the join; rows of it are read across, too, where they are rows of x
  static_assert(kStages >= 3 && (kPair || BN * kPitch * 4 <= kStages * kStageBytes), "a tile's sums lie where the stages were");
};

__device__ __forceinline__ void umma_f8_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// By one thread for both CTAs of a pair: rows and columns of the operands from either one's shared memory, at the same places.
__device__ __forceinline__ void umma_f8_ss_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this place in both CTAs of a pair.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// To this CTA's shared memory, with the bytes counted by a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_2d_pair(void* dst_smem, const CUtensorMap* map, int c0, int c1, uint32_t bar_of_first) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst_smem)), "l"(map),
               "r"(c0), "r"(c1), "r"(bar_of_first)
               : "memory");
}
__device__ __forceinline__ void cp_async_4(void* dst_smem, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst_smem)), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void arrive_in_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1), "r"(src) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 32 lanes x 32 columns of TMEM.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, "
      "[%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
        "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]) {
  if constexpr (N == 16) tmem_ld_16(taddr, v);
  else tmem_ld_32(taddr, v);
}

// Waits for the phase with the given parity, giving up after 2^20 tries of a microsecond each at most: about a second.  The first tries are plain ones, which come back sooner
// (509 rows of 2048 to 6144: 1 us less than without them, of 15).  (The timer takes longer to read than most of these waits, and code that may read it costs registers.)
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity) {
  uint32_t done = 0;
#pragma unroll 1
  for (int i = 0; !done && i < 64; ++i) done = mbar_try_wait(bar, parity);
#pragma unroll 1
  for (int i = 0; !done && i < (1 << 20); ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000)
        : "memory");
  return done != 0;
}
// The same by a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait_one(bar, parity)); }

__device__ __forceinline__ float bias_at(const TrisE4m3Linear& a, int n) {
  if (!a.bias) return 0.f;
  if (a.bias_dtype == TRIS_DTYPE_F32) return static_cast<const float*>(a.bias)[n];
  return a.bias_dtype == TRIS_DTYPE_F16 ? __half2float(static_cast<const __half*>(a.bias)[n]) : __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
}
__device__ __forceinline__ void store_output(const TrisE4m3Linear& a, int64_t at, float v) {
  if (a.dtype == TRIS_DTYPE_F32) static_cast<float*>(a.out)[at] = v;
  else if (a.dtype == TRIS_DTYPE_F16) static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
}

// grid (CTAs, 1, CTAs of a cluster), or (2 pairs, 1, 1) in clusters of two.  A CTA (a pair) walks over tiles; where the groups are cut among a cluster's CTAs it has one.
template <int BN, int WGS, Mode M>
__global__ void __launch_bounds__(LinearShape<BN, WGS, M>::kThreads, LinearShape<BN, WGS, M>::kCtasPerSm)
    e4m3_linear_kernel(const __grid_constant__ LinearArgs args, const __grid_constant__ LinearMaps maps) {
  using S = LinearShape<BN, WGS, M>;
  constexpr bool kSwap = S::kSwap, kPair = S::kPair;
  extern __shared__ uint4 smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem_raw) + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[S::kStages], empty[S::kStages], tile_full[S::kTiles][S::kHalves], tile_empty[S::kTiles][S::kHalves];
  __shared__ uint32_t tmem_base;
  __shared__ int timed_out;
  __shared__ __align__(16) float row_scales[2][kSwap ? BN : 4];
  __shared__ __align__(16) float biases[kSwap ? 4 : BN];
  const TrisE4m3Linear& a = args.a;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int tiles = args.row_tiles * args.feature_tiles;
  const int rank = kPair ? blockIdx.x & 1 : 0, split = gridDim.z, walker = kPair ? blockIdx.x / 2 : blockIdx.x, walkers = kPair ? gridDim.x / 2 : gridDim.x;
  const int first = blockIdx.z * args.per_cta, count = min(args.per_cta, args.groups - first);  // groups of this CTA; at least one

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < S::kTiles; ++i)
      for (int h = 0; h < S::kHalves; ++h) {
        mbar_init(&tile_full[i][h], 1);
        mbar_init(&tile_empty[i][h], S::kWarps / S::kHalves * (kPair ? 2 : 1));
      }
    fence_mbar_init();
    timed_out = 0;
  }
  if (warp == 0) {
    if constexpr (kPair) tmem_alloc_pair(&tmem_base, S::kTmem);
    else tmem_alloc(&tmem_base, S::kTmem);
  }
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();  // the other CTA's barriers are there
  tcgen05_fence_after();
  const uint32_t tmem = warp_uniform(tmem_base);
  pdl_wait();
  pdl_launch_dependents();

  // tiles in strips of 16 along the rows: what runs at one time shares rows and features
  auto place = [&](int tile, int& row_tile, int& feature_tile) {
    constexpr int kStrip = kPair ? 8 : 16;
    const int strip = tile / (kStrip * args.feature_tiles), in = tile - strip * (kStrip * args.feature_tiles);
    const int height = min(kStrip, args.row_tiles - strip * kStrip);
    feature_tile = in / height;
    row_tile = strip * kStrip + in - feature_tile * height;
  };

  int asked = 0;  // stages that the producer has asked for
  if (warp == S::kWarps) {
    if (lane == 0) {
      bool ok = true;
      for (int tile = walker; tile < tiles && ok; tile += walkers) {
        int rt, ft;
        place(tile, rt, ft);
        const int lane0 = kSwap ? ft * kLanes : (rt * (kPair ? 2 : 1) + rank) * kLanes, column0 = (kSwap ? rt : ft) * BN + rank * (S::kLoaded / S::kHalves);
        for (int g = 0; g < count; ++g, ++asked) {
          const int s = asked % S::kStages;
          if (asked >= S::kStages && !wait_one(&empty[s], (asked / S::kStages - 1) & 1)) {
            timed_out = 1;
            ok = false;
            break;
          }
          uint8_t* to = ring + s * S::kStageBytes;
          if constexpr (kPair) {
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * S::kStageBytes);  // the other CTA's bytes, too
            const uint32_t bar = in_cta(smem_u32(&full[s]), 0);
            tma_load_2d_pair(to, &maps.lanes, (first + g) * kGroup, lane0, bar);
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)  // of either half's columns one half
              tma_load_2d_pair(to + (kLanes + h * (S::kHalf / 2)) * kGroup, &maps.columns, (first + g) * kGroup, column0 + h * S::kHalf, bar);
          } else {
            mbar_arrive_expect_tx(&full[s], S::kStageBytes);
            tma_load_2d(to, &maps.lanes, (first + g) * kGroup, lane0, &full[s]);
            tma_load_2d(to + kLanes * kGroup, &maps.columns, (first + g) * kGroup, column0, &full[s]);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == S::kWarps + 1) {
    const uint32_t idesc = umma_idesc_f16(kPair ? 2 * kLanes : kLanes, S::kHalf);  // the same fields: fp32 sums, operand types 0 (here e4m3), K-major
    bool ok = true;
    int i = 0;
    for (int tile = walker; rank == 0 && tile < tiles && ok; tile += walkers) {
      for (int g = 0; g < count; ++g, ++i) {
        const int s = i % S::kStages, turn = i % S::kTiles;
        ok = wait_for(&full[s], (i / S::kStages) & 1);
        const uint32_t at = smem_u32(ring + s * S::kStageBytes);
        const uint64_t da = umma_smem_desc_sw128(at), db = umma_smem_desc_sw128(at + kLanes * kGroup);
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
          ok = ok && (i < S::kTiles || wait_for(&tile_empty[turn][h], (i / S::kTiles - 1) & 1));
          if (!ok) break;
          tcgen05_fence_after();
          if (elect_one()) {
            const uint32_t to = tmem + turn * BN + h * S::kHalf;
#pragma unroll
            for (int j = 0; j < kGroup / 32; ++j) {
              if constexpr (kPair) umma_f8_ss_pair(to, da + 2 * j, db + 2 * j + h * (S::kHalf / 2 * kGroup / 16), idesc, j > 0 ? 1u : 0u);
              else umma_f8_ss(to, da + 2 * j, db + 2 * j, idesc, j > 0 ? 1u : 0u);
            }
            if constexpr (kPair) {
              if (h == S::kHalves - 1) umma_commit_pair(&empty[s]);
              umma_commit_pair(&tile_full[turn][h]);
            } else {
              umma_commit(&empty[s]);
              umma_commit(&tile_full[turn][h]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
    if (!ok && lane == 0) timed_out = 1;
    __syncwarp();
  } else {
    const int wg = warp >> 2, in_tile = 32 * (warp & 3) + lane;  // lane of the tile
    const uint32_t from = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + wg * S::kColumns;
    constexpr int kPart = S::kColumns < 32 ? S::kColumns : 32;  // columns that leave TMEM at a time
    constexpr int kQuad = kSwap ? 1 : 4;
    uint8_t* out_stage = ring + S::kStages * S::kStageBytes + wg * kLanes * 128;
    // Scales of four groups: this thread's row's, and the weights' block's for its warp.  They are asked for by asynchronous copies of their own, four groups ahead:
    // loads to registers kept eight of them occupied, and the sums went to local memory.
    float4* x_scales = reinterpret_cast<float4*>(ring + S::kStages * S::kStageBytes + S::kOutBytes) + threadIdx.x;
    float4* w_scales = reinterpret_cast<float4*>(ring + S::kStages * S::kStageBytes + S::kOutBytes) + 2 * 32 * S::kWarps + warp;
    bool ok = true;
    int i = 0;
    for (int tile = walker; tile < tiles; tile += walkers) {
      int rt, ft;
      place(tile, rt, ft);
      // the scales of a thread's row, or of a row for each thread to pass on, and of the weights' block: kQuad groups, and the next ones on their way
      const int row = kSwap ? rt * BN + static_cast<int>(threadIdx.x) : (rt * (kPair ? 2 : 1) + rank) * kLanes + in_tile;
      const int feature0 = ft * BN + wg * S::kColumns;  // unless kSwap
      const int block = kSwap ? ft : feature0 / kGroup;
      const bool has_row = row < a.rows && (!kSwap || threadIdx.x < BN), has_block = block * kGroup < a.out_features;
      const float* xs = a.x_scales + static_cast<int64_t>(has_row ? row : 0) * a.x_scales_stride + first;
      const float* ws = a.weight_scales + static_cast<int64_t>(has_block ? block : 0) * a.weight_scales_stride + first;
      float x_next = 0.f, w_next = 0.f;
      auto ask_scales = [&](int g) {
        float4 *x_to = x_scales + (g / 4 & 1) * 32 * S::kWarps, *w_to = w_scales + (g / 4 & 1) * S::kWarps;
        if (g < count) {
          if (args.wide_scales && g + 4 <= count) {
            cp_async_16(x_to, xs + g, has_row);
            if (lane == 0) cp_async_16(w_to, ws + g);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const bool there = g + q < count;
              cp_async_4(reinterpret_cast<float*>(x_to) + q, there ? xs + g + q : xs, there && has_row);
              if (lane == 0) cp_async_4(reinterpret_cast<float*>(w_to) + q, there ? ws + g + q : ws, there);
            }
          }
        }
        cp_async_commit();
      };
      if constexpr (kSwap) {
        x_next = has_row ? xs[0] : 0.f;
        w_next = ws[0];
      } else {
        ask_scales(0);
      }
      if constexpr (!kSwap) {
        named_barrier_sync(1 + wg, 128);  // the biases of the tile before have been read
        if (in_tile < S::kColumns) biases[wg * S::kColumns + in_tile] = feature0 + in_tile < a.out_features ? bias_at(a, feature0 + in_tile) : 0.f;
        named_barrier_sync(1 + wg, 128);
      }
      float acc[S::kColumns];
#pragma unroll
      for (int c = 0; c < S::kColumns; ++c) acc[c] = 0.f;
#pragma unroll 1
      for (int g0 = 0; g0 < count; g0 += kQuad) {
        float scales[kQuad];
        if constexpr (kSwap) {
          scales[0] = x_next * w_next;
          if (g0 + 1 < count) {
            x_next = has_row ? xs[g0 + 1] : 0.f;
            w_next = ws[g0 + 1];
          }
          // two places take turns: who writes the next but one has met everybody who reads this one
          if (threadIdx.x < BN) row_scales[i & 1][threadIdx.x] = scales[0];
          named_barrier_sync(1, 32 * S::kWarps);
        } else {
          __syncwarp();  // the last four have been read
          ask_scales(g0 + 4);
          cp_async_wait<1>();
          __syncwarp();
          const float4 x = x_scales[(g0 / 4 & 1) * 32 * S::kWarps], w = w_scales[(g0 / 4 & 1) * S::kWarps];
          scales[0] = has_row ? x.x * w.x : 0.f;
          scales[kQuad - 3] = has_row ? x.y * w.y : 0.f;
          scales[kQuad - 2] = has_row ? x.z * w.z : 0.f;
          scales[kQuad - 1] = has_row ? x.w * w.w : 0.f;
        }
#pragma unroll
        for (int q = 0; q < kQuad; ++q) {
          if (g0 + q >= count) break;
          const int half = i & 1, turn = i % S::kTiles, parity = (i / S::kTiles) & 1;
          const float scale = scales[q];
          ++i;
          if (ok) ok = wait_for(&tile_full[turn][kPair ? wg : 0], parity);
          if (!ok) continue;
          tcgen05_fence_after();
#pragma unroll
          for (int c = 0; c < S::kColumns; c += kPart) {
            float v[kPart];
            tmem_ld<kPart>(from + turn * BN + c, v);
            if (c + kPart == S::kColumns) {
              tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) {
                if constexpr (kPair) arrive_in_cluster(in_cta(smem_u32(&tile_empty[turn][wg]), 0));
                else mbar_arrive(&tile_empty[turn][0]);
              }
            }
            if constexpr (kSwap) {
#pragma unroll
              for (int j = 0; j < kPart; j += 4) {
                const float4 s = *reinterpret_cast<const float4*>(&row_scales[half][c + j]);
                acc[c + j] = fmaf(v[j], s.x, acc[c + j]);
                acc[c + j + 1] = fmaf(v[j + 1], s.y, acc[c + j + 1]);
                acc[c + j + 2] = fmaf(v[j + 2], s.z, acc[c + j + 2]);
                acc[c + j + 3] = fmaf(v[j + 3], s.w, acc[c + j + 3]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < kPart; ++j) acc[c + j] = fmaf(v[j], scale, acc[c + j]);
            }
          }
        }
      }
      if (!ok) {  // a wait has run out: what is stored says so
        timed_out = 1;
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) acc[c] = NAN;
      }
      if (split > 1) {
        // the ring is idle: this CTA's only tile has been multiplied
        float* part = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) part[(wg * S::kColumns + c) * S::kPitch + in_tile] = acc[c];
      } else if constexpr (kSwap) {
        const int n = ft * kLanes + in_tile;
        if (n < a.out_features) {
          const float bias = bias_at(a, n);
#pragma unroll
          for (int c = 0; c < S::kColumns; ++c) {
            const int t = rt * BN + c;
            if (t < a.rows) store_output(a, static_cast<int64_t>(t) * a.out_stride + n, acc[c] + bias);
          }
        }
      } else if (args.store_map) {
        // 128 bytes of every row at a time, in the order that the tensor copy expects: 16-byte chunk c of row r at place c ^ (r & 7)
        auto put = [&](int chunk, uint4 v) { *reinterpret_cast<uint4*>(out_stage + in_tile * 128 + ((chunk ^ (in_tile & 7)) << 4)) = v; };
        const int row0 = row - in_tile;
        auto stage_out = [&](int c0, auto write) {
          if (in_tile == 0) tma_stores_read();
          named_barrier_sync(1 + wg, 128);
          write();
          fence_proxy_async();
          named_barrier_sync(1 + wg, 128);
          if (in_tile == 0 && feature0 + c0 < a.out_features && row0 < a.rows) tma_store_2d(&maps.out, feature0 + c0, row0, smem_u32(out_stage));
        };
        if (a.dtype == TRIS_DTYPE_F32) {
#pragma unroll
          for (int c0 = 0; c0 < S::kColumns; c0 += 32)
            stage_out(c0, [&] {
#pragma unroll
              for (int c = 0; c < 32; c += 4) {
                const float4 b = *reinterpret_cast<const float4*>(&biases[wg * S::kColumns + c0 + c]);
                put(c / 4, make_uint4(__float_as_uint(acc[c0 + c] + b.x), __float_as_uint(acc[c0 + c + 1] + b.y), __float_as_uint(acc[c0 + c + 2] + b.z), __float_as_uint(acc[c0 + c + 3] + b.w)));
              }
            });
        } else {
#pragma unroll
          for (int c0 = 0; c0 < S::kColumns; c0 += 64)
            stage_out(c0, [&] {
#pragma unroll
              for (int c = 0; c < 64; c += 8) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float2 b = *reinterpret_cast<const float2*>(&biases[wg * S::kColumns + c0 + c + 2 * k]);
                  const float x = acc[c0 + c + 2 * k] + b.x, y = acc[c0 + c + 2 * k + 1] + b.y;
                  w[k] = a.dtype == TRIS_DTYPE_F16 ? Pair<__half>::pack(x, y) : Pair<__nv_bfloat16>::pack(x, y);
                }
                put(c / 8, make_uint4(w[0], w[1], w[2], w[3]));
              }
            });
        }
      } else if (row < a.rows) {
        const int64_t at = static_cast<int64_t>(row) * a.out_stride + feature0;
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c)
          if (feature0 + c < a.out_features) store_output(a, at + c, acc[c] + biases[wg * S::kColumns + c]);
      }
    }
    if (!kSwap && in_tile == 0) tma_stores_done();
  }
  __syncthreads();
  if (timed_out) {
    if (threadIdx.x == 0 && a.status_dev) atomicExch(a.status_dev, TRIS_ERR_TIMEOUT);
    if (warp == S::kWarps && lane == 0 && rank == 0)  // copies in flight have to land before this memory is another's
      for (int s = 0; s < S::kStages && s < asked; ++s) mbar_wait_bounded(&full[s], ((asked - 1 - s) / S::kStages) & 1);
    __syncthreads();
  }
  if constexpr (kPair) {
    cluster_sync();  // neither CTA leaves, or gives back TMEM, while the other's products or barriers need it
    if (warp == 0) tmem_dealloc_pair(tmem, S::kTmem);
    return;
  }
  if (warp == 0) tmem_dealloc(tmem, S::kTmem);
  if (split == 1) return;

  // Every CTA of the cluster joins its share of the tile's columns, in the order of the CTAs.  A thread has some of them on their way, of up to four CTAs.
  // (us, and with one of a thread after the other and rows of x written across: 64 x 2048 to 6144 9.3 and 15.9, 256 x 14336 to 4096 33.5 and 45.0.)
  cluster_sync();
  if (warp < S::kWarps) {
    int rt, ft;
    place(blockIdx.x, rt, ft);
    float* const mine = reinterpret_cast<float*>(ring);
    const uint32_t local = smem_u32(ring);
    const int rows = min(a.rows - rt * (kSwap ? BN : kLanes), kSwap ? BN : kLanes), features = min(a.out_features - ft * (kSwap ? kLanes : BN), kSwap ? kLanes : BN);
    const int lanes_there = kSwap ? features : rows, columns_there = kSwap ? rows : features, share = (columns_there + split - 1) / split;
    const int in_tile = threadIdx.x % kLanes, u0 = blockIdx.z * share, u1 = min(u0 + share, columns_there);
    constexpr int kAtOnce = 4;
    for (int u = u0 + static_cast<int>(threadIdx.x) / kLanes; u < u1; u += kAtOnce * WGS) {
      float v[kAtOnce] = {};
      for (int r0 = 0; r0 < split; r0 += 4) {
        float w[4][kAtOnce];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) w[r][k] = r0 + r < split && u + k * WGS < u1 ? load_cluster(in_cta(local, r0 + r) + ((u + k * WGS) * S::kPitch + in_tile) * 4) : 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) v[k] += w[r][k];
      }
      if constexpr (kSwap) {
        if (in_tile >= lanes_there) continue;
        const int n = ft * kLanes + in_tile;
        const float bias = bias_at(a, n);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (u + k * WGS < u1) store_output(a, static_cast<int64_t>(rt * BN + u + k * WGS) * a.out_stride + n, v[k] + bias);
      } else {  // no other CTA reads this one's share
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (u + k * WGS < u1) mine[(u + k * WGS) * S::kPitch + in_tile] = v[k] + biases[u + k * WGS];
      }
    }
    if constexpr (!kSwap) {  // and out, features side by side
      named_barrier_sync(1 + WGS, 32 * S::kWarps);
      const int wide = 1 << (31 - __clz(max(1, min(32, share)))), across = threadIdx.x % wide;
      for (int row = threadIdx.x / wide; row < lanes_there; row += 32 * S::kWarps / wide)
        for (int u = u0 + across; u < u1; u += wide)
          store_output(a, static_cast<int64_t>(rt * kLanes + row) * a.out_stride + ft * BN + u, mine[u * S::kPitch + row]);
    }
  }
  cluster_sync();  // nobody leaves while another reads its shared memory
}

template <int BN, int WGS, Mode M>
int launch_linear(LinearArgs& args, int split, cudaStream_t stream) {
  using S = LinearShape<BN, WGS, M>;
  constexpr bool kSwap = S::kSwap, kPair = S::kPair;
  constexpr auto kernel = e4m3_linear_kernel<BN, WGS, M>;
  if (int st = allow_shared_memory<e4m3_linear_kernel<BN, WGS, M>>(static_cast<int>(S::kSmem))) return st;
  const TrisE4m3Linear& a = args.a;
  args.row_tiles = ceil_div(a.rows, kSwap ? BN : kPair ? 2 * kLanes : kLanes);
  args.feature_tiles = ceil_div(a.out_features, kSwap ? kLanes : BN);
  args.per_cta = ceil_div(args.groups, split);
  split = ceil_div(args.groups, args.per_cta);  // every CTA has a group
  args.wide_scales = aligned_to(a.x_scales, 16) && aligned_to(a.weight_scales, 16) && (a.rows == 1 || a.x_scales_stride % 4 == 0) &&
                     (a.out_features <= kGroup || a.weight_scales_stride % 4 == 0) && (split == 1 || args.per_cta % 4 == 0);
  LinearMaps maps;
  const bool ok = encode_bytes_map(&maps.lanes, kSwap ? a.weight : a.x, kSwap ? a.out_features : a.rows, a.in_features, kSwap ? a.weight_stride : a.x_stride, kLanes) &&
                  encode_bytes_map(&maps.columns, kSwap ? a.x : a.weight, kSwap ? a.rows : a.out_features, a.in_features, kSwap ? a.x_stride : a.weight_stride, S::kLoaded / S::kHalves);
  TRIS_REQUIRE(ok, TRIS_ERR_CUDA, "e4m3_linear: no tensor map for these matrices");
  const int elt = dtype_size(a.dtype);
  args.store_map = !kSwap && split == 1 && aligned_to(a.out, 16) && a.out_stride * elt % 16 == 0;
  if (args.store_map)
    TRIS_REQUIRE(encode_output_map(&maps.out, a.out, a.rows, a.out_features, elt, a.out_stride * elt), TRIS_ERR_CUDA, "e4m3_linear: no tensor map for the output");
  const int64_t tiles = static_cast<int64_t>(args.row_tiles) * args.feature_tiles, room = static_cast<int64_t>(sm_count()) * S::kCtasPerSm / (kPair ? 2 : 1);
  TRIS_REQUIRE(tiles < (1ll << 31) - room, TRIS_ERR_UNSUPPORTED, "e4m3_linear: more than 2^31 tiles");
  const int ctas = static_cast<int>(split > 1 || tiles < room ? tiles : room);
  if constexpr (kPair) {  // the CTAs of a pair are neighbours along x
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * ctas);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = 2;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = programmatic_launch_default() ? 2 : 1;
    TRIS_CUDA(cudaLaunchKernelEx(&cfg, kernel, args, maps));
  } else {
    TRIS_CUDA(launch_step(kernel, dim3(ctas, 1, split), dim3(S::kThreads), S::kSmem, stream, programmatic_launch_default(), split, args, maps));
  }
  return TRIS_OK;
}

// CTAs of a cluster that cut the groups of a tile among themselves: a power of two up to 8, as many as run at one time, each with `least` groups to itself.
//   kFeatures, 4: 1 x 2048 to 6144, 48 tiles of 16 groups, us: 7.4 uncut, 6.4 by two, 6.7 by three, 6.1 by four; 10.0 by six and 8.9 by eight, which no more run at
//   one time.  64 x 14336 to 4096, 32 tiles of 112 groups: 43.0 uncut, 15.6 by eight.
//   kRows, 16: its join has 128 rows.  128 x 2048 to 6144: 10.9 uncut, 14.1 by two; 128 x 14336 to 4096: 48.4 uncut, 21.1 by four.
int split_of(int64_t tiles, int room, int groups, int least) {
  int split = 1;
  while (split < 8 && 2 * tiles * split <= room && groups >= 2 * least * split) split *= 2;
  return split;
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_e4m3_linear(const TrisE4m3Linear* linear, void* stream) {
  TRIS_REQUIRE(linear, TRIS_ERR_INVALID_ARG, "e4m3_linear: null arguments");
  const TrisE4m3Linear& a = *linear;
  TRIS_REQUIRE(a.dtype == TRIS_DTYPE_F16 || a.dtype == TRIS_DTYPE_BF16 || a.dtype == TRIS_DTYPE_F32, TRIS_ERR_INVALID_ARG, "e4m3_linear: outputs are fp16, bf16 or fp32");
  TRIS_REQUIRE(!a.bias || a.bias_dtype == TRIS_DTYPE_F16 || a.bias_dtype == TRIS_DTYPE_BF16 || a.bias_dtype == TRIS_DTYPE_F32, TRIS_ERR_INVALID_ARG,
               "e4m3_linear: the bias is fp16, bf16 or fp32");
  TRIS_REQUIRE(a.rows >= 0 && a.out_features >= 0 && a.in_features >= 1, TRIS_ERR_INVALID_ARG, "e4m3_linear: negative sizes, or no columns");
  if (a.rows == 0 || a.out_features == 0) return TRIS_OK;
  TRIS_REQUIRE(a.x && a.weight && a.x_scales && a.weight_scales && a.out, TRIS_ERR_INVALID_ARG, "e4m3_linear: null x, weight, scales or out");
  TRIS_REQUIRE(a.in_features <= (1 << 30) && a.rows <= (1 << 30) && a.out_features <= (1 << 30), TRIS_ERR_UNSUPPORTED, "e4m3_linear: sizes beyond 2^30");
  TRIS_REQUIRE(aligned_to(a.x, 16) && aligned_to(a.weight, 16) && (a.rows == 1 || a.x_stride % 16 == 0) && (a.out_features == 1 || a.weight_stride % 16 == 0),
               TRIS_ERR_UNSUPPORTED, "e4m3_linear: rows of x and weight must start on 16-byte boundaries");
  const int line = ceil_div(a.in_features, 16) * 16;
  TRIS_REQUIRE((a.rows == 1 || a.x_stride >= a.in_features) && (a.out_features == 1 || a.weight_stride >= a.in_features), TRIS_ERR_INVALID_ARG,
               "e4m3_linear: rows of x or weight overlap");
  TRIS_REQUIRE(a.rows == 1 || a.out_stride >= a.out_features, TRIS_ERR_INVALID_ARG, "e4m3_linear: rows of out overlap");
  TRIS_REQUIRE(sm_count() > 0, TRIS_ERR_CUDA, "e4m3_linear: no device");
  LinearArgs args{a};
  if (a.rows == 1) args.a.x_stride = line;  // of no account, but a tensor map wants one
  if (a.out_features == 1) args.a.weight_stride = line;
  args.groups = ceil_div(a.in_features, kGroup);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  // Features along the lanes while one tile has all rows.  us, features and rows along the lanes: 64 x 2048 to 6144 9.3 and 10.5, 64 x 14336 to 4096 15.6 and 20.6, 64 x 4096 to
  // 14336 20 either way; 128 rows in two such tiles 28, 29 and 44, rows along the lanes 11, 21 and 19.  (One row as a tile of 64 columns instead of 16: 7.9 and 14.6 for 6.2 and 11.2.)
  if (a.rows <= 64) {
    const int split = split_of(ceil_div(a.out_features, kLanes), 2 * sms, args.groups, 4);
    if (a.rows <= 16) return launch_linear<16, 1, Mode::kFeatures>(args, split, s);
    if (a.rows <= 32) return launch_linear<32, 1, Mode::kFeatures>(args, split, s);
    return launch_linear<64, 1, Mode::kFeatures>(args, split, s);
  }
  const int64_t pairs = static_cast<int64_t>(ceil_div(a.rows, 2 * kLanes)) * ceil_div(a.out_features, 256);
  const int64_t small = static_cast<int64_t>(ceil_div(a.rows, kLanes)) * ceil_div(a.out_features, 128);
  // Rounds of all SMs; one of pairs takes six fifths of one of small tiles.  us, pairs and small tiles: 256 x 2048 to 6144, a round either way, 13.9 and 11.1; 512 x 2048 to 6144,
  // one round and two, 14.3 and 18.1; 768 x 14336 to 4096, one and two, 60 and 95; 8192 x 4096 to 14336, 25 and 49, at one clock 546 and 728.
  const int64_t rounds_of_pairs = (pairs + sms / 2 - 1) / (sms / 2), rounds_of_small = (small + sms - 1) / sms;
  if (a.rows > kLanes && 6 * rounds_of_pairs <= 5 * rounds_of_small) return launch_linear<256, 2, Mode::kPair>(args, 1, s);
  return launch_linear<128, 2, Mode::kRows>(args, split_of(small, sms, args.groups, 16), s);
}
