// Products of e4m3 rows with e4m3 weights, a scale for each row and 128 columns of x and for each 128 x 128 block of the weights.
//
// y[t, n] = sum_g xs[t, g] ws[n / 128, g] sum_{k in g} x[t, k] w[n, k] + bias[n].  The inner sums are products of 128 columns on the tensor cores
// (tcgen05.mma, kind::f8f6f4, fp32 accumulators in TMEM); the scales differ from one group to the next, so every group's tile leaves TMEM and is added
// to 32-bit sums in registers, times its scale.  Two TMEM tiles take turns: one is filled while the other is read.
//
// Roles: one warp asks for operands (TMA, a ring of stages), one issues the MMAs, and one or two groups of four warps add up.
//   rows many: the 128 lanes of a tile are rows of x, its columns are features.  A thread has one row and its scale.
//   rows few (kSwap): the lanes are features, the columns rows of x, so that a tile wastes nothing on rows that do not exist; a thread has one
//   feature, and the rows' scales come from shared memory.  Bound by the weights' bytes; the groups are cut among the CTAs of a cluster, whose sums
//   are joined in the order of the CTAs over distributed shared memory.
#include <type_traits>

#include "decode_step.cuh"
#include "umma.cuh"

namespace tris {

// Row-major rows of `cols` bytes, `stride` bytes apart; one copy = 128 columns of box_rows rows, 128-byte-swizzled, zeros past the matrix (tc_gemm.cu).
bool encode_bytes_map(CUtensorMap* map, const void* base, int rows, int cols, int64_t stride, int box_rows);

namespace {

constexpr int kGroup = 128;  // columns of a scale, and bytes of a swizzled line
constexpr int kLanes = 128;  // rows of a tile's first operand

struct LinearArgs {
  TrisE4m3Linear a;
  int groups;       // of K
  int per_cta;      // of them, that a CTA adds up
  int row_tiles, feature_tiles;
  int wide_store;   // whether 32 bytes of a row can be stored at once
};
struct LinearMaps {
  CUtensorMap lanes, columns;
};

// BN: columns of a tile.  WGS: groups of four warps that add up, each BN / WGS columns.
template <int BN, int WGS, bool kSwap>
struct LinearShape {
  static constexpr int kStageBytes = (kLanes + BN) * kGroup;
  static constexpr int kCtasPerSm = kSwap ? 2 : 1;
  static constexpr int kStagesThatFit = ((228 / kCtasPerSm - 2) * 1024 - 1024 - 1024) / kStageBytes;
  static constexpr int kStages = kStagesThatFit > 8 ? 8 : kStagesThatFit;
  static constexpr int kWarps = 4 * WGS, kThreads = 32 * (kWarps + 2);
  static constexpr int kColumns = BN / WGS;  // of a thread
  static constexpr int kTmem = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + 1024;
  static_assert(kStages >= 3 && BN * kLanes * 4 <= kStages * kStageBytes, "a tile's sums lie where the stages were");
};

__device__ __forceinline__ void umma_f8_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
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
__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// Neighbouring features n, n + 1, ... of one row.
template <int N>
__device__ __forceinline__ void store_features(const LinearArgs& args, int64_t row, int n, const float (&v)[N]) {
  const TrisE4m3Linear& a = args.a;
  const int64_t at = row * a.out_stride + n;
  static_assert(N % 16 == 0, "32 bytes of 16-bit numbers");
  if (args.wide_store && n + N <= a.out_features) {
#pragma unroll
    for (int i = 0; i < N; i += 16) {
      float f[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] = v[i + j] + (a.bias ? bias_at(a, n + i + j) : 0.f);
      uint32_t r[8];
      if (a.dtype == TRIS_DTYPE_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(f[8 * h + j]);
          store_32_bytes(static_cast<float*>(a.out) + at + i + 8 * h, r);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = a.dtype == TRIS_DTYPE_F16 ? Pair<__half>::pack(f[2 * j], f[2 * j + 1]) : Pair<__nv_bfloat16>::pack(f[2 * j], f[2 * j + 1]);
        store_32_bytes(static_cast<__half*>(a.out) + at + i, r);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (n + i < a.out_features) store_output(a, at + i, v[i] + bias_at(a, n + i));
  }
}

// grid (CTAs, 1, CTAs of a cluster).  A CTA walks over tiles; where the groups are cut among a cluster's CTAs it has one.
template <int BN, int WGS, bool kSwap>
__global__ void __launch_bounds__(LinearShape<BN, WGS, kSwap>::kThreads, LinearShape<BN, WGS, kSwap>::kCtasPerSm)
    e4m3_linear_kernel(const __grid_constant__ LinearArgs args, const __grid_constant__ LinearMaps maps) {
  using S = LinearShape<BN, WGS, kSwap>;
  extern __shared__ uint4 smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem_raw) + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[S::kStages], empty[S::kStages], tile_full[2], tile_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int timed_out;
  __shared__ __align__(16) float row_scales[2][kSwap ? BN : 4];
  const TrisE4m3Linear& a = args.a;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int tiles = args.row_tiles * args.feature_tiles;
  const int first = blockIdx.z * args.per_cta, count = min(args.per_cta, args.groups - first);  // groups of this CTA; at least one

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tile_full[i], 1);
      mbar_init(&tile_empty[i], S::kWarps);
    }
    fence_mbar_init();
    timed_out = 0;
  }
  if (warp == 0) tmem_alloc(&tmem_base, S::kTmem);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = warp_uniform(tmem_base);
  pdl_wait();
  pdl_launch_dependents();

  // tiles in strips of 16 along the rows: what runs at one time shares rows and features
  auto place = [&](int tile, int& row_tile, int& feature_tile) {
    constexpr int kStrip = 16;
    const int strip = tile / (kStrip * args.feature_tiles), in = tile - strip * (kStrip * args.feature_tiles);
    const int height = min(kStrip, args.row_tiles - strip * kStrip);
    feature_tile = in / height;
    row_tile = strip * kStrip + in - feature_tile * height;
  };

  int asked = 0;  // stages that the producer has asked for
  if (warp == S::kWarps) {
    if (lane == 0) {
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        int rt, ft;
        place(tile, rt, ft);
        const int lane0 = (kSwap ? ft : rt) * kLanes, column0 = (kSwap ? rt : ft) * BN;
        for (int g = 0; g < count; ++g, ++asked) {
          const int s = asked % S::kStages;
          if (asked >= S::kStages && !mbar_wait_bounded(&empty[s], (asked / S::kStages - 1) & 1)) {
            timed_out = 1;
            ok = false;
            break;
          }
          uint8_t* to = ring + s * S::kStageBytes;
          mbar_arrive_expect_tx(&full[s], S::kStageBytes);
          tma_load_2d(to, &maps.lanes, (first + g) * kGroup, lane0, &full[s]);
          tma_load_2d(to + kLanes * kGroup, &maps.columns, (first + g) * kGroup, column0, &full[s]);
        }
      }
    }
    __syncwarp();
  } else if (warp == S::kWarps + 1) {
    const uint32_t idesc = umma_idesc_f16(kLanes, BN);  // the same fields: fp32 sums, operand types 0 (here e4m3), K-major
    bool ok = true;
    int i = 0;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      for (int g = 0; g < count; ++g, ++i) {
        const int s = i % S::kStages, half = i & 1;
        ok = mbar_wait_warp(&full[s], (i / S::kStages) & 1) && (i < 2 || mbar_wait_warp(&tile_empty[half], (i / 2 - 1) & 1));
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t at = smem_u32(ring + s * S::kStageBytes);
        const uint64_t da = umma_smem_desc_sw128(at), db = umma_smem_desc_sw128(at + kLanes * kGroup);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < kGroup / 32; ++j) umma_f8_ss(tmem + half * BN, da + 2 * j, db + 2 * j, idesc, j > 0 ? 1u : 0u);
          umma_commit(&empty[s]);
          umma_commit(&tile_full[half]);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) timed_out = 1;
    __syncwarp();
  } else {
    const int wg = warp >> 2, in_tile = 32 * (warp & 3) + lane;  // lane of the tile
    const uint32_t from = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + wg * S::kColumns;
    constexpr int kPart = S::kColumns < 32 ? S::kColumns : 32;
    bool ok = true;
    int i = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      int rt, ft;
      place(tile, rt, ft);
      // the scales of a thread's row, or of a row for each thread to pass on, and of the weights' block
      const int row = kSwap ? rt * BN + static_cast<int>(threadIdx.x) : rt * kLanes + in_tile;
      const int block = kSwap ? ft : (ft * BN + wg * S::kColumns) / kGroup;
      const bool has_row = row < a.rows && (!kSwap || threadIdx.x < BN), has_block = block * kGroup < a.out_features;
      const float* xs = a.x_scales + static_cast<int64_t>(has_row ? row : 0) * a.x_scales_stride + first;
      const float* ws = a.weight_scales + static_cast<int64_t>(has_block ? block : 0) * a.weight_scales_stride + first;
      float x_next = has_row ? xs[0] : 0.f, w_next = ws[0];
      uint64_t acc[S::kColumns / 2];
#pragma unroll
      for (int c = 0; c < S::kColumns / 2; ++c) acc[c] = 0;
      for (int g = 0; g < count; ++g, ++i) {
        const int half = i & 1;
        const float scale = x_next * w_next;
        if (g + 1 < count) {
          x_next = has_row ? xs[g + 1] : 0.f;
          w_next = ws[g + 1];
        }
        if constexpr (kSwap) {
          // two places take turns: who writes the next but one has met everybody who reads this one
          if (threadIdx.x < BN) row_scales[half][threadIdx.x] = scale;
          named_barrier_sync(1, 32 * S::kWarps);
        }
        if (ok) ok = mbar_wait_warp(&tile_full[half], (i / 2) & 1);
        if (!ok) continue;
        tcgen05_fence_after();
#pragma unroll
        for (int c = 0; c < S::kColumns; c += kPart) {
          float v[kPart];
          tmem_ld<kPart>(from + half * BN + c, v);
          if (c + kPart == S::kColumns) {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tile_empty[half]);
          }
          if constexpr (kSwap) {
#pragma unroll
            for (int j = 0; j < kPart; j += 4) {
              const float4 s = *reinterpret_cast<const float4*>(&row_scales[half][c + j]);
              acc[(c + j) / 2] = fma_2(pack_2(v[j], v[j + 1]), pack_2(s.x, s.y), acc[(c + j) / 2]);
              acc[(c + j) / 2 + 1] = fma_2(pack_2(v[j + 2], v[j + 3]), pack_2(s.z, s.w), acc[(c + j) / 2 + 1]);
            }
          } else {
            const uint64_t s = pack_2(scale, scale);
#pragma unroll
            for (int j = 0; j < kPart; j += 2) acc[(c + j) / 2] = fma_2(pack_2(v[j], v[j + 1]), s, acc[(c + j) / 2]);
          }
        }
      }
      if (!ok) {  // a wait has run out: what is stored says so
        timed_out = 1;
#pragma unroll
        for (int c = 0; c < S::kColumns / 2; ++c) acc[c] = pack_2(NAN, NAN);
      }
      auto sum = [&](int c) {
        float lo, hi;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(acc[c / 2]));
        return c & 1 ? hi : lo;
      };
      if (gridDim.z > 1) {
        // the ring is idle: this CTA's only tile has been multiplied
        float* part = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) part[(wg * S::kColumns + c) * kLanes + in_tile] = sum(c);
      } else if constexpr (kSwap) {
        const int n = ft * kLanes + in_tile;
        if (n < a.out_features) {
          const float bias = bias_at(a, n);
#pragma unroll
          for (int c = 0; c < S::kColumns; ++c) {
            const int t = rt * BN + c;
            if (t < a.rows) store_output(a, static_cast<int64_t>(t) * a.out_stride + n, sum(c) + bias);
          }
        }
      } else if (row < a.rows) {
#pragma unroll
        for (int c = 0; c < S::kColumns; c += 16) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = sum(c + j);
          store_features(args, row, ft * BN + wg * S::kColumns + c, v);
        }
      }
    }
  }
  __syncthreads();
  if (timed_out) {
    if (threadIdx.x == 0 && a.status_dev) atomicExch(a.status_dev, TRIS_ERR_TIMEOUT);
    if (warp == S::kWarps && lane == 0)  // copies in flight have to land before this memory is another's
      for (int s = 0; s < S::kStages && s < asked; ++s) mbar_wait_bounded(&full[s], ((asked - 1 - s) / S::kStages) & 1);
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem, S::kTmem);
  if (gridDim.z == 1) return;

  // every CTA of the cluster joins its share of the tile's columns, in the order of the CTAs
  cluster_sync();
  if (warp < S::kWarps) {
    int rt, ft;
    place(blockIdx.x, rt, ft);
    const uint32_t local = smem_u32(ring);
    const int in_tile = threadIdx.x % kLanes, part = threadIdx.x / kLanes;
    constexpr int kUnit = kSwap ? 1 : 16;  // columns at a time
    for (int u = blockIdx.z * WGS + part; u < BN / kUnit; u += gridDim.z * WGS) {
      const int t = kSwap ? rt * BN + u : rt * kLanes + in_tile, n = kSwap ? ft * kLanes + in_tile : ft * BN + u * kUnit;
      if (t >= a.rows || n >= a.out_features) continue;
      float v[kUnit];
#pragma unroll
      for (int j = 0; j < kUnit; ++j) v[j] = 0.f;
      for (int r = 0; r < static_cast<int>(gridDim.z); ++r) {
        const uint32_t there = in_cta(local, r);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) v[j] += load_cluster(there + ((u * kUnit + j) * kLanes + in_tile) * 4);
      }
      if constexpr (kSwap) store_output(a, static_cast<int64_t>(t) * a.out_stride + n, v[0] + bias_at(a, n));
      else store_features(args, t, n, v);
    }
  }
  cluster_sync();  // nobody leaves while another reads its shared memory
}

template <int BN, int WGS, bool kSwap>
int launch_linear(LinearArgs& args, int split, cudaStream_t stream) {
  using S = LinearShape<BN, WGS, kSwap>;
  constexpr auto kernel = e4m3_linear_kernel<BN, WGS, kSwap>;
  if (int st = allow_shared_memory<e4m3_linear_kernel<BN, WGS, kSwap>>(static_cast<int>(S::kSmem))) return st;
  const TrisE4m3Linear& a = args.a;
  args.row_tiles = ceil_div(a.rows, kSwap ? BN : kLanes);
  args.feature_tiles = ceil_div(a.out_features, kSwap ? kLanes : BN);
  args.per_cta = ceil_div(args.groups, split);
  split = ceil_div(args.groups, args.per_cta);  // every CTA has a group
  LinearMaps maps;
  const bool ok = encode_bytes_map(&maps.lanes, kSwap ? a.weight : a.x, kSwap ? a.out_features : a.rows, a.in_features, kSwap ? a.weight_stride : a.x_stride, kLanes) &&
                  encode_bytes_map(&maps.columns, kSwap ? a.x : a.weight, kSwap ? a.rows : a.out_features, a.in_features, kSwap ? a.x_stride : a.weight_stride, BN);
  TRIS_REQUIRE(ok, TRIS_ERR_CUDA, "e4m3_linear: no tensor map for these matrices");
  const int64_t tiles = static_cast<int64_t>(args.row_tiles) * args.feature_tiles, room = static_cast<int64_t>(sm_count()) * S::kCtasPerSm;
  TRIS_REQUIRE(tiles < (1ll << 31) - room, TRIS_ERR_UNSUPPORTED, "e4m3_linear: more than 2^31 tiles");
  const int ctas = static_cast<int>(split > 1 || tiles < room ? tiles : room);
  TRIS_CUDA(launch_step(kernel, dim3(ctas, 1, split), dim3(S::kThreads), S::kSmem, stream, programmatic_launch_default(), split, args, maps));
  return TRIS_OK;
}

// CTAs of a cluster that cut the groups of a tile among themselves: as many as run at one time, up to 8.
int split_of(int64_t tiles, int room, int groups) {
  int split = 1;
  while (split < 8 && tiles * (split + 1) <= room && groups >= 2 * (split + 1)) ++split;
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
  args.wide_store = aligned_to(a.out, 32) && a.out_stride * dtype_size(a.dtype) % 32 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  if (a.rows <= 64) {
    const int split = split_of(ceil_div(a.out_features, kLanes), 2 * sms, args.groups);
    if (a.rows <= 16) return launch_linear<16, 1, true>(args, split, s);
    if (a.rows <= 32) return launch_linear<32, 1, true>(args, split, s);
    return launch_linear<64, 1, true>(args, split, s);
  }
  const int64_t row_tiles = ceil_div(a.rows, kLanes), large = row_tiles * ceil_div(a.out_features, 256), small = row_tiles * ceil_div(a.out_features, 128);
  // time of the whole, in MMAs of 128 x 128: large tiles unless small ones leave fewer SMs without work
  const int64_t t_large = (large + sms - 1) / sms * 2, t_small = (small + sms - 1) / sms;
  if (t_large <= t_small) return launch_linear<256, 2, false>(args, 1, s);
  return launch_linear<128, 2, false>(args, split_of(small, sms, args.groups), s);
}
