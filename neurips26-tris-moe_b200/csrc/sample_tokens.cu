// A token drawn from each row of logits: temperature, top-k, top-p and min-p, by given random numbers.
//
// In the order of falling logits (equal ones by rising index) a token is kept while its place is below k, while the weights ahead of it are less than
// p times those of the first k, and while its weight exp((z - max) / T) is at least min_p; of those kept, in the order of the vocabulary, the first
// whose running sum exceeds u times the whole is drawn.  All three ends are one place in the order, so no order is made: a histogram over max - z
// finds the interval in which the k-th token lies, or the one that ends the share p, and the few tokens of that interval are ranked one against another.
//
// Weights are integers, exp in units of 2^-46 of the largest (fewer bits for vocabularies beyond 65536): their sums are exact, so neither the order of
// atomics nor that of threads counts, and u falls where it does in 64-bit arithmetic.  With 32-bit exponentials one row in some hundred would
// draw a neighbour.  A row belongs to one CTA or, for few rows, to a cluster that cuts the vocabulary and reads one another's histograms; its logits are
// read from memory once and some three times from L1.
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 1024, kBins = kThreads, kFew = 256;
constexpr int kMostCtas = 8;  // of a cluster
constexpr int kTable = 256;   // powers 2^(i / kTable)

struct SampleArgs {
  TrisSampleTokens s;
  int slice;  // logits of a CTA, a multiple of 8
  int wide;   // whether four logits can be read at once
  int bits;   // the largest weight is 2^bits
  int chunk;  // logits whose weights are added up by a warp, a multiple of 128
};

struct Histogram {
  uint32_t count[kBins], low[kBins], high[kBins];  // tokens, and the sum of their weights
};
struct Found {
  int bin;
  uint32_t tokens, count_before;
  uint64_t weight_before;
};

__device__ __forceinline__ uint32_t load_cluster_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t load_cluster_u64(uint32_t at) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}

// What stands for a token in the order: the logit's bits, brought into the order of unsigned numbers, then the lower index first.
__device__ __forceinline__ uint64_t place_of(float z, uint32_t token) {
  const uint32_t b = __float_as_uint(z + 0.f);  // -0 is 0
  return (static_cast<uint64_t>(b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u)) << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float logit_of(uint64_t place) {
  const uint32_t k = static_cast<uint32_t>(place >> 32);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Sum of the threads' values ahead of each, and all of them.  red has a place for every warp; it may be used again after a barrier.
template <typename N>
__device__ __forceinline__ N scan(N v, N* red, N& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N upto = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const N below = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += below;
  }
  if (lane == 31) red[warp] = upto;
  __syncthreads();
  N sum = red[lane];
  static_assert(kThreads == 1024, "a lane for every warp");
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const N below = __shfl_up_sync(0xFFFFFFFFu, sum, d);
    if (lane >= d) sum += below;
  }
  total = __shfl_sync(0xFFFFFFFFu, sum, 31);
  const N before = __shfl_sync(0xFFFFFFFFu, sum, warp ? warp - 1 : 0);
  return upto - v + (warp ? before : 0);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_tokens_kernel(const __grid_constant__ SampleArgs args) {
  __shared__ __align__(16) Histogram first, finer;
  __shared__ double powers[kTable];
  __shared__ uint64_t lists[2][kFew];  // tokens of the interval that was found, of this CTA
  __shared__ ulonglong2 merged[kFew];  // and of all, each with its weight
  __shared__ uint32_t listed[2];
  __shared__ uint64_t ends[2][2];  // the last and the first of them in the order, where they are many
  __shared__ __align__(8) float extremes[2];
  __shared__ uint64_t part, red64[32];
  __shared__ uint32_t red32[32], best;
  __shared__ Found found;
  __shared__ uint64_t cut, cut_weight;
  const TrisSampleTokens& s = args.s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y;
  const int ctas = gridDim.z, v0 = blockIdx.z * args.slice, n = max(0, min(args.slice, s.vocab - v0));
  auto meet = [&] {
    if (ctas > 1) cluster_sync();
    else __syncthreads();
  };
  auto there = [&](const void* mine, int r) { return in_cta(smem_u32(mine), r); };

  if (tid < kTable) powers[tid] = exp2(static_cast<double>(tid) / kTable);
  first.count[tid] = first.low[tid] = first.high[tid] = 0;
  if (tid < 2) {
    listed[tid] = 0;
    ends[tid][0] = ~0ull;
    ends[tid][1] = 0;
  }
  if (tid == 0) best = 0xFFFFFFFFu;
  pdl_wait();
  pdl_launch_dependents();
  const T* in = static_cast<const T*>(s.logits) + row * s.logits_stride + v0;
  // Four logits of the slice; what is not there, and what is not a number, is -inf.
  auto fetch = [&](int at, float (&z)[4]) {
    if (args.wide && at + 4 <= n) {
      if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4*>(in + at);
        z[0] = f.x, z[1] = f.y, z[2] = f.z, z[3] = f.w;
      } else {
        const uint2 raw = *reinterpret_cast<const uint2*>(in + at);
        const float2 lo = Pair<T>::unpack(raw.x), hi = Pair<T>::unpack(raw.y);
        z[0] = lo.x, z[1] = lo.y, z[2] = hi.x, z[3] = hi.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] = at + k < n ? to_float(in[at + k]) : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = z[k] == z[k] ? z[k] : -INFINITY;
  };
  const float temperature = s.temperature ? s.temperature[row] : 1.f;
  const int top_k = s.top_k ? s.top_k[row] : 0;
  const float top_p = s.top_p ? s.top_p[row] : 1.f, min_p = s.min_p ? s.min_p[row] : 0.f;

  // The largest logit, and the smallest that is one.
  float top = -INFINITY, low = INFINITY;
#pragma unroll 4
  for (int at = 4 * tid; at < n; at += 4 * kThreads) {
    float z[4];
    fetch(at, z);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      top = fmaxf(top, z[k]);
      if (z[k] > -INFINITY) low = fminf(low, z[k]);
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, d));
  }
  if (lane == 0) red64[warp] = (static_cast<uint64_t>(__float_as_uint(top)) << 32) | __float_as_uint(low);
  __syncthreads();
  top = __uint_as_float(static_cast<uint32_t>(red64[lane] >> 32));
  low = __uint_as_float(static_cast<uint32_t>(red64[lane]));
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, d));
  }
  if (ctas > 1) {
    if (tid == 0) extremes[0] = top, extremes[1] = low;
    cluster_sync();
    for (int r = 0; r < ctas; ++r) {
      const float2 other = load_cluster_2(there(extremes, r));
      top = fmaxf(top, other.x);
      low = fminf(low, other.y);
    }
  }
  if (top == -INFINITY) {  // nothing can be drawn
    if (blockIdx.z == 0 && tid == 0) s.out[row] = -1;
    meet();
    return;
  }

  if (!(temperature > 0.f) || top_k == 1 || top_p <= 0.f) {  // the first of the largest
    uint32_t mine = 0xFFFFFFFFu;
    for (int at = 4 * tid; at < n && mine == 0xFFFFFFFFu; at += 4 * kThreads) {
      float z[4];
      fetch(at, z);
#pragma unroll
      for (int k = 3; k >= 0; --k)
        if (z[k] == top) mine = v0 + at + k;
    }
    mine = __reduce_min_sync(0xFFFFFFFFu, mine);
    if (lane == 0 && mine != 0xFFFFFFFFu) atomicMin(&best, mine);
    meet();
    if (blockIdx.z == 0 && tid == 0) {
      uint32_t token = best;
      for (int r = 1; r < ctas; ++r) token = min(token, load_cluster_u32(there(&best, r)));
      s.out[row] = token;
    }
    meet();
    return;
  }

  // exp((z - top) / temperature) in units of 2^-bits.
  const double per_unit = 1.4426950408889634074 / static_cast<double>(temperature);
  auto weight_of = [&](float z) -> uint64_t {
    if (z == top) return 1ull << args.bits;
    // (rounded one by one, so that every place of the code finds the same weight)
    const double y = __dmul_rn(static_cast<double>(z) - static_cast<double>(top), per_unit);
    if (!(y > -60.)) return 0;
    constexpr double kShift = 6755399441055744. / kTable;  // 1.5 * 2^52 / kTable: the last bit is 1 / kTable
    const double t = __dadd_rn(y, kShift);
    const int64_t steps = static_cast<int32_t>(__double_as_longlong(t));  // y * kTable, rounded
    const double f = __dsub_rn(y, __dsub_rn(t, kShift));                   // up to 1 / (2 kTable)
    // 2^f = sum of (f ln 2)^i / i!
    const double p = fma(fma(fma(fma(9.6181291076284772e-3, f, 5.5504108664821580e-2), f, 2.4022650695910072e-1), f, 6.9314718055994531e-1), f, 1.);
    const double w = __dmul_rn(powers[steps & (kTable - 1)], p);
    const int64_t exponent = (steps >> 8) + args.bits;  // w * 2^exponent: the exponent's bits are added to
    if (exponent < -2) return 0;
    return static_cast<uint64_t>(__double2ull_rn(__longlong_as_double(__double_as_longlong(w) + (exponent << 52))));
  };
  static_assert(kTable == 256, "steps >> 8");
  const uint64_t least = min_p > 0.f ? static_cast<uint64_t>(ceil(fmin(static_cast<double>(min_p), 1.) * static_cast<double>(1ull << args.bits))) : 0;

  uint64_t from = 0;  // the last place that is kept
  const bool by_count = top_k > 0 && top_k < s.vocab, by_weight = top_p < 1.f;
  if (by_count || by_weight) {
    const float range = fminf(40.f * temperature, top - low);
    const float per_bin = range > 0.f ? fminf(kBins / range, 1e30f) : 0.f;
    auto bin_of = [&](float z) { return z == top ? 0 : static_cast<int>(fminf((top - z) * per_bin, kBins - 1.f)); };
    auto enter = [&](Histogram& h, int bin, uint64_t w) {
      atomicAdd(&h.count[bin], 1u);
      const uint32_t w_low = static_cast<uint32_t>(w);
      uint32_t w_high = static_cast<uint32_t>(w >> 32);
      if (w_low) w_high += atomicAdd(&h.low[bin], w_low) + w_low < w_low;  // and what is carried
      if (w_high) atomicAdd(&h.high[bin], w_high);
    };
    // All CTAs' tokens and weights of bin `tid`, and those ahead of it.
    uint32_t count, count_before, all_tokens;
    uint64_t weight, weight_before, all_weight;
    auto gather = [&](const Histogram& h) {
      count = 0;
      weight = 0;
      for (int r = 0; r < ctas; ++r) {
        count += load_cluster_u32(there(&h.count[tid], r));
        weight += (static_cast<uint64_t>(load_cluster_u32(there(&h.high[tid], r))) << 32) + load_cluster_u32(there(&h.low[tid], r));
      }
      count_before = scan(count, red32, all_tokens);
      weight_before = scan(weight, red64, all_weight);
      __syncthreads();
    };
#pragma unroll 2
    for (int at = 4 * tid; at < n; at += 4 * kThreads) {
      float z[4];
      fetch(at, z);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (z[k] > -INFINITY) {
          const uint64_t w = by_weight ? weight_of(z[k]) : 0;
          if (by_count || w) enter(first, bin_of(z[k]), w);
        }
    }
    meet();
    gather(first);
    const uint32_t count0 = count, count_before0 = count_before;
    const uint64_t weight0 = weight, weight_before0 = weight_before;

    // The place of the token that is the count_to-th, or with which the weights reach weight_to; and the weights up to and with it.
    auto select = [&](int use, uint32_t count_to, uint64_t weight_to, uint64_t& upto) -> uint64_t {
      count = count0, count_before = count_before0, weight = weight0, weight_before = weight_before0;
      uint64_t high = 0, shift = 0;  // of a finer histogram: the first place, and bits of a bin
      uint64_t interval_low = 0, interval_high = 0;
      bool finer_bins = false;
      // every turn leaves a 1024th of the places, of which there are less than 2^62
      for (int turn = 0; turn < 8; ++turn) {
        const bool here = count_to ? count_before < count_to && count_before + count >= count_to : weight_before < weight_to && weight_before + weight >= weight_to;
        if (here) found = {tid, count, count_before, weight_before};
        __syncthreads();
        const Found f = found;
        if (finer_bins) {
          interval_high = high - (static_cast<uint64_t>(f.bin) << shift);
          const uint64_t width = (1ull << shift) - 1;
          interval_low = interval_high - interval_low < width ? interval_low : interval_high - width;
        }
        auto inside = [&](float z, uint64_t at) { return z > -INFINITY && (finer_bins ? at >= interval_low && at <= interval_high : bin_of(z) == f.bin); };
        const bool few = f.tokens <= kFew;
        if (!few && finer_bins) {
          // the interval's bounds are known
        } else {
          uint64_t lo = ~0ull, hi = 0;
#pragma unroll 2
          for (int at = 4 * tid; at < n; at += 4 * kThreads) {
            float z[4];
            fetch(at, z);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t place = place_of(z[k], v0 + at + k);
              if (!inside(z[k], place) || (!count_to && weight_of(z[k]) == 0)) continue;
              if (few) {
                const uint32_t i = atomicAdd(&listed[use], 1u);
                if (i < kFew) lists[use][i] = place;
              }
              lo = min(lo, place);
              hi = max(hi, place);
            }
          }
          if (!few) {
#pragma unroll
            for (int d = 16; d; d >>= 1) {
              lo = min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
              hi = max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
            }
            if (lane == 0) {
              atomicMin(reinterpret_cast<unsigned long long*>(&ends[use][0]), lo);
              atomicMax(reinterpret_cast<unsigned long long*>(&ends[use][1]), hi);
            }
          }
          meet();
          if (few) {
            // every CTA ranks them all
            int ahead = 0;
            for (int r = 0; r < ctas; ++r) {
              const int many = min(static_cast<int>(load_cluster_u32(there(&listed[use], r))), kFew - ahead);
              if (tid >= ahead && tid < ahead + many) {
                const uint64_t place = load_cluster_u64(there(&lists[use][tid - ahead], r));
                merged[tid] = make_ulonglong2(place, weight_of(logit_of(place)));
              }
              ahead += many;
            }
            __syncthreads();
            if (tid < ahead) {
              const uint64_t mine = merged[tid].x, own = merged[tid].y;
              uint64_t sum = f.weight_before;
              uint32_t rank = f.count_before;
              for (int i = 0; i < ahead; ++i) {
                const ulonglong2 other = merged[i];
                rank += other.x > mine;
                sum += other.x > mine ? other.y : 0;
              }
              if (count_to ? rank + 1 == count_to : sum < weight_to && sum + own >= weight_to) {
                cut = mine;
                cut_weight = sum + own;
              }
            }
            __syncthreads();
            const uint64_t place = cut;
            upto = cut_weight;
            __syncthreads();
            return place;
          }
          interval_low = ~0ull;
          interval_high = 0;
          for (int r = 0; r < ctas; ++r) {
            interval_low = min(interval_low, load_cluster_u64(there(&ends[use][0], r)));
            interval_high = max(interval_high, load_cluster_u64(there(&ends[use][1], r)));
          }
        }
        // too many: a histogram of this interval alone
        finer_bins = true;
        high = interval_high;
        shift = 64 - __clzll(static_cast<long long>(interval_high - interval_low));
        shift = shift > 10 ? shift - 10 : 0;
        static_assert(kBins == 1 << 10, "bins of a finer histogram");
        finer.count[tid] = finer.low[tid] = finer.high[tid] = 0;
        __syncthreads();
#pragma unroll 2
        for (int at = 4 * tid; at < n; at += 4 * kThreads) {
          float z[4];
          fetch(at, z);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t place = place_of(z[k], v0 + at + k);
            if (z[k] > -INFINITY && place >= interval_low && place <= interval_high) {
              const uint64_t w = by_weight ? weight_of(z[k]) : 0;
              if (count_to || w) enter(finer, static_cast<int>((high - place) >> shift), w);
            }
          }
        }
        meet();
        gather(finer);
        count_before += f.count_before;
        weight_before += f.weight_before;
        meet();
      }
      return 0;
    };

    uint64_t share = all_weight;
    const uint32_t tokens = all_tokens;
    if (by_count && static_cast<uint32_t>(top_k) < tokens) from = select(0, top_k, 0, share);
    if (by_weight) {
      const double to = static_cast<double>(top_p) * static_cast<double>(share);
      const uint64_t reach = to <= 1. ? 1 : static_cast<uint64_t>(ceil(to));
      uint64_t upto;
      from = max(from, select(1, 0, reach < share ? reach : share, upto));
    }
  }

  // Sums of what is kept, chunk by chunk; a warp has a chunk.
  auto kept_weight = [&](float z, int at) -> uint64_t {
    if (!(z > -INFINITY) || place_of(z, v0 + at) < from) return 0;
    const uint64_t w = weight_of(z);
    return w >= least ? w : 0;
  };
  if (tid == 0) part = 0;
  uint64_t* sums = reinterpret_cast<uint64_t*>(&finer);  // kThreads of them
  static_assert(sizeof(Histogram) >= kThreads * sizeof(uint64_t), "sums");
  __syncthreads();
  sums[tid] = 0;
  __syncthreads();
  for (int c = warp; c * args.chunk < n; c += kThreads / 32) {
    uint64_t sum = 0;
    for (int at = c * args.chunk + 4 * lane; at < min(n, (c + 1) * args.chunk); at += 128) {
      float z[4];
      fetch(at, z);
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += kept_weight(z[k], at + k);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) sums[c] = sum;
  }
  __syncthreads();
  uint64_t mine = sums[tid], all;
  const uint64_t before = scan(mine, red64, all);
  uint64_t ahead = 0, whole = all;
  if (ctas > 1) {
    if (tid == 0) part = all;
    cluster_sync();
    whole = 0;
    for (int r = 0; r < ctas; ++r) {
      const uint64_t other = load_cluster_u64(there(&part, r));
      if (r < static_cast<int>(blockIdx.z)) ahead += other;
      whole += other;
    }
  }
  const double u = fmax(static_cast<double>(s.random[row]), 0.);  // not a number: 0
  const double at_sum = floor(u * static_cast<double>(whole));
  const uint64_t target = at_sum >= static_cast<double>(whole) ? whole - 1 : min(static_cast<uint64_t>(at_sum), whole - 1);
  if (tid == 0) found.bin = -1;
  __syncthreads();
  if (target >= ahead + before && target < ahead + before + mine) {
    found.bin = tid;
    found.weight_before = target - ahead - before;
  }
  __syncthreads();
  if (warp == 0 && found.bin >= 0) {
    uint64_t rest = found.weight_before;  // of the chunk's weights, ahead of what is drawn
    for (int at = found.bin * args.chunk + 4 * lane;; at += 128) {
      float z[4];
      uint64_t w[4], sum = 0;
      fetch(at, z);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = at + k < n ? kept_weight(z[k], at + k) : 0;
        sum += w[k];
      }
      uint64_t upto = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint64_t below = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += below;
      }
      const bool here = upto > rest && upto - sum <= rest;
      if (here) {
        uint64_t left = rest - (upto - sum);
        int k = 0;
        while (k < 3 && left >= w[k]) left -= w[k++];
        s.out[row] = v0 + at + k;
      }
      if (__any_sync(0xFFFFFFFFu, here) || at - 4 * lane + 128 >= n) break;
      rest -= __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }
  meet();  // nobody leaves while another reads its shared memory
}

template <typename T>
int launch_sample(SampleArgs& a, cudaStream_t stream) {
  // few rows: a cluster for each, as large as all of them run at one time
  int ctas = 1;
  while (ctas < kMostCtas && 2 * ctas * a.s.rows <= sm_count() && a.s.vocab > 2 * ctas * kThreads) ctas *= 2;
  a.slice = (ceil_div(a.s.vocab, ctas) + 7) / 8 * 8;
  a.chunk = 128;
  while (static_cast<int64_t>(a.chunk) * kThreads < a.slice) a.chunk *= 2;
  TRIS_CUDA(launch_step(sample_tokens_kernel<T>, dim3(1, a.s.rows, ctas), dim3(kThreads), 0, stream, programmatic_launch_default(), ctas, a));
  return TRIS_OK;
}

}  // namespace
}  // namespace tris

using namespace tris;

extern "C" int tris_sample_tokens(const TrisSampleTokens* args, void* stream) {
  TRIS_REQUIRE(args, TRIS_ERR_INVALID_ARG, "sample_tokens: null arguments");
  const TrisSampleTokens& s = *args;
  TRIS_REQUIRE(s.dtype == TRIS_DTYPE_F16 || s.dtype == TRIS_DTYPE_BF16 || s.dtype == TRIS_DTYPE_F32, TRIS_ERR_INVALID_ARG, "sample_tokens: logits are fp16, bf16 or fp32");
  TRIS_REQUIRE(s.rows >= 0 && s.vocab >= 1, TRIS_ERR_INVALID_ARG, "sample_tokens: negative sizes, or no vocabulary");
  if (s.rows == 0) return TRIS_OK;
  TRIS_REQUIRE(s.rows <= 65535 && s.vocab <= (1 << 28), TRIS_ERR_UNSUPPORTED, "sample_tokens: more than 65535 rows or 2^28 tokens");
  TRIS_REQUIRE(s.logits && s.random && s.out, TRIS_ERR_INVALID_ARG, "sample_tokens: null logits, random or out");
  SampleArgs a{s};
  a.wide = aligned_to(s.logits, 4 * dtype_size(s.dtype)) && (s.rows == 1 || s.logits_stride % 4 == 0);
  a.bits = 46;  // 2^bits * vocab stays below 2^62
  while (a.bits > 8 && (static_cast<int64_t>(s.vocab) << a.bits) >= (1ll << 62)) --a.bits;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return s.dtype == TRIS_DTYPE_F16 ? launch_sample<__half>(a, st) : s.dtype == TRIS_DTYPE_BF16 ? launch_sample<__nv_bfloat16>(a, st) : launch_sample<float>(a, st);
}
