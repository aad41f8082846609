// A token drawn from each row of logits: temperature, top-k, top-p and min-p, by given random numbers.
//
// In the order of falling logits (equal ones by rising index) a token is kept while its place is below k, while the weights ahead of it are less than
// p times those of the first k, and while its weight exp((z - max) / T) is at least min_p; of those kept, in the order of the vocabulary, the first
// whose running sum exceeds u times the whole is drawn.  All three ends are one place in the order, so no order is made: a histogram over max - z
// finds the interval in which the k-th token lies, or the one that ends the share p, and the few tokens of that interval are ranked one against another.
// Where the first k tokens are few, all that follows is done on a list of them.
//
// Weights are integers, exp in units of 2^-46 of the largest (fewer bits for vocabularies beyond 65536): their sums are exact, so neither the order of
// atomics nor that of threads counts, and u falls where it does in 64-bit arithmetic.  (With 32-bit exponentials one row in some hundred would
// draw a neighbour.)  A row belongs to one CTA or, for few rows, to a cluster that cuts the vocabulary and reads one another's histograms; its logits are
// read from memory once and two or three times from L1.  Bound by instructions: some 30 for a weight, of which every token has one and every kept token two.
// Rows of 50304 in fp32, top-k, top-p and min-p at once: 128 of them 50 us, one 13.4 - of which the start and its table take 1.3, the largest logit 1.7, the histogram by count 2.4,
// its sums 1.3, the list of the k 1.7, its weights 2.0 and what is drawn of it 3.
#include "decode_step.cuh"

namespace tris {
namespace {

constexpr int kThreads = 1024, kBins = kThreads, kFew = 512;
constexpr int kMostCtas = 8;   // of a cluster
constexpr int kTable = 1024;   // powers 2^(i / kTable)

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
  __shared__ union Buffer {
    Histogram bins;
    float kept[kThreads / 32][128];  // logits of a warp's tokens, one after the other
  } buffer;
  __shared__ double powers[kTable];
  __shared__ union Second {
    uint64_t sums[kThreads];   // of a chunk's weights
    ulonglong2 merged[kFew];  // tokens of the interval that was found, of all CTAs, each with its weight
  } second;
  __shared__ uint64_t red64[32], part;
  __shared__ uint64_t lists[2][kFew];  // those of this CTA
  __shared__ uint32_t listed[2], red32[32], best;
  __shared__ uint64_t ends[2][2];  // the last and the first of them in the order
  __shared__ __align__(8) float extremes[2];
  __shared__ Found found;
  __shared__ uint64_t cut;
  Histogram& bins = buffer.bins;
  auto& sums = second.sums;
  auto& merged = second.merged;
  const TrisSampleTokens& s = args.s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y;
  const int ctas = gridDim.z, v0 = blockIdx.z * args.slice, n = max(0, min(args.slice, s.vocab - v0));
  auto meet = [&] {
    if (ctas > 1) cluster_sync();
    else __syncthreads();
  };
  auto there = [&](const void* mine, int r) { return in_cta(smem_u32(mine), r); };
  // The same word of every CTA of the cluster; all of them are asked for before the first has arrived.
  auto words_of_all = [&](const uint32_t* mine, uint32_t (&v)[kMostCtas]) {
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) v[r] = 0;
    if (ctas == 1) {
      v[0] = *mine;
      return;
    }
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r)
      if (r < ctas) v[r] = load_cluster_u32(there(mine, r));
  };
  auto clear_bins = [&] { bins.count[tid] = bins.low[tid] = bins.high[tid] = 0; };

  powers[tid] = exp2(static_cast<double>(tid) / kTable);
  static_assert(kTable == kThreads, "a power to a thread");
  clear_bins();
  if (tid < 2) {
    listed[tid] = 0;
    ends[tid][0] = ~0ull;
    ends[tid][1] = 0;
  }
  if (tid == 0) best = 0xFFFFFFFFu;
  pdl_wait();
  pdl_launch_dependents();
  const T* in = static_cast<const T*>(s.logits) + row * s.logits_stride + v0;
  // Four logits of the slice, -inf where there is none.  What is not a number fails every comparison below.
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
  };
  const float temperature = s.temperature ? s.temperature[row] : 1.f;
  const int top_k = s.top_k ? s.top_k[row] : 0;
  const float top_p = s.top_p ? s.top_p[row] : 1.f, min_p = s.min_p ? s.min_p[row] : 0.f;
  const double u = fmax(static_cast<double>(s.random[row]), 0.);  // not a number: 0

  // The largest logit, and the smallest.
  float top = -INFINITY, low = INFINITY;
#pragma unroll 4
  for (int at = 4 * tid; at < n; at += 4 * kThreads) {
    float z[4];
    fetch(at, z);
    top = fmaxf(fmaxf(fmaxf(top, z[0]), fmaxf(z[1], z[2])), z[3]);
    low = fminf(fminf(fminf(low, z[0]), fminf(z[1], z[2])), z[3]);
  }
  auto all_lanes = [&] {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
      low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, d));
    }
  };
  all_lanes();
  if (lane == 0) red64[warp] = (static_cast<uint64_t>(__float_as_uint(top)) << 32) | __float_as_uint(low);
  __syncthreads();
  top = __uint_as_float(static_cast<uint32_t>(red64[lane] >> 32));
  low = __uint_as_float(static_cast<uint32_t>(red64[lane]));
  all_lanes();
  if (ctas > 1) {
    if (tid == 0) extremes[0] = top, extremes[1] = low;
    cluster_sync();
    float2 other = make_float2(top, low);
    if (lane < ctas) other = load_cluster_2(there(extremes, lane));
    top = other.x, low = other.y;
    all_lanes();
  }
  if (top == -INFINITY) {  // nothing can be drawn
    if (blockIdx.z == 0 && tid == 0) s.out[row] = -1;
    meet();
    return;
  }

  if (!(temperature > 0.f) || top_k == 1 || top_p <= 0.f || top == INFINITY) {  // the first of the largest
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

  // exp((z - top) / temperature) in units of 2^-bits.  (Rounded step by step, so that every place of the code finds the same weight.)
  const double per_step = 1.4426950408889634074 * kTable / fmax(static_cast<double>(temperature), 1e-30);
  const float per_power = static_cast<float>(per_step / kTable);
  auto weight_of = [&](float z) -> uint64_t {
    // (no branch: several of them are computed side by side)
    const bool some = (z - top) * per_power > -50.f;
    constexpr double kRound = 6755399441055744.;  // 1.5 * 2^52: what is added to it is rounded to a whole number
    const double y = __dmul_rn(static_cast<double>(z) - static_cast<double>(top), per_step);
    const double t = __dadd_rn(y, kRound);
    const int steps = __double2loint(t);
    const double f = __dsub_rn(y, __dsub_rn(t, kRound));  // up to 1/2
    // 2^(f / kTable) = sum of (f ln 2 / kTable)^i / i!
    constexpr double c1 = 0.69314718055994531 / kTable, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    const double w = __dmul_rn(powers[steps & (kTable - 1)], fma(fma(fma(c3, f, c2), f, c1), f, 1.));
    static_assert(kTable == 1 << 10, "steps of a power");
    const double scaled = __hiloint2double(__double2hiint(w) + (((steps >> 10) + args.bits) << 20), __double2loint(w));
    const double whole = __dadd_rn(scaled, 4503599627370496.);  // + 2^52
    const uint32_t high = some ? static_cast<uint32_t>(__double2hiint(whole)) & 0xFFFFFu : 0, low_part = some ? static_cast<uint32_t>(__double2loint(whole)) : 0;
    return static_cast<uint64_t>(high) << 32 | low_part;
  };
  const uint64_t least = min_p > 0.f ? static_cast<uint64_t>(ceil(fmin(static_cast<double>(min_p), 1.) * static_cast<double>(1ull << args.bits))) : 0;
  // The tokens ahead of which less than p of `share` lies: weights that those ahead of the last one do not reach.
  auto reach_of = [&](uint64_t share) {
    const double to = ceil(static_cast<double>(top_p) * static_cast<double>(share));
    return to <= 1. ? 1 : to >= static_cast<double>(share) ? share : static_cast<uint64_t>(to);
  };
  // What u falls on: the sum that the drawn token is the first to exceed.
  auto target_of = [&](uint64_t whole) {
    const double at = floor(u * static_cast<double>(whole));
    return at >= static_cast<double>(whole) ? whole - 1 : min(static_cast<uint64_t>(at), whole - 1);
  };
  auto sum_of_all = [&](uint64_t v) {
    uint64_t total;
    scan(v, red64, total);
    __syncthreads();
    return total;
  };

  uint64_t from = 0;  // the last place that is kept
  const bool by_count = top_k > 0 && top_k < s.vocab, by_weight = top_p < 1.f;
  if (by_count || by_weight) {
    const float range = fminf(40.f * temperature, top - low);
    const float per_bin = range > 0.f ? fminf(kBins / range, 1e30f) : 0.f;
    // (rounded by what is added to it, which takes no turn of the slow pipe for conversions)
    auto bin_of = [&](float z) { return static_cast<int>(__float_as_uint(fminf((top - z) * per_bin, kBins - 1.f) + 12582912.f) & (2 * kBins - 1)); };
    auto enter = [&](int bin, uint64_t w) {
      const uint32_t w_low = static_cast<uint32_t>(w);
      uint32_t w_high = static_cast<uint32_t>(w >> 32);
      w_high += atomicAdd(&bins.low[bin], w_low) + w_low < w_low;  // and what is carried
      if (w_high) atomicAdd(&bins.high[bin], w_high);
    };
    // Adds to the list the tokens for which `inside` holds.
    auto list_tokens = [&](int use, auto inside) {
#pragma unroll 2
      for (int at = 4 * tid; at < n; at += 4 * kThreads) {
        float z[4];
        fetch(at, z);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (inside(z[k], v0 + at + k)) {
            const uint32_t i = atomicAdd(&listed[use], 1u);
            if (i < kFew) lists[use][i] = place_of(z[k], v0 + at + k);
          }
      }
    };
    // The last and the first of them in the order, for too many of them to be listed.
    auto find_ends = [&](int use, auto inside) {
      uint64_t last = ~0ull, first = 0;
      for (int at = 4 * tid; at < n; at += 4 * kThreads) {
        float z[4];
        fetch(at, z);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (inside(z[k], v0 + at + k)) {
            last = min(last, place_of(z[k], v0 + at + k));
            first = max(first, place_of(z[k], v0 + at + k));
          }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        last = min(last, __shfl_xor_sync(0xFFFFFFFFu, last, d));
        first = max(first, __shfl_xor_sync(0xFFFFFFFFu, first, d));
      }
      if (lane == 0 && first) {
        atomicMin(reinterpret_cast<unsigned long long*>(&ends[use][0]), last);
        atomicMax(reinterpret_cast<unsigned long long*>(&ends[use][1]), first);
      }
    };

    // The lists of all CTAs as one, with weights; their number, or more than kFew.
    auto merge_lists = [&](int use) {
      uint32_t many[kMostCtas];
      words_of_all(&listed[use], many);
      uint32_t ahead = 0;
#pragma unroll
      for (int r = 0; r < kMostCtas; ++r) {
        if (tid >= ahead && tid - ahead < min(many[r], kFew) && tid < kFew) {
          const uint64_t place = ctas == 1 ? lists[use][tid] : load_cluster_u64(there(&lists[use][tid - ahead], r));
          merged[tid] = make_ulonglong2(place, weight_of(logit_of(place)));
        }
        ahead += many[r];
      }
      __syncthreads();
      return ahead;
    };

    // The place of the token that is the count_to-th or, if that is 0, with which the weights of places >= from reach weight_to.
    auto select = [&](int use, uint32_t count_to, uint64_t weight_to, uint64_t weight, uint64_t weight_before, uint32_t count, uint32_t count_before) -> uint64_t {
      uint64_t last = 0, first = ~0ull, shift = 0;
      bool places = false;  // whether the bins are intervals of places
      // every turn leaves a 1024th of the places, of which there are less than 2^62
      for (int turn = 0; turn < 8; ++turn) {
        const bool here = count_to ? count_before < count_to && count_before + count >= count_to : weight_before < weight_to && weight_before + weight >= weight_to;
        if (here) found = {tid, count, count_before, weight_before};
        __syncthreads();
        const Found f = found;
        // a bin's tokens: what is rounded to its number
        auto in_bin = [&](float z, int token) { return bin_of(z) == f.bin && z > -INFINITY && (from == 0 || place_of(z, token) >= from); };
        if (!places) {
          list_tokens(use, in_bin);
        } else {
          first -= static_cast<uint64_t>(f.bin) << shift;
          const uint64_t width = (1ull << shift) - 1;
          last = first - last < width ? last : first - width;
          if (tid == 0) listed[use] = 0;
          meet();
          list_tokens(use, [&](float z, int token) {
            const uint64_t place = place_of(z, token);
            return z > -INFINITY && place >= last && place <= first;
          });
        }
        meet();
        const uint32_t many = merge_lists(use);
        if (many <= kFew) {
          if (tid < many) {
            const uint64_t mine = merged[tid].x, own = merged[tid].y;
            uint64_t sum = f.weight_before;
            uint32_t rank = f.count_before;
#pragma unroll 4
            for (uint32_t i = 0; i < many; ++i) {
              const ulonglong2 other = merged[i];
              rank += other.x > mine;
              sum += other.x > mine ? other.y : 0;
            }
            if (count_to ? rank + 1 == count_to : sum < weight_to && sum + own >= weight_to) cut = mine;
          }
          __syncthreads();
          const uint64_t place = cut;
          __syncthreads();
          return place;
        }
        // too many: a histogram of their places alone
        if (!places) {
          find_ends(use, in_bin);
          meet();
          for (int r = 0; r < ctas; ++r) {
            last = r ? min(last, load_cluster_u64(there(&ends[use][0], r))) : load_cluster_u64(there(&ends[use][0], 0));
            first = r ? max(first, load_cluster_u64(there(&ends[use][1], r))) : load_cluster_u64(there(&ends[use][1], 0));
          }
          places = true;
        }
        shift = 64 - __clzll(static_cast<long long>(first - last));
        shift = shift > 10 ? shift - 10 : 0;
        static_assert(kBins == 1 << 10, "bins of places");
        clear_bins();
        __syncthreads();
#pragma unroll 1
        for (int at = 4 * tid; at < n; at += 4 * kThreads) {
          float z[4];
          fetch(at, z);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t place = place_of(z[k], v0 + at + k);
            if (z[k] > -INFINITY && place >= last && place <= first) {
              const int bin = static_cast<int>((first - place) >> shift);
              if (count_to) atomicAdd(&bins.count[bin], 1u);
              else enter(bin, weight_of(z[k]));
            }
          }
        }
        meet();
        uint32_t counts[kMostCtas], lows[kMostCtas], highs[kMostCtas], all_count;
        uint64_t all_weight;
        words_of_all(&bins.count[tid], counts);
        words_of_all(&bins.low[tid], lows);
        words_of_all(&bins.high[tid], highs);
        count = 0, weight = 0;
        for (int r = 0; r < kMostCtas; ++r) count += counts[r], weight += (static_cast<uint64_t>(highs[r]) << 32) + lows[r];
        count_before = f.count_before + scan(count, red32, all_count);
        weight_before = f.weight_before + scan(weight, red64, all_weight);
        meet();  // nobody clears what another still reads
      }
      return 0;
    };

    if (by_count) {
#pragma unroll 2
      for (int at = 4 * tid; at < n; at += 4 * kThreads) {
        float z[4];
        fetch(at, z);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (z[k] > -INFINITY) atomicAdd(&bins.count[bin_of(z[k])], 1u);
      }
      meet();
      uint32_t counts[kMostCtas], count = 0, all_count;
      words_of_all(&bins.count[tid], counts);
#pragma unroll
      for (int r = 0; r < kMostCtas; ++r) count += counts[r];
      const uint32_t before = scan(count, red32, all_count);
      if (tid == 0) found.bin = -1;
      __syncthreads();
      const bool here = before < top_k && before + count >= top_k;
      if (here) found = {tid, count, before, 0};
      __syncthreads();
      const Found f = found;  // bin -1: there are fewer tokens than that
      const int last_bin = f.bin < 0 ? kBins - 1 : f.bin;
      if ((f.bin < 0 ? all_count : f.count_before + f.tokens) <= kFew) {
        // all that can be drawn fits a list
        list_tokens(0, [&](float z, int) { return z > -INFINITY && bin_of(z) <= last_bin; });
        meet();
        if (blockIdx.z == 0) {
          const uint32_t many = min(merge_lists(0), kFew);
          uint32_t rank = 0;
          uint64_t ahead = 0, own = 0;
          ulonglong2 mine{0, 0};
          if (tid < many) {
            mine = merged[tid];
#pragma unroll 4
            for (uint32_t i = 0; i < many; ++i) {
              const ulonglong2 other = merged[i];
              rank += other.x > mine.x;
              ahead += other.x > mine.x ? other.y : 0;
            }
            if (rank < top_k) own = mine.y;
          }
          if (by_weight) {
            const uint64_t reach = reach_of(sum_of_all(own));
            if (ahead >= reach) own = 0;
          }
          if (own < least) own = 0;
          __syncthreads();
          if (tid < many) merged[tid].y = own;
          const uint64_t target = target_of(sum_of_all(own));
          if (own) {
            uint64_t upto = 0;  // in the order of the vocabulary
#pragma unroll 4
            for (uint32_t i = 0; i < many; ++i) {
              const ulonglong2 other = merged[i];
              upto += static_cast<uint32_t>(other.x) >= static_cast<uint32_t>(mine.x) ? other.y : 0;
            }
            if (upto > target && upto - own <= target) s.out[row] = 0xFFFFFFFFu - static_cast<uint32_t>(mine.x);
          }
        }
        meet();
        return;
      }
      if (f.bin >= 0) from = select(0, top_k, 0, 0, 0, count, before);
      else meet();
      clear_bins();
      __syncthreads();
    }
    if (by_weight) {
#pragma unroll 2
      for (int at = 4 * tid; at < n; at += 4 * kThreads) {
        float z[4];
        uint64_t w[4];
        fetch(at, z);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = weight_of(z[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (w[k] && (from == 0 || place_of(z[k], v0 + at + k) >= from)) enter(bin_of(z[k]), w[k]);
      }
      meet();
      uint32_t lows[kMostCtas], highs[kMostCtas];
      words_of_all(&bins.low[tid], lows);
      words_of_all(&bins.high[tid], highs);
      uint64_t weight = 0, share;
#pragma unroll
      for (int r = 0; r < kMostCtas; ++r) weight += (static_cast<uint64_t>(highs[r]) << 32) + lows[r];
      const uint64_t before = scan(weight, red64, share);
      from = max(from, select(1, 0, reach_of(share), weight, before, 0, 0));
    }
  }

  // Sums of what is kept, chunk by chunk; a warp has a chunk.  Its kept tokens move together, so that few of them take few turns.
  const float last_logit = from ? logit_of(from) : -INFINITY;
  const int last_token = from ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(from)) : -1;
  auto is_kept = [&](float z, int token) { return z > last_logit || (z == last_logit && token <= last_token); };
  auto kept_weight = [&](float z) -> uint64_t {
    const uint64_t w = weight_of(z);
    return w >= least ? w : 0;
  };
  __syncthreads();
  sums[tid] = 0;
  __syncthreads();
  // A warp's pieces of 128 tokens, chunk after chunk; the next one's logits are on their way.
  auto next_piece = [&](int& c, int& at) {
    at += 128;
    if (at >= (c + 1) * args.chunk || at >= n) {
      c += kThreads / 32;
      at = c * args.chunk;
    }
  };
  int chunk = warp, piece = warp * args.chunk;
  float next[4];
  if (piece < n) fetch(piece + 4 * lane, next);
  uint64_t sum = 0;
#pragma unroll 1
  while (piece < n) {
    const float z[4] = {next[0], next[1], next[2], next[3]};
    const int at = piece + 4 * lane, now = chunk;
    next_piece(chunk, piece);
    if (piece < n) fetch(piece + 4 * lane, next);
    int many = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool kept = is_kept(z[k], v0 + at + k);
      const uint32_t all = __ballot_sync(0xFFFFFFFFu, kept);
      if (kept) buffer.kept[warp][many + __popc(all & ((1u << lane) - 1))] = z[k];
      many += __popc(all);
    }
    __syncwarp();
    for (int i = lane; i < many; i += 32) sum += kept_weight(buffer.kept[warp][i]);
    __syncwarp();
    if (chunk != now) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
      if (lane == 0) sums[now] = sum;
      sum = 0;
    }
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
  const uint64_t target = target_of(whole);
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
        w[k] = is_kept(z[k], v0 + at + k) ? kept_weight(z[k]) : 0;
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
  // few rows: a cluster for each, as large as all of them run at one time (one row of 50304 by 8, 4, 2 and 1 CTAs: 13.0, 14.1, 15.5 and 16.2 us)
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
