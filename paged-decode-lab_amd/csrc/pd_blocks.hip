// Attention of one token a sequence over the blocks of a paged cache, and the
// choice of the blocks, for MI355X (gfx950).
//
//   pd_select_blocks   score(j) = max over the heads h of a kv head's group of
//                      sum_d max(q_hd, 0) hi_jd + min(q_hd, 0) lo_jd, the
//                      largest q . k that keys within the block's bounds allow;
//                      the kept blocks of the highest scores
//   pd_block_decode    out = softmax(scale k_scale q K^T) V v_scale over the
//                      listed blocks, or over all of them
//
// A block is 64 tokens, a quarter of a page.
//
// Attention: bound by the bytes of K and V.  Wavefronts walk the tiles of a
// sequence (or list) with private softmax states, K and V in registers from
// their loads to the matrix instructions, and are joined in LDS at the end of a
// workgroup; the splits of a sequence by a second launch.  Vector instructions
// take a third of the time that the bytes do (counters: 64 sequences of up to
// 32768 e4m3 tokens, Hq 32 / Hkv 8 / D 128, 35% of the SIMDs' clocks), which is
// what the products in three bf16 terms of the probabilities and the e4m3
// conversions are paid from.  Measured on MI355X, both launches:
//   64 sequences of 1 to 32768 e4m3 tokens, Hq 32 / Hkv 8 / D 128   391 us  5.5 TB/s
//   128 of 1 to 4096, Hq = Hkv = 16, D 64                           124 us  4.5 TB/s
//   64 sequences, 64 listed bf16 blocks, Hq 32 / Hkv 8 / D 128      176 us  5.6 TB/s
//   17 sequences, 37 listed e4m3 blocks, Hq 32 / Hkv 4 / D 256     23.1 us  3.4 TB/s
//   one, 64 listed bf16 blocks, Hq 16 / Hkv 4 / D 256              10.0 us, launches and
//   one of 2064 e4m3 tokens, the same heads                         8.6 us  latencies
// (a copy of 2 GiB reads and writes 4.85 TB/s; reads alone reach 6.3).  Of the
// last two 6 to 7 us are the attention's chain: length, table, K, softmax, join,
// write.  The bf16 decode's partition does its own chain in 4.3 us for the same
// heads and 2064 tokens, so that one is no bound of the hardware.
//
// Selection, by the method of ranking blocks of keys by the extremes of their
// channels: the scores are bound by their vector instructions (57% of the SIMDs'
// clocks where the bounds' bytes would take 14 us: 64 sequences of up to 32768
// tokens, 22 us), the choice by its barriers (4 to 6 us).  Groups of more than
// four heads take the query again for every run of blocks, four heads at a time:
// 32 sequences of up to 16384 tokens, Hq 32 / Hkv 4 / D 256, 22 us where the bytes
// take 4.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "pd_blocks.h"
#include "pd_device.h"
#include "pd_internal.h"
#include "pd_launch.h"

namespace {

using namespace pdk;
using pd::all_aligned16;
using pd::as_stream;
using pd::launch_status;
using pd::u16;

constexpr int kBlock = pd::kBlock, kPerPage = pd::kPageSize / pd::kBlock;

__device__ __forceinline__ int block_count(const int32_t* lengths, int b, int width) {
  const int64_t most = int64_t(width) * pd::kPageSize;
  const int64_t len = min(int64_t(max(lengths[b], 0)), most);
  return int((len + kBlock - 1) / kBlock);
}

// ------------------------------------------------------------------ selection

// A score takes of each channel the corner that the query's sign asks for and
// never the other, however large that is.  The products are exact in 64 bits, the
// sums off by 2^-53 of the taken products' sizes: two implementations pick the
// same blocks unless scores agree to some 15 digits of their terms without being
// equal.
//
// Two launches: one workgroup for a (sequence, kv head), with its keys in LDS, is
// 7.7 instead of 10.3 us for 16 sequences of up to 16384 tokens of 16 kv heads,
// and 31 instead of 8 for one sequence of 32768 of 4.
struct SelectArgs {
  const int32_t *lengths, *table;
  const uint16_t *q, *bounds;
  uint64_t* keys;  // [batch][hkv][width * 4]
  int64_t qsb, qsh, tsb;
  int width, hkv, num_pages, group, kept, first, last;
};

// Larger for a larger score; a NaN counts as +infinity, -0 as +0.
__device__ __forceinline__ uint64_t score_key(double s) {
  s = s != s ? __builtin_inf() : s + 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | (uint64_t(1) << 63);
}

template <int M>
__device__ __forceinline__ double xor_lanes64(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __float_as_uint(xor_lanes<M>(__uint_as_float(uint32_t(u)), lane));
  const uint32_t hi = __float_as_uint(xor_lanes<M>(__uint_as_float(uint32_t(u >> 32)), lane));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// A block's bounds are kLanes lanes of eight channels; a run is the 64 / kLanes
// blocks of a wavefront.  kHeads query heads at a time are held as doubles.
template <int D>
struct Scores {
  static constexpr int kLanes = D / 8, kPer = 64 / kLanes;
};

template <int D, int kHeads>
struct Query {
  double x[kHeads][8];
  // Heads head0.. of the group; past its end the last one again, which moves no maximum.
  __device__ __forceinline__ void load(const SelectArgs& p, int b, int g, int head0, int part) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int64_t head = int64_t(g) * p.group + min(head0 + h, p.group - 1);
      float f[8];
      unpack8(load16(p.q + b * p.qsb + head * p.qsh + 8 * part), f);
      // f - f: an infinity becomes a NaN, with which every score is one.
#pragma unroll
      for (int i = 0; i < 8; ++i) x[h][i] = f[i] + (f[i] - f[i]);
    }
  }
};

// Bounds of block j of sequence b, this lane's channels; a page outside the pool: known false.
template <int D>
struct Bounds {
  u32x4_t lo, hi;
  bool known;
  __device__ __forceinline__ void load(const SelectArgs& p, int b, int g, int j, int part) {
    j = min(j, p.width * kPerPage - 1);  // past the last candidate: any entry, not used
    const int64_t page = p.table[b * p.tsb + j / kPerPage];
    known = page >= 0 && page < p.num_pages;
    const uint16_t* at =
        p.bounds + (((known ? page : 0) * kPerPage + j % kPerPage) * p.hkv + g) * 2 * D + 8 * part;
    lo = load16(at);
    hi = load16(at + D);
  }
};

// A bf16 as a double is the upper word of it, above a word of zeros.
__device__ __forceinline__ uint32_t upper(float x) {
  return uint32_t(__builtin_bit_cast(uint64_t, double(x)) >> 32);
}
__device__ __forceinline__ double of_upper(uint32_t w) {
  return __builtin_bit_cast(double, uint64_t(w) << 32);
}

// The corners of one block, this lane's channels.
struct Corners {
  uint32_t lo[8], hi[8];
  bool finite;
  __device__ __forceinline__ Corners(u32x4_t raw_lo, u32x4_t raw_hi) {
    float l[8], h[8];
    unpack8(raw_lo, l);
    unpack8(raw_hi, h);
    float most = 0.f;  // NaN where one is
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = upper(l[i]), hi[i] = upper(h[i]);
      most = __builtin_elementwise_maximum(
          __builtin_elementwise_maximum(most, __builtin_fabsf(l[i])), __builtin_fabsf(h[i]));
    }
    finite = most < INFINITY;
  }
};

// sum_d max(q, 0) hi + min(q, 0) lo: q times the corner of its sign, and zero times the other
// one, which only moves a sum where bounds are not finite (kFinite false).  The largest of
// kHeads heads' sums, in every lane of the block: a lane pair splits the heads between them at
// each of the first steps, so that a step moves half of the sums of the one before.
template <int D, int kHeads, bool kFinite>
__device__ __forceinline__ double best_of(const Query<D, kHeads>& q, const Corners& c, int lane) {
  double s[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    s[h] = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double x = q.x[h][i];
      s[h] = __builtin_fma(x, of_upper(x < 0.0 ? c.lo[i] : c.hi[i]), s[h]);
      if constexpr (!kFinite)
        s[h] = __builtin_fma(0.0, of_upper(x < 0.0 ? c.hi[i] : c.lo[i]), s[h]);
    }
  }
  double x;
  if constexpr (kHeads == 4) {
    const bool odd = lane & 1, second = lane & 2;
    const double a0 = (odd ? s[2] : s[0]) + xor_lanes64<1>(odd ? s[0] : s[2], lane);
    const double a1 = (odd ? s[3] : s[1]) + xor_lanes64<1>(odd ? s[1] : s[3], lane);
    x = (second ? a1 : a0) + xor_lanes64<2>(second ? a0 : a1, lane);
  } else if constexpr (kHeads == 2) {
    const bool odd = lane & 1;
    x = (odd ? s[1] : s[0]) + xor_lanes64<1>(odd ? s[0] : s[1], lane);
    x += xor_lanes64<2>(x, lane);
  } else {
    x = s[0] + xor_lanes64<1>(s[0], lane);
    x += xor_lanes64<2>(x, lane);
  }
  x += xor_lanes64<4>(x, lane);
  if constexpr (Scores<D>::kLanes > 8) x += xor_lanes64<8>(x, lane);
  if constexpr (Scores<D>::kLanes > 16) x += xor_lanes64<16>(x, lane);
  if (x != x) x = __builtin_inf();
  if constexpr (kHeads > 1) x = fmax(x, xor_lanes64<1>(x, lane));
  if constexpr (kHeads > 2) x = fmax(x, xor_lanes64<2>(x, lane));
  return x;
}

// Scores of blocks j0 + lane / kLanes, every `step` blocks, below end_of(), which waits for the
// length, to store(j, key).  kWhole (kHeads >= group): the query stays in registers; else it
// is taken again for every run, kHeads heads at a time.
template <int D, int kHeads, bool kWhole, typename End, typename Store>
__device__ __forceinline__ void score_blocks(const SelectArgs& p, int b, int g, int j0, int step,
                                             int lane, End end_of, Store store) {
  using S = Scores<D>;
  const int part = lane % S::kLanes, mine = lane / S::kLanes;
  Bounds<D> next;
  next.load(p, b, g, j0 + mine, part);
  Query<D, kHeads> q;
  if constexpr (kWhole) q.load(p, b, g, 0, part);
  const int end = end_of();
  for (int j = j0; j < end; j += step) {
    const Bounds<D> here = next;
    if (j + step < end) next.load(p, b, g, j + step + mine, part);
    Corners corners(here.lo, here.hi);
    const auto best_by = [&](auto finite) {
      if constexpr (kWhole) return best_of<D, kHeads, finite.value>(q, corners, lane);
      double best = -__builtin_inf();
      for (int head = 0; head < p.group; head += kHeads) {
        q.load(p, b, g, head, part);
        best = fmax(best, best_of<D, kHeads, finite.value>(q, corners, lane));
      }
      return best;
    };
    double best;
    if (__all(corners.finite)) {
      best = best_by(std::true_type{});
    } else {
      // The rare path's own copies: corners picked for both paths ahead of the branch would be
      // moved once more each (64 sequences of up to 32768 tokens, both launches: 34.2 us, 28.0
      // so).
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(corners.lo[i]), "+v"(corners.hi[i]));
      best = best_by(std::false_type{});
    }
    if (part == 0 && j + mine < end) store(j + mine, here.known ? score_key(best) : 0);
  }
}

// The scores of one (sequence, kv head), cut over the workgroups of grid.x.
template <int D, int kHeads, bool kWhole>
__global__ void __launch_bounds__(256)
score_kernel(const int32_t* lengths, const int32_t* table, const uint16_t* q,
             const uint16_t* bounds, uint64_t* keys_of, int64_t tsb, int width, int hkv,
             int num_pages, int kept, int first, int last, int group, int64_t qsb, int64_t qsh) {
  const SelectArgs p{lengths, table, q,     bounds, keys_of, qsb,   qsh, tsb,
                     width,   hkv,   num_pages, group, kept,    first, last};
  constexpr int kPer = Scores<D>::kPer;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int g = blockIdx.y, b = blockIdx.z;
  uint64_t* keys = p.keys + (int64_t(b) * p.hkv + g) * p.width * kPerPage;
  score_blocks<D, kHeads, kWhole>(
      p, b, g, p.first + (blockIdx.x * 4 + w) * kPer, gridDim.x * 4 * kPer, lane,
      [&] {
        const int n = block_count(p.lengths, b, p.width);
        return n > p.kept ? n - p.last : 0;
      },
      [&](int j, uint64_t key) { keys[j] = key; });
}

template <int M>
__device__ __forceinline__ uint64_t xor_lanes_u64(uint64_t x, int lane) {
  return __builtin_bit_cast(uint64_t, xor_lanes64<M>(__builtin_bit_cast(double, x), lane));
}

// The blocks of one (sequence, kv head) by its candidates' keys, begin <= j < end: the
// threshold is found digit by digit from the highest bit in which the keys differ, then one
// ordered pass writes the forced blocks, those above the threshold and the first at it.
constexpr int kDigit = 11, kBins = 1 << kDigit;

constexpr int kCached = 8;  // keys that a thread holds in its registers

template <int kWaves>
struct Picker {
  uint32_t bins[kBins];
  uint64_t wave_keys[2][kWaves];
  uint64_t close_keys[64];  // the keys of the threshold's bin, where they are few
  int32_t close_blocks[64];
  uint32_t wave_counts[kCached][kWaves], found[2], close;
  uint64_t edge;
};

// kAll: `cached` holds all of the thread's keys, begin + its number + i threads of them.
template <int kWaves, bool kAll>
__device__ __forceinline__ void pick_blocks(Picker<kWaves>& t, const uint64_t* __restrict__ keys,
                                            const uint64_t (&cached)[kCached], int n, int begin,
                                            int end, uint32_t need, int32_t* out) {
  constexpr int kCache = kAll ? kCached : 0;
  constexpr int kThreads = 64 * kWaves;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const auto each = [&](auto use) {  // use(j, key) of the thread's candidates
    if constexpr (kCache > 0) {
#pragma unroll
      for (int i = 0; i < kCache; ++i)
        if (begin + i * kThreads < end) {
          const int j = begin + tid + i * kThreads;
          if (j < end) use(j, cached[i]);
        }
    } else {
      for (int j = begin + tid; j < end; j += kThreads) use(j, keys[j]);
    }
  };
  for (int i = tid; i < kBins; i += kThreads) t.bins[i] = 0;
  if (tid == 0) t.close = 0;
  uint64_t every = ~uint64_t(0), some = 0;
  each([&](int, uint64_t key) { every &= key, some |= key; });
  every &= xor_lanes_u64<1>(every, lane), some |= xor_lanes_u64<1>(some, lane);
  every &= xor_lanes_u64<2>(every, lane), some |= xor_lanes_u64<2>(some, lane);
  every &= xor_lanes_u64<4>(every, lane), some |= xor_lanes_u64<4>(some, lane);
  every &= xor_lanes_u64<8>(every, lane), some |= xor_lanes_u64<8>(some, lane);
  every &= xor_lanes_u64<16>(every, lane), some |= xor_lanes_u64<16>(some, lane);
  every &= xor_lanes_u64<32>(every, lane), some |= xor_lanes_u64<32>(some, lane);
  if (lane == 0) t.wave_keys[0][w] = every, t.wave_keys[1][w] = some;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) every &= t.wave_keys[0][i], some |= t.wave_keys[1][i];

  // Keys whose bits from `shift` (below 64) up are above `edge` are in, and `need` of those
  // at it.
  const uint64_t differ = every ^ some;
  int shift = differ ? 64 - __builtin_clzll(differ) : 0;
  uint64_t edge = shift < 64 ? some >> shift : 0;
  uint32_t at_edge = end - begin;
  const uint32_t taken = need;
  if (need == 0) edge = ~uint64_t(0), shift = 0;
  bool clear = true;  // bins
  while (need && shift > 0 && at_edge != need) {
    if (!clear && at_edge <= 64) {
      // Few keys share the edge: the need-th of them by their ranks.
      each([&](int j, uint64_t key) {
        if (key >> shift == edge) {
          const uint32_t at = atomicAdd(&t.close, 1u);
          if (at < 64) t.close_keys[at] = key, t.close_blocks[at] = j;
        }
      });
      __syncthreads();
      if (w == 0) {
        const uint64_t key = t.close_keys[lane];
        const int j = t.close_blocks[lane];
        uint32_t above = 0, same = 0;
        for (uint32_t i = 0; i < at_edge; ++i) {
          above += t.close_keys[i] > key;
          same += t.close_keys[i] == key && t.close_blocks[i] < j;
        }
        if (lane < int(at_edge) && above + same == need - 1) t.edge = key, t.found[0] = same + 1;
      }
      __syncthreads();
      edge = t.edge, need = t.found[0], shift = 0;
      break;
    }
    const int next = max(shift - kDigit, 0);
    if (!clear) {
      for (int i = tid; i < kBins; i += kThreads) t.bins[i] = 0;
      __syncthreads();
    }
    clear = false;
    each([&](int, uint64_t key) {
      if ((shift < 64 ? key >> shift : 0) == edge)
        atomicAdd(&t.bins[(key >> next) & ((1u << (shift - next)) - 1)], 1u);
    });
    __syncthreads();
    // From the highest bin down: the one in which the count reaches `need`.
    constexpr int kOwn = kBins / kThreads;
    const int top = kBins - 1 - tid * kOwn;
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += t.bins[top - i];
    uint32_t before = sum;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const uint32_t x = __shfl_up(before, m);
      if (lane >= m) before += x;
    }
    if (lane == 63) t.wave_counts[0][w] = before;
    __syncthreads();
    for (int i = 0; i < w; ++i) before += t.wave_counts[0][i];
    before -= sum;
    if (before < need && before + sum >= need) {
      uint32_t above = before;
      int bin = top;
      while (above + t.bins[bin] < need) above += t.bins[bin--];
      t.found[0] = bin, t.found[1] = above;
    }
    __syncthreads();
    const uint32_t bin = t.found[0];
    need -= t.found[1];
    at_edge = t.bins[bin];
    edge = (shift < 64 ? edge << (shift - next) : 0) | bin;
    shift = next;
    __syncthreads();
  }

  for (int j = tid; j < begin; j += kThreads) out[j] = j;
  for (int i = tid; i < n - end; i += kThreads) out[begin + taken + i] = end + i;
  // In order: a block a thread at a time, a thread's place by the counts ahead of it.
  const uint64_t below = (uint64_t(1) << lane) - 1;
  uint32_t written = begin, ties = 0;
  const auto marks = [&](int j, uint64_t key, bool& in, bool& tie) {
    if (shift < 64) key >>= shift;
    in = j < end && shift < 64 && key > edge;
    tie = j < end && (shift == 64 || key == edge);
  };
  const auto place = [&](int j, bool in, bool tie, const uint32_t (&counts)[kWaves]) {
    uint32_t ahead = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < w) ahead += counts[i];
      all += counts[i];
    }
    // Ties ahead of this block that are in: the first `need` of them.
    const uint32_t tied = ties + (ahead >> 16) + __popcll(__ballot(tie) & below);
    const uint32_t at = written + (ahead & 0xffff) + __popcll(__ballot(in) & below) + min(tied, need);
    if ((in || (tie && tied < need)) && at < begin + taken) out[at] = j;
    written += all & 0xffff;
    ties += all >> 16;
  };
  const auto count = [&](bool in, bool tie, uint32_t& cell) {
    const uint32_t both = uint32_t(__popcll(__ballot(in))) | uint32_t(__popcll(__ballot(tie))) << 16;
    if (lane == 0) cell = both;
  };
  bool in, tie;
  if constexpr (kCache > 0) {
#pragma unroll
    for (int i = 0; i < kCache; ++i)
      if (begin + i * kThreads < end) {
        marks(begin + tid + i * kThreads, cached[i], in, tie);
        count(in, tie, t.wave_counts[i][w]);
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCache; ++i)
      if (begin + i * kThreads < end) {
        marks(begin + tid + i * kThreads, cached[i], in, tie);
        place(begin + tid + i * kThreads, in, tie, t.wave_counts[i]);
      }
  } else {
    for (int base = begin; base < end; base += kThreads) {
      marks(base + tid, keys[min(base + tid, end - 1)], in, tie);
      count(in, tie, t.wave_counts[0][w]);
      __syncthreads();
      place(base + tid, in, tie, t.wave_counts[0]);
      __syncthreads();
    }
  }
}

__device__ __forceinline__ void list_all(int32_t* out, int kept, int n) {
  for (int i = threadIdx.x; i < kept; i += blockDim.x) out[i] = i < n ? i : -1;
}

// One sequence of 512 blocks: 7.7 us for both launches with 4 wavefronts, 8.0 with 8, 9.4 with
// 16, whose barriers cost more than their keys.
constexpr int kPickWaves = 4;

__global__ void __launch_bounds__(64 * kPickWaves)
pick_kernel(const int32_t* __restrict__ lengths, const uint64_t* __restrict__ all_keys,
            int32_t* __restrict__ blocks, int width, int hkv, int kept, int first, int last) {
  __shared__ Picker<kPickWaves> picker;
  const int g = blockIdx.x, b = blockIdx.y;
  const uint64_t* keys = all_keys + (int64_t(b) * hkv + g) * width * kPerPage;
  // A thread's first keys are on their way while the length is.
  uint64_t cached[kCached];
#pragma unroll
  for (int i = 0; i < kCached; ++i)
    cached[i] = keys[min(int64_t(first) + int(threadIdx.x) + i * 64 * kPickWaves,
                         int64_t(width) * kPerPage - 1)];
  const int n = block_count(lengths, b, width);
  int32_t* out = blocks + (int64_t(b) * hkv + g) * kept;
  if (n <= kept) return list_all(out, kept, n);
  const int end = n - last;
  const uint32_t need = uint32_t(kept - first - last);
  if (end - first <= kCached * 64 * kPickWaves)
    pick_blocks<kPickWaves, true>(picker, keys, cached, n, first, end, need, out);
  else
    pick_blocks<kPickWaves, false>(picker, keys, cached, n, first, end, need, out);
}

// ------------------------------------------------------------------ attention

// Splits that a sequence of `len` tokens uses: as many as leave every wavefront a tile of it
// (of the list, where that has fewer), or two.  The others end at once.  A table's width is a
// capacity: 64 sequences of 500 to 1500 tokens with room for 131072 take 45 us, 35 with room
// for 1500, and 81 in as many splits as there are.
struct SplitRule {
  int width, listed, tile, two, splits;  // listed: tiles of a list, 0: every block
  __device__ __forceinline__ int length(const int32_t* lengths, int b) const {
    return min(max(lengths[b], 0), width * pd::kPageSize);  // width below 2^22
  }
  __device__ __forceinline__ int used(int len) const {
    const int filled = (len + tile - 1) >> __builtin_ctz(tile);
    const int count = listed ? min(listed, filled) : filled;
    return max(1, min(splits, (count + (4 << two) - 1) >> (2 + two)));
  }
};

struct DecodeArgs {
  const float *k_scale, *v_scale;
  float *part_o, *part_ml;  // [batch][heads][splits][D], [batch][heads][splits][2]
  uint16_t* out;
  int64_t qsb, qsh;
  int group, tiles;  // tiles: of 16 query heads a kv head
  int two;           // SplitRule's
  float scale2;      // scale log2 e
};

// A wavefront's tile: kTile tokens, 8 KB of a bf16 K and V.  S^T = K Q^T and
// O^T = V^T P^T with 16 x 16 x 32 MFMAs.  In both results a lane's column is query head
// lane % 16, so the softmax state is one scalar a lane, and the layout of the scores (tokens
// 16 u + 4 (lane / 16) + r in element r of result u) is the operand layout of P^T with its
// tokens in that order, which V's rows are loaded in too.  V^T's operand wants eight tokens
// of a channel in a lane: a lane loads kRun channels of eight tokens and turns the 8 x kRun
// square with byte permutes; row m of the MFMA of channel j is channel kRun m + j.  No value
// crosses a lane or the LDS before the end.  A bf16 tile at head_dim 256 is 16 tokens, its
// P V MFMAs 16 x 16 x 16: 32 tokens did not fit two wavefronts a SIMD without spills (32
// sequences of 64 blocks, Hq 16 / Hkv 4: 110 us, 94 with 16).
//
// Tiles of 64 e4m3 tokens: 26.7 instead of 23.5 us for 8 sequences of 1000 to 9000 (Hkv 8, D
// 128), 38.5 and 35 for 16 (Hkv 16, D 64), 408 and 415 for 64 of up to 32768; of 32 bf16
// tokens at D 64: 107 instead of 93 for 64 sequences of 32 blocks.  A second tile on its way
// is no faster at D 64 and slower at D 128 (455 instead of 388), where it costs a wavefront.
template <int D, bool kE4m3>
struct Decode {
  static constexpr int kBytes = kE4m3 ? 1 : 2;
  static constexpr int kTile = kE4m3 ? 32 : 4096 / D;
  static constexpr int kSums = kTile / 16;               // results of S^T
  static constexpr int kGroups = kTile < 32 ? 1 : kTile / 32;
  static constexpr int kPer = kTile < 32 ? 4 : 8;        // tokens of a lane's P V operand
  static constexpr int kStepsQ = D / 32;
  static constexpr int kKLoads = D * kBytes / 64;        // 16-byte loads a lane and 16 tokens
  static constexpr int kRun = D / 16 < 16 / kBytes ? D / 16 : 16 / kBytes;  // channels a load
  static constexpr int kChunks = D / 16 / kRun;
  static constexpr int kWords = kRun * kBytes / 4;       // dwords a load
  static constexpr int kOut = D / 16;                    // MFMAs of O^T

  // Channel of element i of a lane's operand of step s (row = lane / 16).
  static __device__ __forceinline__ int channel(int s, int row) {
    return kE4m3 ? (s / 2) * 64 + row * 16 + (s % 2) * 8 : s * 32 + row * 8;
  }
  // Token of element i of group a's operand.
  static __device__ __forceinline__ int token(int a, int i, int row) {
    return 32 * a + 16 * (i >> 2) + 4 * row + (i & 3);
  }
};

template <int N>
struct Words {
  uint32_t w[N];
};

// Rows of 512 bytes pass the caches by (32 sequences of 64 blocks: 94 -> 87 us); the lines of
// shorter ones are still to be read by another load (64 e4m3 sequences of 128-byte rows: 394
// -> 511).
template <typename V, int kRowBytes>
__device__ __forceinline__ V load_row(const char* p) {
  if constexpr (kRowBytes >= 512)
    return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else
    return *reinterpret_cast<const V*>(p);
}

template <int N, int kRowBytes>
__device__ __forceinline__ Words<N> load_words(const char* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const u32x4_t x = load_row<u32x4_t, kRowBytes>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else if constexpr (N == 2) {
    const u32x2_t x = load_row<u32x2_t, kRowBytes>(p);
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
    r.w[0] = load_row<uint32_t, kRowBytes>(p);
  }
  return r;
}

// Two e4m3 bytes of x (the lower or the upper ones) as bf16, exactly.
template <bool kUpper>
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, kUpper));
}

typedef short short4v_t __attribute__((ext_vector_type(4)));

// D += A B over kPer tokens a lane.
template <int kPer>
__device__ __forceinline__ floatx4_t mfma_pv(const Words<kPer / 2>& a, const Words<kPer / 2>& b,
                                             floatx4_t c) {
  if constexpr (kPer == 8)
    return mfma16(__builtin_bit_cast(u32x4_t, a), __builtin_bit_cast(u32x4_t, b), c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v_t, a),
                                                     __builtin_bit_cast(short4v_t, b), c, 0, 0, 0);
}

// A probability as three bf16, in the upper halves of the words: 8 bits each of its 24, by
// cutting.  One term's error would be as large as the output's own rounding; two (16 bits) move
// some outputs to the other side of theirs (64 sequences of up to 32768 e4m3 tokens: 1.3e-4
// from the float32 form, relative, 2.2e-5 with three) and are hardly cheaper (398 us both; 16
// of up to 8192, Hkv 16, D 64: 34.3 and 35.5).  Where p is not zero, neither is any of them
// (2^-133 at least), so that an infinite V times each is that infinity: 2^-132 more than p at
// most, which float32 does not see for p above 2^-108.
struct Terms {
  uint32_t hi, mid, lo;
  __device__ __forceinline__ explicit Terms(float p) {
    hi = __float_as_uint(p);
    const uint32_t least = min(hi, 0x10000u);
    mid = max(__float_as_uint(p - __uint_as_float(hi & 0xffff0000u)), least);
    lo = max(__float_as_uint(__uint_as_float(mid) - __uint_as_float(mid & 0xffff0000u)), least);
  }
};

template <int D, bool kE4m3>
struct Tile {
  using T = Decode<D, kE4m3>;
  u32x4_t k[T::kSums][T::kKLoads];
  Words<T::kWords> v[T::kGroups][T::kChunks][T::kPer];

  // Rows of kTile tokens at `base`, `token` bytes apart.
  __device__ __forceinline__ void load_k(const char* base, uint32_t token, int lane) {
    const uint32_t at = uint32_t(lane & 15) * token + uint32_t(lane >> 4) * 16;
#pragma unroll
    for (int u = 0; u < T::kSums; ++u)
#pragma unroll
      for (int i = 0; i < T::kKLoads; ++i)
        k[u][i] = load_row<u32x4_t, D * T::kBytes>(base + (at + u * 16 * token + i * 64));
  }
  __device__ __forceinline__ void load_v(const char* base, uint32_t token, int lane) {
    const uint32_t at =
        uint32_t(lane >> 4) * 4 * token + uint32_t(lane & 15) * T::kRun * T::kBytes;
#pragma unroll
    for (int a = 0; a < T::kGroups; ++a)
#pragma unroll
      for (int i = 0; i < T::kPer; ++i)
#pragma unroll
        for (int c = 0; c < T::kChunks; ++c)
          v[a][c][i] = load_words<T::kWords, D * T::kBytes>(
              base + (at + T::token(a, i, 0) * token + c * 16 * T::kRun * T::kBytes));
  }
  __device__ __forceinline__ u32x4_t k_operand(int u, int s) const {
    if constexpr (kE4m3) {
      const uint32_t a = k[u][s / 2][2 * (s % 2)], b = k[u][s / 2][2 * (s % 2) + 1];
      return u32x4_t{e4m3_to_bf16<false>(a), e4m3_to_bf16<true>(a), e4m3_to_bf16<false>(b),
                     e4m3_to_bf16<true>(b)};
    } else {
      return k[u][s];
    }
  }
  // Channel j of chunk c, tokens in the order of the scores.
  __device__ __forceinline__ Words<T::kPer / 2> v_operand(int group, int c, int j) const {
    Words<T::kPer / 2> r;
#pragma unroll
    for (int i = 0; i < T::kPer / 2; ++i) {
      uint32_t a, b;
      if constexpr (kE4m3) {
        const uint32_t x = v[group][c][2 * i].w[j / 4], y = v[group][c][2 * i + 1].w[j / 4];
        a = (j & 2) ? e4m3_to_bf16<true>(x) : e4m3_to_bf16<false>(x);
        b = (j & 2) ? e4m3_to_bf16<true>(y) : e4m3_to_bf16<false>(y);
      } else {
        a = v[group][c][2 * i].w[j / 2], b = v[group][c][2 * i + 1].w[j / 2];
      }
      r.w[i] = __builtin_amdgcn_perm(b, a, (j & 1) ? 0x07060302u : 0x05040100u);
    }
    return r;
  }
};

// The leading arguments are in registers when a wavefront starts, the others are loaded
// while the length and the table are.
template <int D, bool kE4m3>
__global__ void __launch_bounds__(256, D == 256 || (D == 64 && !kE4m3) ? 2 : 3)
block_decode_kernel(const int32_t* __restrict__ lengths, const int32_t* __restrict__ blocks,
                    const int32_t* __restrict__ table, int64_t tsb, int width, int kept, int hkv,
                    int num_pages, const char* __restrict__ k, const char* __restrict__ v,
                    const uint16_t* __restrict__ q_rows, const DecodeArgs p) {
  using T = Decode<D, kE4m3>;
  constexpr int kTile = T::kTile, kTiles = pd::kPageSize / kTile, kParts = kBlock / kTile;
  extern __shared__ floatx4_t shared[];  // [4][16] (m, l) pairs, then [4][kOut][4][heads]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane >> 4, col = lane & 15;
  int x = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
  const int splits = gridDim.y;
  // Workgroups of neighbouring x go to the XCDs in turn.  Where two heads' rows share a
  // 128-byte line, those of such a pair are eight apart, so that one XCD's L2 reads the line
  // once.
  constexpr int kPair = D * T::kBytes < 128 ? 2 : 1;
  if constexpr (kPair == 2) {
    const uint32_t all = gridDim.x * gridDim.y * gridDim.z;
    uint32_t id = x + gridDim.x * (split + gridDim.y * b);
    if ((id | 15) < all) id = (id & ~15u) | (id & 7) * 2 | (id >> 3 & 1);
    x = id % gridDim.x, id /= gridDim.x;
    split = id % gridDim.y, b = id / gridDim.y;
  }
  // The heads take turns on an XCD from sequence to sequence: where many workgroups follow
  // one another, a head that stays on its XCD is slower (64 sequences of 16384 e4m3 tokens,
  // Hkv 8, D 128, 8 splits: 441 and 386 us; 128 of 2048, Hkv 16, D 64: 137 and 111), where
  // few do it is faster by 4 to 6% (one split: 423 and 451).
  if (D == 64 || splits > 2) x = uint32_t(x + kPair * b) % gridDim.x;
  int g = x, head_tile = 0;
  if (int(gridDim.x) != hkv) g = x / p.tiles, head_tile = x % p.tiles;
  const int heads = min(p.group - 16 * head_tile, 16);
  const int head0 = g * p.group + 16 * head_tile;

  // Tiles of the sequence, parts of its blocks or of the listed ones; the wavefronts of all
  // its splits take them in turn, so that a short list's end is no split's alone.
  // Tile u, one a lane (below 0: no block of the table), and its page; the first of them are
  // looked up while the length is on its way.
  struct Place {
    int tile, page;
  };
  const auto look = [&](int u) {
    Place at;
    at.tile = u;
    if (blocks) {
      const int j = blocks[(int64_t(b) * hkv + g) * kept + min(u / kParts, kept - 1)];
      at.tile = uint32_t(j) < uint32_t(width * kPerPage) ? kParts * j + u % kParts : -1;
    }
    at.page = table[b * tsb + min(max(at.tile, 0) / kTiles, width - 1)];
    return at;
  };
  Place here = look(split + splits * (w + 4 * lane));
  const SplitRule rule{width, blocks ? kParts * kept : 0, kTile, p.two, splits};
  const int len = rule.length(lengths, b), used = rule.used(len);
  if (split >= used) return;
  if (used != splits) here = look(split + used * (w + 4 * lane));
  const int count = blocks ? kParts * kept : (len + kTile - 1) / kTile;
  const int mine = split + used * w, step_tiles = 4 * used;

  floatx4_t o[T::kOut];
#pragma unroll
  for (int i = 0; i < T::kOut; ++i) o[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  if (split < count) {
    u32x4_t q[T::kStepsQ];
    const uint16_t* qrow = q_rows + b * p.qsb + (head0 + min(col, heads - 1)) * p.qsh;
#pragma unroll
    for (int s = 0; s < T::kStepsQ; ++s) q[s] = load16(qrow + T::channel(s, row));
    const float scale2 = p.scale2 * (kE4m3 && p.k_scale ? p.k_scale[g] : 1.f);
    const uint32_t token = uint32_t(hkv) * D * T::kBytes;

    // One tile: scores of the loaded K, then the next tile's K is on its way
    // while the softmax and P V run, and its V while its scores do.
    Tile<D, kE4m3> t;
    const auto step = [&](int live, auto next_k, auto next_v) {
      floatx4_t s[T::kSums];
#pragma unroll
      for (int u = 0; u < T::kSums; ++u) s[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < T::kStepsQ; ++i)
#pragma unroll
        for (int u = 0; u < T::kSums; ++u) s[u] = mfma16(t.k_operand(u, i), q[i], s[u]);
      next_k();
      float x[T::kGroups][T::kPer], top = m;
#pragma unroll
      for (int a = 0; a < T::kGroups; ++a)
#pragma unroll
        for (int i = 0; i < T::kPer; ++i) x[a][i] = s[2 * a + (i >> 2)][i & 3] * scale2;
      if (live < kTile) {
#pragma unroll
        for (int a = 0; a < T::kGroups; ++a)
#pragma unroll
          for (int i = 0; i < T::kPer; ++i) {
            const bool in = T::token(a, i, row) < live;
            x[a][i] = in ? x[a][i] : -INFINITY;
            // A zero probability must not meet an infinity or NaN.
#pragma unroll
            for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
              for (int e = 0; e < T::kWords; ++e)
                t.v[a][c][i].w[e] = in ? t.v[a][c][i].w[e] : 0u;
          }
      }
#pragma unroll
      for (int a = 0; a < T::kGroups; ++a)
#pragma unroll
        for (int i = 0; i < T::kPer; ++i) top = fmaxf(top, x[a][i]);
      top = max_rows(top);
      const float base = top == -INFINITY ? 0.f : top;  // no score yet: exp2(-inf) = 0
      const float shrink = exp2_fast(m - base);
      m = top;
      float sum = 0.f;
#pragma unroll
      for (int a = 0; a < T::kGroups; ++a)
#pragma unroll
        for (int i = 0; i < T::kPer; ++i) {
          x[a][i] = exp2_fast(x[a][i] - base);
          sum += x[a][i];
        }
      l = l * shrink + sum;
      if (__any(shrink != 1.f)) {
#pragma unroll
        for (int i = 0; i < T::kOut; ++i) o[i] *= shrink;
      }
#pragma unroll
      for (int a = 0; a < T::kGroups; ++a) {
        // p = hi + mid + lo, each a bf16: all 24 bits of p.
        Words<T::kPer / 2> hi, mid, lo;
#pragma unroll
        for (int i = 0; i < T::kPer / 2; ++i) {
          const Terms x0(x[a][2 * i]), x1(x[a][2 * i + 1]);
          hi.w[i] = __builtin_amdgcn_perm(x1.hi, x0.hi, 0x07060302u);
          mid.w[i] = __builtin_amdgcn_perm(x1.mid, x0.mid, 0x07060302u);
          lo.w[i] = __builtin_amdgcn_perm(x1.lo, x0.lo, 0x07060302u);
        }
        // All words before the first product: 2 to 18 registers fewer (bf16, D 128: no spill,
        // 8 lists of 32 blocks 14.8 instead of 15.4 us).
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
          for (int j = 0; j < T::kRun; ++j) {
            const Words<T::kPer / 2> operand = t.v_operand(a, c, j);
            o[c * T::kRun + j] = mfma_pv<T::kPer>(operand, lo, o[c * T::kRun + j]);
            o[c * T::kRun + j] = mfma_pv<T::kPer>(operand, mid, o[c * T::kRun + j]);
            o[c * T::kRun + j] = mfma_pv<T::kPer>(operand, hi, o[c * T::kRun + j]);
          }
      }
      next_v();
    };

    for (int at = mine; at < count; at += 64 * step_tiles) {
      if (at != mine) here = look(at + lane * step_tiles);
      // Live tokens of the lane's tile (none: no such block or page).
      const bool known = at + lane * step_tiles < count && here.tile >= 0 && here.page >= 0 &&
                         here.page < num_pages;
      const int left = len - here.tile * kTile;
      const int live = known ? min(max(left, 0), kTile) : 0;
      const int first = live ? here.page * kTiles + here.tile % kTiles : 0;
      const uint64_t any = __ballot(live > 0);
      if (!any) continue;
      const int last = 63 - __builtin_clzll(any);
      const auto offset = [&](int i) {
        return int64_t(uint32_t(__builtin_amdgcn_readlane(first, i))) * kTile * token +
               int64_t(g) * D * T::kBytes;
      };
      int64_t from = offset(0);
      t.load_k(k + from, token, lane);
      t.load_v(v + from, token, lane);
      for (int i = 0; i < last; ++i) {
        from = offset(i + 1);
        step(__builtin_amdgcn_readlane(live, i), [&] { t.load_k(k + from, token, lane); },
             [&] { t.load_v(v + from, token, lane); });
      }
      step(__builtin_amdgcn_readlane(live, last), [] {}, [] {});
    }
    l = sum_rows(l);
  }

  // The four wavefronts' sums, relative to their largest maximum.
  float* ml = reinterpret_cast<float*>(shared);
  floatx4_t* part = shared + 32;
  if (row == 0) ml[(w * 16 + col) * 2] = m, ml[(w * 16 + col) * 2 + 1] = l;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[(i * 16 + col) * 2]);
  if (col < heads) {
    const float f = exp2_fast(m - (top == -INFINITY ? 0.f : top));
#pragma unroll
    for (int i = 0; i < T::kOut; ++i) part[((w * T::kOut + i) * 4 + row) * heads + col] = o[i] * f;
  }
  __syncthreads();
  const int64_t first = int64_t(b) * hkv * p.group + head0;
  for (int i = threadIdx.x; i < heads * D / 4; i += 256) {
    const int h = i / (D / 4), d = 4 * (i % (D / 4));
    float hm = -INFINITY, hl = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) hm = fmaxf(hm, ml[(j * 16 + h) * 2]);
    const float hb = hm == -INFINITY ? 0.f : hm;
    // Channels d..d+3 are channels j.. of row m of their chunk's MFMAs.
    const int row_m = d / T::kRun, j0 = row_m / 16 * T::kRun + d % T::kRun;
    const float* cell = reinterpret_cast<const float*>(part + ((j0 * 4 + row_m % 16 / 4) * heads + h)) +
                        row_m % 4;
    floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hl += ml[(j * 16 + h) * 2 + 1] * exp2_fast(ml[(j * 16 + h) * 2] - hb);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += cell[(j * T::kOut + e) * 16 * heads];
    }
    if (used == 1) {
      sum *= (kE4m3 && p.v_scale ? p.v_scale[g] : 1.f) / (hl == 0.f ? 1.f : hl);
      *reinterpret_cast<u32x2_t*>(p.out + (first + h) * D + d) =
          u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
    } else {
      const int64_t at = (first + h) * splits + split;
      if (hl != 0.f) *reinterpret_cast<floatx4_t*>(p.part_o + at * D + d) = sum;
      if (d == 0) p.part_ml[2 * at] = hm, p.part_ml[2 * at + 1] = hl;
    }
  }
}

// out = sum of the used splits' o 2^(m - M) over that of their l, times v_scale.  A split
// without tokens has l = 0, and its o is not there; one used split has written the output.
constexpr int kMaxSplits = PD_BLOCK_SPLITS;
constexpr int kFewSplits = 8;

// Up to kFewSplits (kMost of them at most): four columns a thread, every split in its
// registers.
template <int kMost>
__global__ void __launch_bounds__(256)
few_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                 uint16_t* __restrict__ out, const int32_t* __restrict__ lengths,
                 const SplitRule rule, int dim, int64_t total, const float* __restrict__ v_scale,
                 int group, int heads) {
  const int splits = rule.splits;
  const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  const int64_t bh = at / dim;
  const int col = int(at - bh * dim);
  const int used = rule.used(rule.length(lengths, int(bh / heads)));
  if (used == 1) return;
  floatx2_t ml[kMost];
  floatx4_t o[kMost];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int64_t from = bh * splits + min(i, used - 1);
    ml[i] = *reinterpret_cast<const floatx2_t*>(part_ml + 2 * from);
    o[i] = *reinterpret_cast<const floatx4_t*>(part_o + from * dim + col);
    top = fmaxf(top, ml[i][0]);
  }
  const float base = top == -INFINITY ? 0.f : top;
  floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const bool real = i < used && ml[i][1] != 0.f;
    const float f = exp2_fast(ml[i][0] - base);
    l += real ? f * ml[i][1] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += real ? f * o[i][e] : 0.f;
  }
  sum *= (v_scale ? v_scale[bh % heads / group] : 1.f) / (l == 0.f ? 1.f : l);
  *reinterpret_cast<u32x2_t*>(out + at) =
      u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
}

// More: 64 columns a workgroup, 16 rows of threads over the splits, kMost splits a thread.
constexpr int kMergeCols = 64;

template <int kMost>
__global__ void __launch_bounds__(256)
many_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                  uint16_t* __restrict__ out, const int32_t* __restrict__ lengths,
                  const SplitRule rule, int dim, const float* __restrict__ v_scale, int group,
                  int heads) {
  const int splits = rule.splits;
  constexpr int kLanes = kMergeCols / 4, kRows = 256 / kLanes;
  __shared__ float weight[kMaxSplits];
  __shared__ float waves[4][2];
  __shared__ floatx4_t sums[kRows][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t bh = blockIdx.x;
  const int col = blockIdx.y * kMergeCols + 4 * (tid % kLanes), row = tid / kLanes;
  const float* mine = part_o + bh * splits * dim + col;
  const int used = rule.used(rule.length(lengths, int(bh / heads)));
  if (used == 1) return;
  // The rows are on their way while the weights are made.
  floatx4_t o[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i)
    o[i] = *reinterpret_cast<const floatx4_t*>(mine +
                                               int64_t(min(row + i * kRows, used - 1)) * dim);
  float m = -INFINITY, l = 0.f;
  if (tid < used) {
    m = part_ml[(bh * splits + tid) * 2];
    l = part_ml[(bh * splits + tid) * 2 + 1];
  }
  const float wm = wave_max(m);
  if (lane == 0) waves[w][0] = wm;
  __syncthreads();
  const float top = fmaxf(fmaxf(waves[0][0], waves[1][0]), fmaxf(waves[2][0], waves[3][0]));
  const float f = exp2_fast(m - (top == -INFINITY ? 0.f : top));
  if (tid < used) weight[tid] = l == 0.f ? -1.f : f;
  const float wl = wave_sum(l == 0.f ? 0.f : l * f);
  if (lane == 0) waves[w][1] = wl;
  __syncthreads();
  floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const float x = row + i * kRows < used ? weight[row + i * kRows] : -1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += x < 0.f ? 0.f : x * o[i][e];
  }
  sums[row][tid % kLanes] = sum;
  __syncthreads();
  if (row) return;
#pragma unroll
  for (int r = 1; r < kRows; ++r) sum += sums[r][tid];
  const float total = waves[0][1] + waves[1][1] + waves[2][1] + waves[3][1];
  sum *= (v_scale ? v_scale[bh % heads / group] : 1.f) / (total == 0.f ? 1.f : total);
  *reinterpret_cast<u32x2_t*>(out + bh * dim + col) =
      u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
}

// The next power of two: what a batch's plan depends on.
int64_t batch_bucket(int32_t batch) {
  int64_t rows = 1;
  while (rows < batch) rows *= 2;
  return rows;
}

// Strides of Q's rows that keep them 16-byte aligned; that of a dimension of one entry is not
// used.
bool aligned_rows(int64_t stride_b, int64_t stride_h, int32_t batch, int32_t num_heads) {
  return (batch == 1 || stride_b % 8 == 0) && (num_heads == 1 || stride_h % 8 == 0);
}

int tile_tokens(int head_dim, int32_t cache_type) {
  return cache_type == PD_CACHE_E4M3 ? 32 : 4096 / head_dim;
}

int check_geometry(int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                   int32_t table_width, int64_t num_pages) {
  if (batch < 1 || num_heads < 1 || num_kv_heads < 1)
    return pd::fail(PD_EINVAL, "batch and heads must be positive");
  if (!pd::valid_head_dim(head_dim))
    return pd::fail(PD_EINVAL, "custom decode supports head_dim 64, 128, or 256");
  if (num_heads % num_kv_heads)
    return pd::fail(PD_EINVAL, "query heads must be divisible by KV heads");
  if (table_width < 1 || table_width >= 1 << 22)
    return pd::fail(PD_EINVAL, "table width must be in [1, 2^22)");
  if (num_pages < 1 || num_pages > 1 << 28)
    return pd::fail(PD_EINVAL, "the page pool must hold 1 to 2^28 pages");
  if (int64_t(num_kv_heads) * head_dim * 512 > INT32_MAX)
    return pd::fail(PD_EINVAL, "a page of one KV tensor must be below 2 GiB");
  return PD_OK;
}

}  // namespace

extern "C" int pd_select_blocks(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                                const void* bounds, int64_t num_pages, const int32_t* table,
                                int64_t table_stride_b, int32_t table_width,
                                const int32_t* lengths, uint64_t* keys, int32_t* blocks,
                                int32_t kept, int32_t first, int32_t last, int32_t batch,
                                int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                pd_stream_t stream) {
  pd::clear_error();
  if (const int bad =
          check_geometry(batch, num_heads, num_kv_heads, head_dim, table_width, num_pages))
    return bad;
  if (first < 0 || last < 1 || kept < first || kept - first < last)
    return pd::fail(PD_EINVAL, "kept blocks must hold the first ones and at least one last");
  if (!q || !bounds || !table || !lengths || !keys || !blocks || !all_aligned16(q, bounds) ||
      !aligned_rows(q_stride_b, q_stride_h, batch, num_heads))
    return pd::fail(PD_EINVAL, "tensors must be present, query rows and bounds 16-byte aligned");
  if (batch > 65535 || num_kv_heads > 65535)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const int group = num_heads / num_kv_heads;
  const int64_t wide = int64_t(table_width) * kPerPage;
  if (wide > kept) {
    const auto go = [&](auto dim, auto heads, auto whole) {
      // Eight workgroups a CU at most: a wavefront then takes several runs with the query in
      // its registers.  64 sequences of up to 32768 tokens, Hkv 8: 34.1 us with 1024
      // workgroups, 27.9 with 2048, 28.9 with 4096 (both launches); 8 of up to 65536: 14.4,
      // 15.7 and 16.8.
      constexpr int kPer = 4 * Scores<dim.value>::kPer;
      const int64_t groups = (wide + kPer - 1) / kPer;
      const int64_t most = std::max<int64_t>(1, 2048 / (int64_t(batch) * num_kv_heads));
      hipLaunchKernelGGL((score_kernel<dim.value, heads.value, whole.value>),
                         dim3(unsigned(std::min(groups, most)), num_kv_heads, batch), dim3(256), 0,
                         as_stream(stream), lengths, table, u16(q), u16(bounds), keys,
                         table_stride_b, table_width, num_kv_heads, int(num_pages), kept, first,
                         last, group, q_stride_b, q_stride_h);
    };
    const auto with = [&](auto dim) {
      if (group == 1)
        go(dim, std::integral_constant<int, 1>{}, std::true_type{});
      else if (group == 2)
        go(dim, std::integral_constant<int, 2>{}, std::true_type{});
      else if (group <= 4)
        go(dim, std::integral_constant<int, 4>{}, std::true_type{});
      else
        go(dim, std::integral_constant<int, 4>{}, std::false_type{});
    };
    if (head_dim == 64)
      with(std::integral_constant<int, 64>{});
    else if (head_dim == 128)
      with(std::integral_constant<int, 128>{});
    else
      with(std::integral_constant<int, 256>{});
    if (const int bad = launch_status("pd_select_blocks")) return bad;
  }
  hipLaunchKernelGGL(pick_kernel, dim3(num_kv_heads, batch), dim3(64 * kPickWaves), 0,
                     as_stream(stream), lengths, keys, blocks, table_width, num_kv_heads, kept,
                     first, last);
  return launch_status("pd_select_blocks");
}

extern "C" int pd_block_splits(int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                               int32_t head_dim, int32_t cache_type, int32_t entries,
                               int32_t listed, int32_t cus, int32_t* splits) {
  pd::clear_error();
  if (batch < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads ||
      entries < 1 || cus < 1 || !splits)
    return pd::fail(PD_EINVAL, "batch, heads, entries and CUs must be positive");
  if (!pd::valid_head_dim(head_dim) || !pd::valid_cache(cache_type))
    return pd::fail(PD_EINVAL, "unknown head_dim or cache type");
  const int64_t rows =
      batch_bucket(batch) * num_kv_heads * ((num_heads / num_kv_heads + 15) / 16);
  // Listed blocks are about as many for every row: one workgroup a CU, each with the most to
  // do behind its start of some 3 us (32 rows of 64 blocks, Hq 16 / Hkv 4 / D 256, e4m3: 53.4 us
  // in two splits, 59.3 in three, 56.2 in four, 70.8 in one; 17 of 37 blocks, Hq 32, which fill
  // half of their bucket: 23.5, 22.2, 23.7 and 32.8).  Whole caches differ in length: eight a
  // CU, so that no long one is left to a few (64 of 1 to 32768 tokens, Hq 32 / Hkv 8 / D 128:
  // 392 us, 409 with four, 506 with two; a short batch, 8 of 1000 to 9000, 24.7, 22.6 and
  // 23.5).  Nor is a long list or table: 128 tiles a workgroup at most, while the splits that
  // short sequences leave empty are few enough (32768 workgroups).
  const int64_t groups = int64_t(listed ? 1 : 8) * cus;
  const int64_t tiles = int64_t(entries) * (kBlock / tile_tokens(head_dim, cache_type));
  const int64_t want = std::max((groups + rows - 1) / rows, tiles / 128);
  const int64_t most =
      std::min<int64_t>({(tiles + 3) / 4, kMaxSplits, std::max<int64_t>(1, 32768 / rows)});
  *splits = int32_t(std::max<int64_t>(1, std::min(want, most)));
  return PD_OK;
}

extern "C" int pd_block_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                               const void* k, const void* v, int32_t cache_type,
                               int64_t num_pages, const int32_t* table, int64_t table_stride_b,
                               int32_t table_width, const int32_t* lengths,
                               const int32_t* blocks, int32_t kept, const float* k_scale,
                               const float* v_scale, float* part_o, float* part_ml,
                               int32_t splits, void* out, int32_t batch, int32_t num_heads,
                               int32_t num_kv_heads, int32_t head_dim, double scale,
                               pd_stream_t stream) {
  pd::clear_error();
  if (const int bad =
          check_geometry(batch, num_heads, num_kv_heads, head_dim, table_width, num_pages))
    return bad;
  if (!pd::valid_cache(cache_type)) return pd::fail(PD_EINVAL, "unknown cache type");
  if (cache_type == PD_CACHE_BF16 && (k_scale || v_scale))
    return pd::fail(PD_EINVAL, "scales belong to an e4m3 cache");
  if (blocks && (kept < 1 || kept > 1 << 26))
    return pd::fail(PD_EINVAL, "the list must hold at least one block, at most 2^26");
  if (splits < 1 || splits > kMaxSplits)
    return pd::fail(PD_EINVAL, "splits must be in [1, %d]", kMaxSplits);
  if (!q || !k || !v || !table || !lengths || !out || (splits > 1 && (!part_o || !part_ml)) ||
      !all_aligned16(q, k, v, part_o, part_ml, out) ||
      !aligned_rows(q_stride_b, q_stride_h, batch, num_heads))
    return pd::fail(PD_EINVAL, "tensors must be present, with 16-byte aligned rows");
  DecodeArgs p;
  p.k_scale = k_scale, p.v_scale = v_scale, p.part_o = part_o, p.part_ml = part_ml;
  p.out = u16(out), p.qsb = q_stride_b, p.qsh = q_stride_h;
  p.group = num_heads / num_kv_heads, p.tiles = (p.group + 15) / 16;
  p.scale2 = float(scale * 1.4426950408889634);
  // With more workgroups than the device holds, a workgroup's start is worth another tile: 64
  // sequences of 500 to 1500 tokens with room for 32768 take 38.3 us with one, 37.6 with two,
  // 40.1 with four, 8 of 1000 to 9000 24.5, 23.0 and 23.7.
  p.two = batch_bucket(batch) * num_kv_heads * p.tiles * splits > 2048;
  const int64_t columns = int64_t(num_kv_heads) * p.tiles;
  if (batch > 65535 || columns * splits * batch > 0x7fffffff ||
      int64_t(batch) * num_heads > 0x7fffffff)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const dim3 grid = {unsigned(columns), unsigned(splits), unsigned(batch)};
  const unsigned lds = unsigned(128 + 4 * (p.group < 16 ? p.group : 16) * head_dim) * 4;
  bool fits = true;
  pd::for_cache(head_dim, cache_type, [&](auto dim, auto e4m3) {
    const auto kernel = block_decode_kernel<dim.value, e4m3.value>;
    if (lds > 64 * 1024 &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)) != hipSuccess) {
      fits = false;
      return;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds,
                       as_stream(stream), lengths, blocks, table, table_stride_b, table_width,
                       kept, num_kv_heads, int(num_pages), static_cast<const char*>(k),
                       static_cast<const char*>(v), u16(q), p);
  });
  if (!fits) return pd::fail(PD_ELAUNCH, "pd_block_decode: LDS size");
  if (const int bad = launch_status("pd_block_decode")) return bad;
  if (splits == 1) return PD_OK;
  const int tile = tile_tokens(head_dim, cache_type);
  const SplitRule rule{table_width, blocks ? kBlock / tile * kept : 0, tile, p.two, splits};
  if (splits <= kFewSplits) {
    const int64_t total = int64_t(batch) * num_heads * head_dim;
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(unsigned((total + 1023) / 1024)), dim3(256), 0,
                         as_stream(stream), part_o, part_ml, p.out, lengths, rule, head_dim, total,
                         v_scale, p.group, num_heads);
    };
    go(splits <= 2 ? few_merge_kernel<2> : splits <= 4 ? few_merge_kernel<4> : few_merge_kernel<8>);
  } else {
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(unsigned(batch * num_heads), head_dim / kMergeCols),
                         dim3(256), 0, as_stream(stream), part_o, part_ml, p.out, lengths, rule, head_dim,
                         v_scale, p.group, num_heads);
    };
    go(splits <= 16   ? many_merge_kernel<1>
       : splits <= 32 ? many_merge_kernel<2>
       : splits <= 64 ? many_merge_kernel<4>
                      : many_merge_kernel<8>);
  }
  return launch_status("pd_block_decode");
}
