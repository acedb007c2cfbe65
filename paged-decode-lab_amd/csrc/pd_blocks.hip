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
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

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

// Scores are sums of exact products in 64 bits, so the order of a sum moves no
// block: two implementations pick the same ones unless their scores agree to 15
// digits without being equal.
struct SelectArgs {
  const uint16_t *q, *bounds;
  const int32_t *table, *lengths;
  uint64_t* keys;  // [batch][hkv][width * 4]
  int32_t* blocks;
  int64_t qsb, qsh, tsb, num_pages;
  int width, hkv, group, kept, first, last;
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

template <int kLanes>
__device__ __forceinline__ double sum_lanes(double x, int lane) {
  if constexpr (kLanes > 16) x += xor_lanes64<16>(x, lane);
  if constexpr (kLanes > 8) x += xor_lanes64<8>(x, lane);
  x += xor_lanes64<4>(x, lane);
  x += xor_lanes64<2>(x, lane);
  return x + xor_lanes64<1>(x, lane);
}

// A block's bounds are kLanes lanes of eight channels; a wavefront takes kRuns
// runs of 64 / kLanes blocks, so a head's query is widened once for all of them.
template <int D>
struct Scores {
  static constexpr int kLanes = D / 8, kPer = 64 / kLanes, kRuns = 4;
  static constexpr int kBlocks = 4 * kRuns * kPer;  // of a workgroup
};

template <int D>
__global__ void __launch_bounds__(256) score_kernel(const SelectArgs p) {
  using S = Scores<D>;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int g = blockIdx.y, b = blockIdx.z;
  const int n = block_count(p.lengths, b, p.width);
  const int end = n - p.last;
  const int j0 = p.first + blockIdx.x * S::kBlocks + w * S::kRuns * S::kPer;
  if (n <= p.kept || j0 >= end) return;
  const int part = lane % S::kLanes, mine = lane / S::kLanes;
  double lo[S::kRuns][8], hi[S::kRuns][8], best[S::kRuns];
  bool known[S::kRuns];
#pragma unroll
  for (int r = 0; r < S::kRuns; ++r) {
    const int j = min(j0 + r * S::kPer + mine, end - 1);
    const int64_t page = p.table[b * p.tsb + j / kPerPage];
    known[r] = page >= 0 && page < p.num_pages;
    const uint16_t* at =
        p.bounds + (((known[r] ? page : 0) * kPerPage + j % kPerPage) * p.hkv + g) * 2 * D + 8 * part;
    float x[8], y[8];
    unpack8(load16(at), x);
    unpack8(load16(at + D), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[r][i] = x[i], hi[r][i] = y[i];
    best[r] = -__builtin_inf();
  }
  const uint16_t* q = p.q + b * p.qsb + int64_t(g) * p.group * p.qsh + 8 * part;
  for (int h = 0; h < p.group; ++h, q += p.qsh) {
    float x[8];
    unpack8(load16(q), x);
    double sum[S::kRuns] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double up = x[i] != x[i] ? x[i] : fmaxf(x[i], 0.f);
      const double down = fminf(x[i], 0.f);
#pragma unroll
      for (int r = 0; r < S::kRuns; ++r)
        sum[r] = __builtin_fma(up, hi[r][i], __builtin_fma(down, lo[r][i], sum[r]));
    }
#pragma unroll
    for (int r = 0; r < S::kRuns; ++r) {
      const double s = sum_lanes<S::kLanes>(sum[r], lane);
      best[r] = s > best[r] || s != s ? s : best[r];
    }
  }
  if (part) return;
  uint64_t* keys = p.keys + (int64_t(b) * p.hkv + g) * p.width * kPerPage;
#pragma unroll
  for (int r = 0; r < S::kRuns; ++r) {
    const int j = j0 + r * S::kPer + mine;
    if (j < end) keys[j] = known[r] ? score_key(best[r]) : 0;  // no such page: last
  }
}

// The r highest keys of a (sequence, kv head): the threshold found digit by
// digit from the highest bit in which the keys differ, then one ordered pass
// that writes the forced blocks, those above the threshold and the first ones at
// it.
constexpr int kDigit = 11, kBins = 1 << kDigit;

__global__ void __launch_bounds__(256) pick_kernel(const SelectArgs p) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint64_t wave_keys[2][4];
  __shared__ uint32_t wave_counts[4], found[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = blockIdx.x, b = blockIdx.y;
  const int n = block_count(p.lengths, b, p.width);
  int32_t* out = p.blocks + (int64_t(b) * p.hkv + g) * p.kept;
  if (n <= p.kept) {
    for (int i = tid; i < p.kept; i += 256) out[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* keys = p.keys + (int64_t(b) * p.hkv + g) * p.width * kPerPage;
  const int begin = p.first, end = n - p.last;
  uint32_t need = p.kept - p.first - p.last;  // < end - begin
  uint64_t every = ~uint64_t(0), some = 0;
  for (int j = begin + tid; j < end; j += 256) every &= keys[j], some |= keys[j];
  for (int m = 1; m < 64; m *= 2) {
    every &= __shfl_xor(every, m);
    some |= __shfl_xor(some, m);
  }
  if (lane == 0) wave_keys[0][w] = every, wave_keys[1][w] = some;
  __syncthreads();
  every = wave_keys[0][0] & wave_keys[0][1] & wave_keys[0][2] & wave_keys[0][3];
  some = wave_keys[1][0] | wave_keys[1][1] | wave_keys[1][2] | wave_keys[1][3];

  // Keys above `edge` (of the bits at `shift` and up) are in; `need` of those at it.
  uint64_t edge = 0;
  const uint64_t differ = every ^ some;
  int shift = differ ? 64 - __builtin_clzll(differ) : 0;
  uint32_t at_edge = end - begin;  // keys that agree with the edge so far
  edge = shift < 64 ? some >> shift : 0;
  if (need == 0) {
    edge = ~uint64_t(0), shift = 0, at_edge = 0;
  } else {
    while (shift > 0 && at_edge != need) {
      const int next = max(shift - kDigit, 0);
      for (int i = tid; i < kBins; i += 256) bins[i] = 0;
      __syncthreads();
      for (int j = begin + tid; j < end; j += 256) {
        const uint64_t key = keys[j];
        if ((shift < 64 ? key >> shift : 0) == edge)
          atomicAdd(&bins[(key >> next) & ((1u << (shift - next)) - 1)], 1u);
      }
      __syncthreads();
      // From the highest bin down: the one in which the count reaches `need`.
      uint32_t sum = 0;
      constexpr int kOwn = kBins / 256;
      const int top = kBins - 1 - tid * kOwn;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) sum += bins[top - i];
      uint32_t before = sum;
      for (int m = 1; m < 64; m *= 2) {
        const uint32_t x = __shfl_up(before, m);
        if (lane >= m) before += x;
      }
      if (lane == 63) wave_counts[w] = before;
      __syncthreads();
      for (int i = 0; i < w; ++i) before += wave_counts[i];
      before -= sum;
      if (before < need && before + sum >= need) {
        uint32_t above = before;
        int bin = top;
        while (above + bins[bin] < need) above += bins[bin--];
        found[0] = bin, found[1] = above;
      }
      __syncthreads();
      const uint32_t bin = found[0];
      need -= found[1];
      at_edge = bins[bin];
      edge = (shift < 64 ? edge << (shift - next) : 0) | bin;
      shift = next;
      __syncthreads();
    }
  }
  uint32_t written = 0, ties = 0;
  for (int base = 0; base < n; base += 256) {
    const int j = base + tid;
    bool in = j < n && (j < begin || j >= end), tie = false;
    if (j >= begin && j < end) {
      const uint64_t key = shift < 64 ? keys[j] >> shift : 0;
      in = key > edge;
      tie = key == edge;
    }
    const uint64_t below = (uint64_t(1) << lane) - 1;
    const uint64_t mask_in = __ballot(in), mask_tie = __ballot(tie);
    __syncthreads();
    if (lane == 0)
      wave_counts[w] = uint32_t(__popcll(mask_in)) | uint32_t(__popcll(mask_tie)) << 16;
    __syncthreads();
    uint32_t ahead = 0, all = 0;
    for (int i = 0; i < 4; ++i) {
      if (i < w) ahead += wave_counts[i];
      all += wave_counts[i];
    }
    // Ties ahead of this block that are in: the first `need` of them.
    const uint32_t tied = ties + (ahead >> 16) + __popcll(mask_tie & below);
    const uint32_t place = written + (ahead & 0xffff) + __popcll(mask_in & below) + min(tied, need);
    if (in || (tie && tied < need)) out[place] = j;
    written += all & 0xffff;
    ties += all >> 16;
  }
}

// ------------------------------------------------------------------ attention

struct DecodeArgs {
  const uint16_t* q;
  const char *k, *v;
  const int32_t *table, *lengths, *blocks;  // blocks null: every block
  const float *k_scale, *v_scale;
  float *part_o, *part_ml;  // [batch][heads][splits][D], [batch][heads][splits][2]
  uint16_t* out;
  int64_t qsb, qsh, tsb, num_pages;
  int width, hkv, group, tiles, kept, splits;  // tiles: of 16 query heads a kv head
  float scale2;                                // scale log2 e
};

// A wavefront's tile: 32 tokens.  S^T = K Q^T and O^T = V^T P^T with 16 x 16 x 32
// MFMAs.  In both results a lane's column is query head lane % 16, so the softmax
// state is one scalar a lane, and the layout of the scores (tokens 16 u + 4 (lane /
// 16) + r in element r of half u) is the operand layout of P^T with its tokens in
// that order, which V's rows are loaded in too.  V^T's operand wants eight tokens
// of a channel in a lane: a lane loads kRun channels of eight tokens and turns the
// 8 x kRun square with byte permutes; row m of the MFMA of channel j is channel
// kRun m + j.  No value crosses a lane or the LDS before the end.
template <int D, bool kE4m3>
struct Decode {
  static constexpr int kBytes = kE4m3 ? 1 : 2;
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
};

template <int N>
struct Words {
  uint32_t w[N];
};

template <int N>
__device__ __forceinline__ Words<N> load_words(const char* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else if constexpr (N == 2) {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

// Two e4m3 bytes of x (the lower or the upper ones) as bf16, exactly.
template <bool kUpper>
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, kUpper));
}

template <int D, bool kE4m3>
struct Tile {
  using T = Decode<D, kE4m3>;
  u32x4_t k[2][T::kKLoads];
  Words<T::kWords> v[T::kChunks][8];

  // `token`: bytes between tokens; rows of 32 tokens at `base`.
  __device__ __forceinline__ void load_k(const char* base, uint32_t token, int lane) {
    const uint32_t at = uint32_t(lane & 15) * token + uint32_t(lane >> 4) * 16;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < T::kKLoads; ++i)
        k[u][i] = *reinterpret_cast<const u32x4_t*>(base + (at + u * 16 * token + i * 64));
  }
  __device__ __forceinline__ void load_v(const char* base, uint32_t token, int lane) {
    const uint32_t at =
        uint32_t(lane >> 4) * 4 * token + uint32_t(lane & 15) * T::kRun * T::kBytes;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < T::kChunks; ++c)
        v[c][i] = load_words<T::kWords>(
            base + (at + ((i & 3) + 16 * (i >> 2)) * token + c * 16 * T::kRun * T::kBytes));
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
  __device__ __forceinline__ u32x4_t v_operand(int c, int j) const {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      if constexpr (kE4m3) {
        a = (j & 2) ? e4m3_to_bf16<true>(v[c][2 * i].w[j / 4])
                    : e4m3_to_bf16<false>(v[c][2 * i].w[j / 4]);
        b = (j & 2) ? e4m3_to_bf16<true>(v[c][2 * i + 1].w[j / 4])
                    : e4m3_to_bf16<false>(v[c][2 * i + 1].w[j / 4]);
      } else {
        a = v[c][2 * i].w[j / 2], b = v[c][2 * i + 1].w[j / 2];
      }
      r[i] = __builtin_amdgcn_perm(b, a, (j & 1) ? 0x07060302u : 0x05040100u);
    }
    return r;
  }
};

template <int D, bool kE4m3>
__global__ void __launch_bounds__(256) block_decode_kernel(const DecodeArgs p) {
  using T = Decode<D, kE4m3>;
  extern __shared__ float shared[];  // [4][16][2] (m, l), then [4][heads][D]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane >> 4, col = lane & 15;
  // Kv heads of a sequence's split are neighbours: their rows of a token are too.
  int id = blockIdx.x;
  const int tile = id % p.tiles;
  id /= p.tiles;
  const int g = id % p.hkv;
  id /= p.hkv;
  const int split = id % p.splits, b = id / p.splits;
  const int heads = min(p.group - 16 * tile, 16);
  const int head0 = g * p.group + 16 * tile;

  // Whole blocks of the list a split, the same for each of a sequence's splits; a
  // multiple of 4, so that no wavefront gets more than the others' and one.
  const int64_t len = min(int64_t(max(p.lengths[b], 0)), int64_t(p.width) * pd::kPageSize);
  int entries = int((len + kBlock - 1) / kBlock);
  if (p.blocks) entries = min(entries ? p.kept : 0, p.kept);
  const int chunk = ((entries + p.splits - 1) / p.splits + 3) & ~3;
  const int s0 = split * chunk, s1 = min(s0 + chunk, entries);

  floatx4_t o[T::kOut];
#pragma unroll
  for (int i = 0; i < T::kOut; ++i) o[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  if (s0 < s1) {
    u32x4_t q[T::kStepsQ];
    const uint16_t* qrow = p.q + b * p.qsb + (head0 + min(col, heads - 1)) * p.qsh;
#pragma unroll
    for (int s = 0; s < T::kStepsQ; ++s) q[s] = load16(qrow + T::channel(s, row));
    const float scale2 = p.scale2 * (kE4m3 && p.k_scale ? p.k_scale[g] : 1.f);
    const uint32_t token = uint32_t(p.hkv) * D * T::kBytes;

    // One tile: scores of the loaded K, then the next tile's K is on its way
    // while the softmax and P V run, and its V while its scores do.
    Tile<D, kE4m3> t;
    const auto step = [&](int live, auto next_k, auto next_v) {
      floatx4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int i = 0; i < T::kStepsQ; ++i) {
        s[0] = mfma16(t.k_operand(0, i), q[i], s[0]);
        s[1] = mfma16(t.k_operand(1, i), q[i], s[1]);
      }
      next_k();
      float x[8], top = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * scale2;
      if (live < 32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool in = 16 * (i >> 2) + 4 * row + (i & 3) < live;
          x[i] = in ? x[i] : -INFINITY;
          // A zero probability must not meet an infinity or NaN.
#pragma unroll
          for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
            for (int e = 0; e < T::kWords; ++e) t.v[c][i].w[e] = in ? t.v[c][i].w[e] : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
      top = max_rows(top);
      const float base = top == -INFINITY ? 0.f : top;  // no score yet: exp2(-inf) = 0
      const float shrink = exp2_fast(m - base);
      m = top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = exp2_fast(x[i] - base);
        sum += x[i];
      }
      l = l * shrink + sum;
      // p = hi + lo to 16 significant bits: bf16 probabilities alone would add an
      // error as large as the output's own rounding.
      u32x4_t hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(x[2 * i]), c = __float_as_uint(x[2 * i + 1]);
        hi[i] = __builtin_amdgcn_perm(c, a, 0x07060302u);
        lo[i] = pack_bf16(x[2 * i] - __uint_as_float(a & 0xffff0000u),
                          x[2 * i + 1] - __uint_as_float(c & 0xffff0000u));
      }
      if (__any(shrink != 1.f)) {
#pragma unroll
        for (int i = 0; i < T::kOut; ++i) o[i] *= shrink;
      }
#pragma unroll
      for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
        for (int j = 0; j < T::kRun; ++j) {
          const u32x4_t a = t.v_operand(c, j);
          o[c * T::kRun + j] = mfma16(a, lo, o[c * T::kRun + j]);
          o[c * T::kRun + j] = mfma16(a, hi, o[c * T::kRun + j]);
        }
      next_v();
    };

    // Entries w, w + 4, ... of the split, 64 at a time, one a lane: its page and
    // its live tokens (none: no such block or page).
    for (int at = s0 + w; at < s1; at += 4 * 64) {
      const int i = at + 4 * lane;
      int page = 0, live = 0, quarter = 0;
      if (i < s1) {
        const int j = p.blocks ? p.blocks[(int64_t(b) * p.hkv + g) * p.kept + i] : i;
        const int64_t left = len - int64_t(j) * kBlock;
        if (j >= 0 && left > 0) {
          page = p.table[b * p.tsb + j / kPerPage];
          quarter = j % kPerPage;
          live = page >= 0 && page < p.num_pages ? int(min(left, int64_t(kBlock))) : 0;
          if (!live) page = 0;
        }
      }
      const uint64_t any = __ballot(live > 0);
      if (!any) continue;
      const int last = 63 - __builtin_clzll(any);
      // Of tile u: entry u / 2, its first or second 32 tokens.
      const auto offset = [&](int u) {
        const int64_t pg = __builtin_amdgcn_readlane(page, u >> 1);
        const int qt = __builtin_amdgcn_readlane(quarter, u >> 1);
        return ((pg * kPerPage + qt) * kBlock + 32 * (u & 1)) * token + int64_t(g) * D * T::kBytes;
      };
      const auto tokens = [&](int u) {
        return __builtin_amdgcn_readlane(live, u >> 1) - 32 * (u & 1);
      };
      const int tiles = 2 * last + (tokens(2 * last + 1) > 0 ? 2 : 1);
      int64_t here = offset(0);
      t.load_k(p.k + here, token, lane);
      t.load_v(p.v + here, token, lane);
      for (int u = 0; u + 1 < tiles; ++u) {
        here = offset(u + 1);
        step(tokens(u), [&] { t.load_k(p.k + here, token, lane); },
             [&] { t.load_v(p.v + here, token, lane); });
      }
      step(tokens(tiles - 1), [] {}, [] {});
    }
    l = sum_rows(l);
  }

  // The four wavefronts' sums, relative to their largest maximum.
  float* ml = shared;
  float* part = shared + 128;
  if (row == 0) ml[(w * 16 + col) * 2] = m, ml[(w * 16 + col) * 2 + 1] = l;
  __syncthreads();
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[(i * 16 + col) * 2]);
  const float base = top == -INFINITY ? 0.f : top;
  if (col < heads) {
    const float f = exp2_fast(m - base);
#pragma unroll
    for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < T::kRun; ++j)
          part[(w * heads + col) * D + (c * 16 + 4 * row + r) * T::kRun + j] =
              o[c * T::kRun + j][r] * f;
  }
  __syncthreads();
  const int64_t first = int64_t(b) * p.hkv * p.group + head0;
  for (int i = threadIdx.x; i < heads * D / 4; i += 256) {
    const int h = i / (D / 4), d = 4 * (i % (D / 4));
    float hm = -INFINITY, hl = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) hm = fmaxf(hm, ml[(k * 16 + h) * 2]);
    const float hb = hm == -INFINITY ? 0.f : hm;
    floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      hl += ml[(k * 16 + h) * 2 + 1] * exp2_fast(ml[(k * 16 + h) * 2] - hb);
      sum += *reinterpret_cast<const floatx4_t*>(part + (k * heads + h) * D + d);
    }
    if (p.splits == 1) {
      const float scale = (kE4m3 && p.v_scale ? p.v_scale[g] : 1.f) / (hl == 0.f ? 1.f : hl);
      sum *= scale;
      *reinterpret_cast<u32x2_t*>(p.out + (first + h) * D + d) =
          u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
    } else {
      const int64_t at = (first + h) * p.splits + split;
      if (hl != 0.f) *reinterpret_cast<floatx4_t*>(p.part_o + at * D + d) = sum;
      if (d == 0) p.part_ml[2 * at] = hm, p.part_ml[2 * at + 1] = hl;
    }
  }
  (void)total;
}

// out = sum of the splits' o 2^(m - M) over that of their l, times v_scale.
// An empty split has l = 0 and its o is not there.
constexpr int kMaxSplits = PD_BLOCK_SPLITS;

template <int D>
__global__ void __launch_bounds__(256)
block_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                   const float* __restrict__ v_scale, uint16_t* __restrict__ out, int group,
                   int heads, int splits) {
  constexpr int kLanes = D / 4, kRows = 256 / kLanes;
  __shared__ float weight[kMaxSplits];
  __shared__ float waves[4][2];
  __shared__ floatx4_t sums[kRows][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t bh = blockIdx.x;
  float m = -INFINITY, l = 0.f;
  if (tid < splits) {
    m = part_ml[(bh * splits + tid) * 2];
    l = part_ml[(bh * splits + tid) * 2 + 1];
  }
  const float wm = wave_max(m);
  if (lane == 0) waves[w][0] = wm;
  __syncthreads();
  const float top = fmaxf(fmaxf(waves[0][0], waves[1][0]), fmaxf(waves[2][0], waves[3][0]));
  const float f = exp2_fast(m - (top == -INFINITY ? 0.f : top));
  if (tid < splits) weight[tid] = l == 0.f ? -1.f : f;
  const float wl = wave_sum(l == 0.f ? 0.f : l * f);
  if (lane == 0) waves[w][1] = wl;
  __syncthreads();
  const int part = tid % kLanes;
  floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int s = tid / kLanes; s < splits; s += kRows) {
    const float x = weight[s];
    if (!(x < 0.f))
      sum += x * *reinterpret_cast<const floatx4_t*>(part_o + (bh * splits + s) * D + 4 * part);
  }
  sums[tid / kLanes][part] = sum;
  __syncthreads();
  if (tid >= kLanes) return;
#pragma unroll
  for (int r = 1; r < kRows; ++r) sum += sums[r][part];
  const float total = waves[0][1] + waves[1][1] + waves[2][1] + waves[3][1];
  sum *= (v_scale ? v_scale[bh % heads / group] : 1.f) / (total == 0.f ? 1.f : total);
  *reinterpret_cast<u32x2_t*>(out + bh * D + 4 * part) =
      u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
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
  if (num_pages < 1 || num_pages > INT32_MAX)
    return pd::fail(PD_EINVAL, "the page pool must hold at least one page");
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
      q_stride_b % 8 || q_stride_h % 8)
    return pd::fail(PD_EINVAL, "tensors must be present, query rows and bounds 16-byte aligned");
  if (batch > 65535 || num_kv_heads > 65535)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  SelectArgs p;
  p.q = u16(q), p.bounds = u16(bounds), p.table = table, p.lengths = lengths, p.keys = keys;
  p.blocks = blocks, p.qsb = q_stride_b, p.qsh = q_stride_h, p.tsb = table_stride_b;
  p.num_pages = num_pages, p.width = table_width, p.hkv = num_kv_heads;
  p.group = num_heads / num_kv_heads, p.kept = kept, p.first = first, p.last = last;
  const int64_t most = int64_t(table_width) * kPerPage - first - last;
  if (table_width * kPerPage > kept && most > 0) {
    const auto go = [&](auto kernel, int per) {
      hipLaunchKernelGGL(kernel, dim3(unsigned((most + per - 1) / per), num_kv_heads, batch),
                         dim3(256), 0, as_stream(stream), p);
    };
    if (head_dim == 64)
      go(score_kernel<64>, Scores<64>::kBlocks);
    else if (head_dim == 128)
      go(score_kernel<128>, Scores<128>::kBlocks);
    else
      go(score_kernel<256>, Scores<256>::kBlocks);
    if (const int bad = launch_status("pd_select_blocks")) return bad;
  }
  hipLaunchKernelGGL(pick_kernel, dim3(num_kv_heads, batch), dim3(256), 0, as_stream(stream), p);
  return launch_status("pd_select_blocks");
}

extern "C" int pd_block_splits(int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                               int32_t entries, int32_t cus, int32_t* splits) {
  pd::clear_error();
  if (batch < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads ||
      entries < 1 || cus < 1 || !splits)
    return pd::fail(PD_EINVAL, "batch, heads, entries and CUs must be positive");
  int64_t rows = 1;
  while (rows < batch) rows *= 2;
  rows *= int64_t(num_kv_heads) * ((num_heads / num_kv_heads + 15) / 16);
  const int64_t want = (8 * int64_t(cus) + rows - 1) / rows;
  const int64_t most = (int64_t(entries) + 3) / 4;
  int64_t s = want < most ? want : most;
  if (s > kMaxSplits) s = kMaxSplits;
  *splits = int32_t(s < 1 ? 1 : s);
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
  if (blocks && kept < 1) return pd::fail(PD_EINVAL, "the list must hold at least one block");
  if (splits < 1 || splits > kMaxSplits)
    return pd::fail(PD_EINVAL, "splits must be in [1, %d]", kMaxSplits);
  if (!q || !k || !v || !table || !lengths || !out || (splits > 1 && (!part_o || !part_ml)) ||
      !all_aligned16(q, k, v, part_o, out) || q_stride_b % 8 || q_stride_h % 8)
    return pd::fail(PD_EINVAL, "tensors must be present, with 16-byte aligned rows");
  DecodeArgs p;
  p.q = u16(q), p.k = static_cast<const char*>(k), p.v = static_cast<const char*>(v);
  p.table = table, p.lengths = lengths, p.blocks = blocks, p.k_scale = k_scale;
  p.v_scale = v_scale, p.part_o = part_o, p.part_ml = part_ml, p.out = u16(out);
  p.qsb = q_stride_b, p.qsh = q_stride_h, p.tsb = table_stride_b, p.num_pages = num_pages;
  p.width = table_width, p.hkv = num_kv_heads, p.group = num_heads / num_kv_heads;
  p.tiles = (p.group + 15) / 16, p.kept = kept, p.splits = splits;
  p.scale2 = float(scale * 1.4426950408889634);
  const int64_t groups = int64_t(batch) * splits * num_kv_heads * p.tiles;
  if (groups > 0x7fffffff || int64_t(batch) * num_heads > 0x7fffffff)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const unsigned lds = unsigned(128 + 4 * (p.group < 16 ? p.group : 16) * head_dim) * 4;
  pd::for_cache(head_dim, cache_type, [&](auto dim, auto e4m3) {
    hipLaunchKernelGGL((block_decode_kernel<dim.value, e4m3.value>), dim3(unsigned(groups)),
                       dim3(256), lds, as_stream(stream), p);
  });
  if (const int bad = launch_status("pd_block_decode")) return bad;
  if (splits == 1) return PD_OK;
  const auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(batch * num_heads)), dim3(256), 0, as_stream(stream),
                       part_o, part_ml, v_scale, p.out, p.group, num_heads, splits);
  };
  if (head_dim == 64)
    merge(block_merge_kernel<64>);
  else if (head_dim == 128)
    merge(block_merge_kernel<128>);
  else
    merge(block_merge_kernel<256>);
  return launch_status("pd_block_decode merge");
}
