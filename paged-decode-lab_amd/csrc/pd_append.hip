// Keys and values of new tokens into a paged cache, with the position rotation
// of queries and keys on the way, for MI355X (gfx950).
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// over the pairs (j, j + half) or (2j, 2j + 1) of a head's leading 2 half
// elements, cos and sin from float32 rows of a table, one row a position.  The
// products and the difference are rounded one by one (no fused multiply-add):
// the same float32 value as separate operations give, so that the rounding to
// bf16 or e4m3 behind it falls the same way too.  An e4m3 cache holds
// clamp(x / scale[kv head], +-448), rounded to nearest even; NaN stays NaN.
//
// Bound: HBM bytes.  A thread takes 16 elements of a head, for a rotated head
// both halves of eight pairs, so nothing crosses a lane.
//
// Bounds (smallest and largest stored key per channel) are made of the blocks of
// 64 slots whose last slot a call writes: for prompts in a second launch, from the
// cache.  A decode step's rows have them made in the launch that writes them.
// A block's other keys may be written by other workgroups of it, so the one that
// makes the bounds takes this call's keys from their source, rotated and rounded
// as they are stored, and the others from the cache; no workgroup waits for
// another.  (In the launch of four prompts of 300 to 4001 rows they cost it its
// occupancy: 67 us, 49 in two launches.)
//
// Measured on MI355X, bounds included: those prompts (bf16, Hq 32 / Hkv 8 / D
// 128, 209 MB) 42.8 + 5.7 us, 4.9 TB/s in the first launch; 2049 e4m3 rows, Hq =
// Hkv = 16, D 64, 8.4 + 4.0; a decode step of 64 rows 4.9 (6.1 in two launches),
// of one row 4.9, launch and latencies.
#include <hip/hip_runtime.h>

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

struct AppendArgs {
  const uint16_t *q, *k, *v;
  const float* rope;
  uint16_t* q_out;
  char *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  uint16_t* bounds;  // or null
  int64_t q_stride, k_stride, v_stride, q_out_stride, max_positions;
  int hq, hkv, half;
};

// A scale of a kv head, and the power of two that takes it into [2^-85, 2^64): there no
// remainder of a quotient has a bit below float32's smallest number.
struct Scale {
  float lift, value, inverse;
  __device__ __forceinline__ Scale(const float* scales, int head) {
    const float d = scales ? scales[head] : 1.f;
    lift = d < 0x1p-62f ? 0x1p64f : d > 0x1p62f ? 0x1p-64f : 1.f;
    value = d * lift;
    inverse = 1.f / value;
  }
};

// x / scale, correctly rounded for positive finite scales: the reciprocal is, and two
// corrections by the remainder, which an FMA gives exactly, leave the correctly rounded quotient
// (the first is within an ulp, the second has the exact remainder of it); six operations, a
// division is ten.  A quotient that is clamped or becomes a zero (whose sign the corrections
// would lose), an infinity or a NaN stays as it is: a lifted x that overflows or loses bits is
// one of the first two.
__device__ __forceinline__ float divide(float x, const Scale& scale) {
  x *= scale.lift;
  const float q = x * scale.inverse;
  float r = __builtin_fmaf(__builtin_fmaf(-q, scale.value, x), scale.inverse, q);
  r = __builtin_fmaf(__builtin_fmaf(-r, scale.value, x), scale.inverse, r);
  const float size = fabsf(q);
  return size > 1e-6f && size < 1e6f ? r : q;
}

__device__ __forceinline__ float e4m3_range(float x) {
  const float y = __builtin_amdgcn_fmed3f(x, 448.f, -448.f);
  return x != x ? x : y;
}

// Eight values as e4m3 bytes.
__device__ __forceinline__ u32x2_t pack8_e4m3(const float (&x)[8]) {
  u32x2_t r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[4 * i]), e4m3_range(x[4 * i + 1]),
                                                   0, false);
    r[i] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[4 * i + 2]),
                                                    e4m3_range(x[4 * i + 3]), lo, true));
  }
  return r;
}

__device__ __forceinline__ void unpack8_e4m3(u32x2_t raw, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const floatx2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(raw[i], false);
    const floatx2_t b = __builtin_amdgcn_cvt_pk_f32_fp8(raw[i], true);
    x[4 * i] = a[0], x[4 * i + 1] = a[1], x[4 * i + 2] = b[0], x[4 * i + 3] = b[1];
  }
}

__device__ __forceinline__ u32x2_t to_e4m3(const float (&x)[8], const Scale& scale) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = divide(x[i], scale);
  return pack8_e4m3(y);
}

// (x, y) of a pair rotated; each operation rounded by itself.
__device__ __forceinline__ void rotate(float& x, float& y, float c, float s) {
#pragma clang fp contract(off)
  const float u = x * c - y * s, w = y * c + x * s;
  x = u, y = w;
}

// (cos, sin) of kPairs pairs from `pair` on.
template <int kPairs>
struct Turn {
  floatx4_t cs[kPairs / 2];
  __device__ __forceinline__ Turn(const float* rope, int64_t position, int half, int pair) {
    const floatx4_t* at = reinterpret_cast<const floatx4_t*>(rope + (position * half + pair) * 2);
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) cs[i] = at[i];
  }
  __device__ __forceinline__ float c(int i) const { return cs[i / 2][2 * (i % 2)]; }
  __device__ __forceinline__ float s(int i) const { return cs[i / 2][2 * (i % 2) + 1]; }
};

// Channels d..d+7 of row `row`'s key as the cache will hold them (not divided by a scale's
// effect: the stored value itself).
template <bool kE4m3, bool kInterleaved>
__device__ __forceinline__ void stored8(const AppendArgs& p, const int64_t* positions, int64_t row,
                                        const uint16_t* head, int d, const Scale& scale,
                                        float (&x)[8]) {
  unpack8(load16(head + d), x);
  if (d < 2 * p.half) {
    const int64_t position = positions[row];
    if constexpr (kInterleaved) {
      const Turn<4> turn(p.rope, position, p.half, d / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) rotate(x[2 * i], x[2 * i + 1], turn.c(i), turn.s(i));
    } else {
      const bool first = d < p.half;
      float y[8];
      unpack8(load16(head + (first ? d + p.half : d - p.half)), y);
      const Turn<8> turn(p.rope, position, p.half, first ? d : d - p.half);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a = first ? x[i] : y[i], b = first ? y[i] : x[i];
        rotate(a, b, turn.c(i), turn.s(i));
        x[i] = first ? a : b;
      }
    }
  }
  if constexpr (kE4m3)
    unpack8_e4m3(to_e4m3(x, scale), x);
  else
    unpack8(pack8(x), x);
}

// Smallest and largest per channel over a workgroup's keys, eight channels of a token a
// thread; a NaN key leaves a NaN.
template <int D>
struct Extremes {
  static constexpr int kLanes = D / 8;
  float lo[8], hi[8];
  __device__ __forceinline__ void add(const float (&x)[8], bool first) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = first ? x[e] : __builtin_elementwise_minimum(lo[e], x[e]);
      hi[e] = first ? x[e] : __builtin_elementwise_maximum(hi[e], x[e]);
    }
  }
  template <int M>
  __device__ __forceinline__ void join(int lane) {
    if constexpr (kLanes <= M) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = __builtin_elementwise_minimum(lo[e], xor_lanes<M>(lo[e], lane));
        hi[e] = __builtin_elementwise_maximum(hi[e], xor_lanes<M>(hi[e], lane));
      }
    }
  }
  // Stored values are bf16 or e4m3: bf16 bounds lose no bit.
  __device__ __forceinline__ void write(float (&low)[4][D], float (&high)[4][D], int tid,
                                        uint16_t* out) {
    const int lane = tid & 63, w = tid >> 6;
    join<32>(lane), join<16>(lane), join<8>(lane);
    if (lane < kLanes) {
#pragma unroll
      for (int e = 0; e < 8; ++e) low[w][lane * 8 + e] = lo[e], high[w][lane * 8 + e] = hi[e];
    }
    __syncthreads();
    if (tid < D) {
      float l = low[0][tid], h = high[0][tid];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        l = __builtin_elementwise_minimum(l, low[i][tid]);
        h = __builtin_elementwise_maximum(h, high[i][tid]);
      }
      out[tid] = uint16_t(bf16_bits(l));
      out[D + tid] = uint16_t(bf16_bits(h));
    }
    __syncthreads();
  }
};

// Bounds of the blocks that end among `per` rows from row0 on, for one kv head; source(t, x)
// gives false where token t is to be taken from the cache, else this thread's channels of
// its key.
template <int D, bool kE4m3, typename Begin, typename Source>
__device__ __forceinline__ void bounds_of_rows(const int32_t* __restrict__ slots, int64_t rows,
                                               int64_t num_slots, int64_t row0, int per,
                                               const char* k_cache, uint16_t* bounds, int hkv,
                                               int kvh, Begin begin, Source source) {
  constexpr int kBytes = D * (kE4m3 ? 1 : 2), kLanes = D / 8, kStep = 256 / kLanes;
  __shared__ float low[4][D], high[4][D];
  const int tid = threadIdx.x, lane = tid & 63;
  int32_t slot = lane < per && row0 + lane < rows ? slots[row0 + lane] : -1;
  if (slot >= num_slots) slot = -1;
  uint64_t full = __ballot(slot >= 0 && (slot & 63) == 63);
  while (full) {
    const int at = __builtin_ctzll(full);
    const int64_t block = __builtin_amdgcn_readlane(slot, at) >> 6;
    full &= full - 1;
    begin(block);
    const char* base = k_cache + (block * 64 * hkv + kvh) * kBytes + (tid % kLanes) * (kBytes / kLanes);
    Extremes<D> extremes;
#pragma unroll 4
    for (int i = 0; i < 64 / kStep; ++i) {
      const int t = i * kStep + tid / kLanes;
      float x[8];
      if (!source(t, x)) {
        const char* row = base + int64_t(t) * hkv * kBytes;
        if constexpr (kE4m3)
          unpack8_e4m3(*reinterpret_cast<const u32x2_t*>(row), x);
        else
          unpack8(*reinterpret_cast<const u32x4_t*>(row), x);
      }
      extremes.add(x, i == 0);
    }
    extremes.write(low, high, tid, bounds + (block * hkv + kvh) * 2 * D);
  }
}

// kBounds: the leading workgroups, one for each row and kv head, make the bounds of the block
// that the row ends, if it does.  The others: 16 elements of a head a thread.
template <int D, bool kE4m3, bool kInterleaved, bool kBounds>
__global__ void __launch_bounds__(256)
append_kernel(const int32_t* __restrict__ slots, const int64_t* __restrict__ positions,
              uint32_t rows, uint32_t items_per_row, int64_t num_slots, const AppendArgs p) {
  constexpr int kItems = D / 16;  // of a head
  const uint32_t bound_groups = kBounds ? rows * p.hkv : 0;
  if (kBounds && blockIdx.x < bound_groups) {
    __shared__ int32_t from[64];  // the row that writes a token of the block, or -1
    const int kvh = int(blockIdx.x % p.hkv), tid = threadIdx.x;
    const Scale scale(kE4m3 ? p.k_scale : nullptr, kvh);
    bounds_of_rows<D, kE4m3>(
        slots, rows, num_slots, blockIdx.x / p.hkv, 1, p.k_cache, p.bounds, p.hkv, kvh,
        [&](int64_t block) {
          if (tid < 64) from[tid] = -1;
          __syncthreads();
          for (uint32_t i = tid; i < rows; i += 256) {
            const int32_t slot = slots[i];
            const int64_t pos = p.half ? positions[i] : 0;
            if (slot >= 0 && slot >> 6 == block &&
                (!p.half || (pos >= 0 && pos < p.max_positions)))
              from[slot & 63] = int32_t(i);
          }
          __syncthreads();
        },
        [&](int t, float(&x)[8]) {
          const int64_t r = from[t];
          if (r < 0) return false;
          stored8<kE4m3, kInterleaved>(p, positions, r, p.k + r * p.k_stride + kvh * D,
                                       tid % (D / 8) * 8, scale, x);
          return true;
        });
    return;
  }

  const uint32_t id = (blockIdx.x - bound_groups) * 256 + threadIdx.x;
  const uint32_t row = id / items_per_row;
  if (row >= rows) return;
  const uint32_t item = id - row * items_per_row;
  const int head = int(item / kItems), t = int(item % kItems);
  const bool query = head < p.hq, value = head >= p.hq + p.hkv;
  const int kvh = query ? 0 : value ? head - p.hq - p.hkv : head - p.hq;
  const int64_t slot = query ? 0 : slots[row];
  const int64_t pos = p.half ? positions[row] : 0;
  // The item's two runs of eight elements.
  const int turned = value ? 0 : p.half / 8;
  const bool apart = !kInterleaved && t < turned;
  const int first = apart ? 8 * t : 16 * t, second = apart ? first + p.half : first + 8;
  const uint16_t* src = query   ? p.q + int64_t(row) * p.q_stride + head * D
                        : value ? p.v + int64_t(row) * p.v_stride + kvh * D
                                : p.k + int64_t(row) * p.k_stride + kvh * D;
  const u32x4_t raw_a = load16(src + first), raw_b = load16(src + second);
  if (slot < 0 || slot >= num_slots) return;
  const bool known = !p.half || (pos >= 0 && pos < p.max_positions);
  if (!known && !query) return;  // no such position: nothing is cached, the query is NaN
  float a[8], b[8];
  unpack8(raw_a, a);
  unpack8(raw_b, b);
  if (t < turned) {
    const Turn<8> turn(p.rope, known ? pos : 0, p.half, 8 * t);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& x = kInterleaved ? (i < 4 ? a[2 * i] : b[2 * i - 8]) : a[i];
      float& y = kInterleaved ? (i < 4 ? a[2 * i + 1] : b[2 * i - 7]) : b[i];
      rotate(x, y, turn.c(i), turn.s(i));
      if (!known) x = y = __builtin_nanf("");
    }
  }
  if (query) {
    uint16_t* dst = p.q_out + int64_t(row) * p.q_out_stride + head * D;
    *reinterpret_cast<u32x4_t*>(dst + first) = pack8(a);
    *reinterpret_cast<u32x4_t*>(dst + second) = pack8(b);
    return;
  }
  char* cache = value ? p.v_cache : p.k_cache;
  const int64_t at = (slot * p.hkv + kvh) * D;
  if constexpr (kE4m3) {
    const Scale scale(value ? p.v_scale : p.k_scale, kvh);
    const u32x2_t x = to_e4m3(a, scale), y = to_e4m3(b, scale);
    if (second == first + 8) {
      *reinterpret_cast<u32x4_t*>(cache + at + first) = u32x4_t{x[0], x[1], y[0], y[1]};
    } else {
      *reinterpret_cast<u32x2_t*>(cache + at + first) = x;
      *reinterpret_cast<u32x2_t*>(cache + at + second) = y;
    }
  } else {
    *reinterpret_cast<u32x4_t*>(cache + 2 * (at + first)) = pack8(a);
    *reinterpret_cast<u32x4_t*>(cache + 2 * (at + second)) = pack8(b);
  }
}

// The same from the cache alone.
template <int D, bool kE4m3>
__global__ void __launch_bounds__(256)
block_bounds_kernel(const int32_t* __restrict__ slots, const char* __restrict__ k_cache,
                    uint16_t* __restrict__ bounds, int64_t rows, int64_t num_slots, int per,
                    int hkv) {
  bounds_of_rows<D, kE4m3>(slots, rows, num_slots, int64_t(blockIdx.x) * per, per, k_cache, bounds,
                           hkv, blockIdx.y, [](int64_t) {},
                           [](int, float(&)[8]) { return false; });
}

// A decode step has at most this many rows here.  Each may end a block: a workgroup for each
// row.  Of 64 rows of a prompt one does.
constexpr int64_t kStepRows = 512;
int rows_per_group(int64_t rows) { return rows <= kStepRows ? 1 : 64; }

int launch_bounds(const void* k_cache, int32_t cache_type, int64_t num_slots,
                  const int32_t* slot_mapping, int64_t rows, void* bounds, int32_t num_kv_heads,
                  int32_t head_dim, pd_stream_t stream) {
  const int per = rows_per_group(rows);
  const int64_t groups = (rows + per - 1) / per;
  if (groups > 0x7fffffff || num_kv_heads > 65535)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(groups), unsigned(num_kv_heads)), dim3(256), 0,
                       as_stream(stream), slot_mapping, static_cast<const char*>(k_cache),
                       u16(bounds), rows, num_slots, per, num_kv_heads);
  };
  pd::for_cache(head_dim, cache_type, [&](auto dim, auto e4m3) {
    go(block_bounds_kernel<dim.value, e4m3.value>);
  });
  return launch_status("pd_block_bounds");
}

int check_cache(int32_t cache_type, int64_t num_slots, const void* bounds, int32_t num_kv_heads,
                int32_t head_dim) {
  if (!pd::valid_head_dim(head_dim))
    return pd::fail(PD_EINVAL, "custom decode supports head_dim 64, 128, or 256");
  if (num_kv_heads < 1) return pd::fail(PD_EINVAL, "heads must be positive");
  if (!pd::valid_cache(cache_type)) return pd::fail(PD_EINVAL, "unknown cache type");
  if (num_slots < 1 || num_slots > INT32_MAX + int64_t(1))
    return pd::fail(PD_EINVAL, "the cache must have 1 to 2^31 slots");
  if (bounds && num_slots % pd::kBlock)
    return pd::fail(PD_EINVAL, "bounds need a cache of whole blocks of 64 slots");
  return PD_OK;
}

}  // namespace

extern "C" int pd_append_kv(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                            const void* v, int64_t v_stride, const int64_t* positions,
                            const float* rope, int64_t max_positions, int32_t half,
                            int32_t interleaved, void* q_out, int64_t q_out_stride, void* k_cache,
                            void* v_cache, int32_t cache_type, int64_t num_slots,
                            const int32_t* slot_mapping, const float* k_scale,
                            const float* v_scale, void* bounds, int64_t rows, int32_t num_heads,
                            int32_t num_kv_heads, int32_t head_dim, pd_stream_t stream) {
  pd::clear_error();
  if (rows < 0 || num_heads < 0) return pd::fail(PD_EINVAL, "rows and heads must be non-negative");
  if (const int bad = check_cache(cache_type, num_slots, bounds, num_kv_heads, head_dim)) return bad;
  if (cache_type == PD_CACHE_BF16 && (k_scale || v_scale))
    return pd::fail(PD_EINVAL, "scales belong to an e4m3 cache");
  if (half < 0 || half % 8 || 2 * half > head_dim)
    return pd::fail(PD_EINVAL, "rotated pairs must be a multiple of 8, at most head_dim / 2");
  if (rows == 0) return PD_OK;
  if (!k || !v || !k_cache || !v_cache || !slot_mapping || (num_heads && (!q || !q_out)) ||
      (half && (!positions || !rope || max_positions < 1)))
    return pd::fail(PD_EINVAL, "null tensor pointer");
  const int64_t strides[4] = {q_stride, q_out_stride, k_stride, v_stride};
  const int64_t least[4] = {0, int64_t(num_heads) * head_dim, 0, 0};
  for (int i = 0; i < 4; ++i)
    if (rows > 1 && (i > 1 || num_heads) && (strides[i] % 8 || strides[i] < least[i]))
      return pd::fail(PD_EINVAL, "row strides must be non-negative multiples of 8, of q_out at "
                                 "least a row");
  if (!all_aligned16(q, k, v, rope, q_out, k_cache, v_cache, bounds))
    return pd::fail(PD_EINVAL, "tensors must be 16-byte aligned");
  const int64_t per_row = (num_heads + 2 * int64_t(num_kv_heads)) * (head_dim / 16);
  if (rows >= INT32_MAX / per_row - 256)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  AppendArgs p;
  p.q = u16(q), p.k = u16(k), p.v = u16(v), p.rope = rope, p.q_out = u16(q_out);
  p.k_cache = static_cast<char*>(k_cache), p.v_cache = static_cast<char*>(v_cache);
  p.k_scale = k_scale, p.v_scale = v_scale, p.bounds = u16(bounds);
  p.q_stride = q_stride, p.k_stride = k_stride, p.v_stride = v_stride;
  p.q_out_stride = q_out_stride, p.max_positions = max_positions;
  p.hq = num_heads, p.hkv = num_kv_heads, p.half = half;
  const bool inside = bounds && rows <= kStepRows;
  const int64_t groups =
      (rows * per_row + 255) / 256 + (inside ? rows * int64_t(num_kv_heads) : 0);
  if (groups > 0x7fffffff) return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(groups)), dim3(256), 0, as_stream(stream),
                       slot_mapping, positions, uint32_t(rows), uint32_t(per_row), num_slots, p);
  };
  pd::for_cache(head_dim, cache_type, [&](auto dim, auto e4m3) {
    if (inside)
      go(interleaved ? append_kernel<dim.value, e4m3.value, true, true>
                     : append_kernel<dim.value, e4m3.value, false, true>);
    else
      go(interleaved ? append_kernel<dim.value, e4m3.value, true, false>
                     : append_kernel<dim.value, e4m3.value, false, false>);
  });
  if (const int bad = launch_status("pd_append_kv")) return bad;
  if (!bounds || inside) return PD_OK;
  return launch_bounds(k_cache, cache_type, num_slots, slot_mapping, rows, bounds, num_kv_heads,
                       head_dim, stream);
}

extern "C" int pd_block_bounds(const void* k_cache, int32_t cache_type, int64_t num_slots,
                               const int32_t* slot_mapping, int64_t rows, void* bounds,
                               int32_t num_kv_heads, int32_t head_dim, pd_stream_t stream) {
  pd::clear_error();
  if (rows < 0) return pd::fail(PD_EINVAL, "rows must be non-negative");
  if (const int bad = check_cache(cache_type, num_slots, bounds, num_kv_heads, head_dim)) return bad;
  if (rows == 0) return PD_OK;
  if (!k_cache || !slot_mapping || !bounds || !all_aligned16(k_cache, bounds))
    return pd::fail(PD_EINVAL, "tensors must be present and 16-byte aligned");
  return launch_bounds(k_cache, cache_type, num_slots, slot_mapping, rows, bounds, num_kv_heads,
                       head_dim, stream);
}
