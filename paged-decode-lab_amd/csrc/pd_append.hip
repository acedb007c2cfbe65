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
  const int64_t* positions;
  const float* rope;
  uint16_t* q_out;
  char *k_cache, *v_cache;
  const int32_t* slots;
  const float *k_scale, *v_scale;
  int64_t q_stride, k_stride, v_stride, q_out_stride, max_positions, num_slots;
  uint32_t rows, items_per_row;
  int hq, hkv, half;
};

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

// x of eight elements to element `at` of a cache.
template <bool kE4m3>
__device__ __forceinline__ void store_cache8(char* cache, int64_t at, float (&x)[8], float scale) {
  if constexpr (kE4m3) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] / scale;
    *reinterpret_cast<u32x2_t*>(cache + at) = pack8_e4m3(x);
  } else {
    *reinterpret_cast<u32x4_t*>(cache + 2 * at) = pack8(x);
  }
}

template <int D, bool kE4m3, bool kInterleaved>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs p) {
#pragma clang fp contract(off)
  constexpr int kItems = D / 16;  // of a head
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = id / p.items_per_row;
  if (row >= p.rows) return;
  const uint32_t item = id - row * p.items_per_row;
  const int head = int(item / kItems), t = int(item % kItems);
  const bool query = head < p.hq, value = head >= p.hq + p.hkv;
  const int kvh = query ? 0 : value ? head - p.hq - p.hkv : head - p.hq;

  int64_t slot = 0;
  if (!query) {
    slot = p.slots[row];
    if (slot < 0 || slot >= p.num_slots) return;
  }
  // The item's two runs of eight elements.
  const int turned = value ? 0 : p.half / 8;
  int first, second;
  if (t < turned) {
    first = kInterleaved ? 16 * t : 8 * t;
    second = kInterleaved ? first + 8 : first + p.half;
  } else {
    first = 16 * t;
    second = first + 8;
  }
  const uint16_t* src = query   ? p.q + int64_t(row) * p.q_stride + head * D
                        : value ? p.v + int64_t(row) * p.v_stride + kvh * D
                                : p.k + int64_t(row) * p.k_stride + kvh * D;
  const u32x4_t raw_a = load16(src + first), raw_b = load16(src + second);
  float a[8], b[8];
  unpack8(raw_a, a);
  unpack8(raw_b, b);
  if (t < turned) {
    const int64_t pos = p.positions[row];
    if (pos < 0 || pos >= p.max_positions) {
      if (!query) return;  // no such position: nothing is cached, the query is NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = __builtin_nanf("");
    } else {
      floatx4_t turn[4];  // (cos, sin) of eight pairs
      const floatx4_t* table =
          reinterpret_cast<const floatx4_t*>(p.rope + (pos * p.half + 8 * t) * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) turn[i] = table[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = turn[i / 2][2 * (i % 2)], s = turn[i / 2][2 * (i % 2) + 1];
        float& x = kInterleaved ? (i < 4 ? a[2 * i] : b[2 * i - 8]) : a[i];
        float& y = kInterleaved ? (i < 4 ? a[2 * i + 1] : b[2 * i - 7]) : b[i];
        const float u = x * c - y * s, w = y * c + x * s;
        x = u, y = w;
      }
    }
  } else if (!query && p.half) {
    const int64_t pos = p.positions[row];
    if (pos < 0 || pos >= p.max_positions) return;
  }
  if (query) {
    uint16_t* dst = p.q_out + int64_t(row) * p.q_out_stride + head * D;
    *reinterpret_cast<u32x4_t*>(dst + first) = pack8(a);
    *reinterpret_cast<u32x4_t*>(dst + second) = pack8(b);
    return;
  }
  const float* scales = value ? p.v_scale : p.k_scale;
  const float scale = kE4m3 && scales ? scales[kvh] : 1.f;
  char* cache = value ? p.v_cache : p.k_cache;
  const int64_t at = (slot * p.hkv + kvh) * D;
  store_cache8<kE4m3>(cache, at + first, a, scale);
  store_cache8<kE4m3>(cache, at + second, b, scale);
}

// Smallest and largest stored key per channel of the blocks of 64 slots whose
// last slot is among `slots`.  A workgroup looks at 16 rows for one kv head; a
// token is kLanes threads of 16 bytes.  A NaN key leaves a NaN.
template <int D, bool kE4m3>
__global__ void __launch_bounds__(256)
block_bounds_kernel(const char* __restrict__ k_cache, const int32_t* __restrict__ slots,
                    int64_t rows, int64_t num_slots, uint16_t* __restrict__ bounds, int hkv) {
  constexpr int kBytes = D * (kE4m3 ? 1 : 2), kLanes = kBytes / 16, kStep = 256 / kLanes;
  constexpr int E = D / kLanes;  // elements of 16 bytes
  __shared__ float low[4][D], high[4][D];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = int64_t(blockIdx.x) * 16 + (lane & 15);
  const int kvh = blockIdx.y;
  int32_t slot = row < rows ? slots[row] : -1;
  if (slot >= num_slots) slot = -1;
  uint64_t full = __ballot(lane < 16 && slot >= 0 && (slot & 63) == 63);
  while (full) {
    const int64_t block = __builtin_amdgcn_readlane(slot, __builtin_ctzll(full)) >> 6;
    full &= full - 1;
    const char* base = k_cache + (block * 64 * hkv + kvh) * kBytes + (tid % kLanes) * 16;
    float lo[E], hi[E];
    u32x4_t raw[64 / kStep];
#pragma unroll
    for (int i = 0; i < 64 / kStep; ++i)
      raw[i] = *reinterpret_cast<const u32x4_t*>(
          base + int64_t(i * kStep + tid / kLanes) * hkv * kBytes);
#pragma unroll
    for (int i = 0; i < 64 / kStep; ++i)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float x, y;
        if constexpr (kE4m3) {
          const floatx2_t f = (e & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8(raw[i][e / 4], true)
                                      : __builtin_amdgcn_cvt_pk_f32_fp8(raw[i][e / 4], false);
          x = f[0], y = f[1];
        } else {
          x = bf16_lo(raw[i][e / 2]), y = bf16_hi(raw[i][e / 2]);
        }
        lo[e] = i ? __builtin_elementwise_minimum(lo[e], x) : x;
        hi[e] = i ? __builtin_elementwise_maximum(hi[e], x) : x;
        lo[e + 1] = i ? __builtin_elementwise_minimum(lo[e + 1], y) : y;
        hi[e + 1] = i ? __builtin_elementwise_maximum(hi[e + 1], y) : y;
      }
#pragma unroll
    for (int e = 0; e < E; ++e) {
#define PD_JOIN(M)                                                                    \
  if constexpr (kLanes <= M) {                                                        \
    lo[e] = __builtin_elementwise_minimum(lo[e], xor_lanes<M>(lo[e], lane));          \
    hi[e] = __builtin_elementwise_maximum(hi[e], xor_lanes<M>(hi[e], lane));          \
  }
      PD_JOIN(32) PD_JOIN(16) PD_JOIN(8) PD_JOIN(4)
#undef PD_JOIN
      if (lane < kLanes) {
        low[w][lane * E + e] = lo[e];
        high[w][lane * E + e] = hi[e];
      }
    }
    __syncthreads();
    for (int d = tid; d < D; d += 256) {
      float l = low[0][d], h = high[0][d];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        l = __builtin_elementwise_minimum(l, low[i][d]);
        h = __builtin_elementwise_maximum(h, high[i][d]);
      }
      // Stored values are bf16 or e4m3: no bit is lost.
      uint16_t* out = bounds + (block * hkv + kvh) * 2 * D + d;
      out[0] = uint16_t(bf16_bits(l));
      out[D] = uint16_t(bf16_bits(h));
    }
    __syncthreads();
  }
}

int launch_bounds(const void* k_cache, int32_t cache_type, int64_t num_slots,
                  const int32_t* slot_mapping, int64_t rows, void* bounds, int32_t num_kv_heads,
                  int32_t head_dim, pd_stream_t stream) {
  const int64_t groups = (rows + 15) / 16;
  if (groups > 0x7fffffff || num_kv_heads > 65535)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(groups), unsigned(num_kv_heads)), dim3(256), 0,
                       as_stream(stream), static_cast<const char*>(k_cache), slot_mapping, rows,
                       num_slots, u16(bounds), num_kv_heads);
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
  if (half < 0 || half % 8 || 2 * half > head_dim)
    return pd::fail(PD_EINVAL, "rotated pairs must be a multiple of 8, at most head_dim / 2");
  if (rows == 0) return PD_OK;
  if (!k || !v || !k_cache || !v_cache || !slot_mapping || (num_heads && (!q || !q_out)) ||
      (half && (!positions || !rope || max_positions < 1)))
    return pd::fail(PD_EINVAL, "null tensor pointer");
  const int64_t strides[4] = {q_stride, q_out_stride, k_stride, v_stride};
  const int64_t least[4] = {0, int64_t(num_heads) * head_dim, 0, 0};
  for (int i = 0; i < 4; ++i)
    if ((i > 1 || num_heads) && (strides[i] % 8 || strides[i] < least[i]))
      return pd::fail(PD_EINVAL, "row strides must be non-negative multiples of 8, of q_out at "
                                 "least a row");
  if (!all_aligned16(q, k, v, rope, q_out, k_cache, v_cache, bounds))
    return pd::fail(PD_EINVAL, "tensors must be 16-byte aligned");
  const int64_t per_row = (num_heads + 2 * int64_t(num_kv_heads)) * (head_dim / 16);
  if (rows >= INT32_MAX / per_row - 256)
    return pd::fail(PD_EINVAL, "grid dimension exceeds device limits");
  AppendArgs p;
  p.q = u16(q), p.k = u16(k), p.v = u16(v), p.positions = positions, p.rope = rope;
  p.q_out = u16(q_out);
  p.k_cache = static_cast<char*>(k_cache), p.v_cache = static_cast<char*>(v_cache);
  p.slots = slot_mapping, p.k_scale = k_scale, p.v_scale = v_scale;
  p.q_stride = q_stride, p.k_stride = k_stride, p.v_stride = v_stride;
  p.q_out_stride = q_out_stride, p.max_positions = max_positions, p.num_slots = num_slots;
  p.rows = uint32_t(rows), p.items_per_row = uint32_t(per_row);
  p.hq = num_heads, p.hkv = num_kv_heads, p.half = half;
  const dim3 grid(unsigned((rows * per_row + 255) / 256));
  pd::for_cache(head_dim, cache_type, [&](auto dim, auto e4m3) {
    const auto kernel = interleaved ? append_kernel<dim.value, e4m3.value, true>
                                    : append_kernel<dim.value, e4m3.value, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), p);
  });
  if (const int bad = launch_status("pd_append_kv")) return bad;
  if (!bounds) return PD_OK;
  return launch_bounds(k_cache, cache_type, num_slots, slot_mapping, rows, bounds, num_kv_heads,
                       head_dim, stream);
}

extern "C" int pd_block_bounds(const void* k_cache, int32_t cache_type, int64_t num_slots,
                               const int32_t* slot_mapping, int64_t rows, void* bounds,
                               int32_t num_kv_heads, int32_t head_dim, pd_stream_t stream) {
  pd::clear_error();
  if (rows < 0) return pd::fail(PD_EINVAL, "rows must be non-negative");
  if (!k_cache || !slot_mapping || !bounds || !all_aligned16(k_cache, bounds))
    return pd::fail(PD_EINVAL, "tensors must be present and 16-byte aligned");
  if (const int bad = check_cache(cache_type, num_slots, bounds, num_kv_heads, head_dim)) return bad;
  if (rows == 0) return PD_OK;
  return launch_bounds(k_cache, cache_type, num_slots, slot_mapping, rows, bounds, num_kv_heads,
                       head_dim, stream);
}
