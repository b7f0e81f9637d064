// Per-head RMS norm of queries and keys, their position rotation, and the write
// of keys and values into the paged cache, in one pass.
//
//   y = x * rsqrt(mean_d x_d^2 + eps) * w_d          (w given)
//   (a, b) -> (a cos - b sin, b cos + a sin)         for the rotary / 2 pairs,
//     pair i = dims (i, i + rotary/2), or neighbours (2i, 2i+1) when interleaved;
//     cos, sin = table[position, i], table[position, rotary/2 + i]
// The other dims keep y.  Everything is held in 32 bits and rounded once to the
// rows' type; the cache gets that rounded value.
//
// Bound by HBM: 2 bytes read and 2 written per element.  D/8 lanes own a row and
// each lane holds both members of its pairs (4 dims and their 4 partners), so the
// rotation needs no exchange.  A block works on one token: its lanes load the
// weights and the token's cos / sin once and go over the token's heads, all loads
// of a round in flight before the first is used.  With few tokens the heads are
// spread over blocks instead (gridDim.y), one round each.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "q4_cache.cuh"

namespace hcp {

constexpr int kRopeThreads = 128;

enum : int { kRopeCacheNone = 0, kRopeCacheSame = 1, kRopeCacheQ4 = 2 };

struct NormRopeParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;           // with a cache
  uint16_t* q_out;
  uint16_t* k_out;
  long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements
  const int64_t* positions;
  const void* table;           // [table_rows, rotary]
  long long table_stride;      // elements
  long long table_rows;
  const uint16_t* q_weight;    // may be null
  const uint16_t* k_weight;
  const int64_t* slot_mapping;
  void* cache;
  long long num_blocks;
  float eps;
  int num_heads;
  int num_kv_heads;
  int rotary;
  int interleaved;
  int block_size;
  int bs_shift;
};

template <bool F16>
__device__ __forceinline__ void rope_up4(const uint2& v, float* x) {
  x[0] = q4_up<F16>(v.x & 0xffffu);
  x[1] = q4_up<F16>(v.x >> 16);
  x[2] = q4_up<F16>(v.y & 0xffffu);
  x[3] = q4_up<F16>(v.y >> 16);
}
template <bool F16>
__device__ __forceinline__ uint2 rope_down4(const float* x) {
  return make_uint2(q4_down<F16>(x[0]) | (q4_down<F16>(x[1]) << 16), q4_down<F16>(x[2]) | (q4_down<F16>(x[3]) << 16));
}

// 4 dims starting at d (a multiple of 4) of a token's K row.
template <int D>
__device__ __forceinline__ void q4_store_k4(uint8_t* tile, int j, int d, const float* x, float s, float m) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= q4_code(x[i], s, m) << (4 * i);
  *reinterpret_cast<uint16_t*>(tile + j * (D / 2) + Q4<D>::k_word(d >> 3) + ((d >> 2) & 1) * 2) =
      static_cast<uint16_t>(w);
}

template <int D, bool F16, bool TAB32, int CACHE>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const NormRopeParams p) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kRopeThreads / kLanes;   // rows of a round
  const long long tok = blockIdx.x;
  const int c = threadIdx.x % kLanes;
  const int H = p.num_heads, Hkv = p.num_kv_heads;
  const int rows = H + Hkv + (CACHE != kRopeCacheNone ? Hkv : 0);
  const long long pos = p.positions[tok];
  if (pos < 0) return;                           // padding row: everything stays
  const bool known = pos < p.table_rows;

  // this lane's dims: a0..a0+3 and a1..a1+3
  const int pairs = p.rotary / 8;                // lanes that rotate
  const bool turns = c < pairs;
  int a0, a1;
  if (!turns) {
    a0 = p.rotary + 8 * (c - pairs);
    a1 = a0 + 4;
  } else if (p.interleaved) {
    a0 = 8 * c;
    a1 = a0 + 4;
  } else {
    a0 = 4 * c;
    a1 = p.rotary / 2 + 4 * c;
  }
  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (turns && known) {
    const long long at = pos * p.table_stride + 4 * c;
    if constexpr (TAB32) {
      const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p.table) + at);
      const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p.table) + at + p.rotary / 2);
      cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w;
      sn[0] = b.x; sn[1] = b.y; sn[2] = b.z; sn[3] = b.w;
    } else {
      rope_up4<F16>(*reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.table) + at), cs);
      rope_up4<F16>(*reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.table) + at + p.rotary / 2), sn);
    }
  }
  long long blk = 0;
  int off = 0;
  bool slot = false;
  if constexpr (CACHE != kRopeCacheNone)
    slot = known && slot_block(p.slot_mapping[tok], p.num_blocks, p.block_size, p.bs_shift, blk, off);

  for (int r0 = blockIdx.y * kRows; r0 < rows; r0 += gridDim.y * kRows) {
    const int r = r0 + threadIdx.x / kLanes;
    const bool is_q = r < H, is_v = r >= H + Hkv, have = r < rows;
    const int h = is_q ? r : is_v ? r - H - Hkv : r - H;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (have) {
      if (is_v) {
        q4_unpack8<F16>(reinterpret_cast<const uint4*>(p.v + tok * p.v_stride + static_cast<long long>(h) * D)[c], x);
      } else {
        const uint16_t* row = (is_q ? p.q + tok * p.q_stride : p.k + tok * p.k_stride) + static_cast<long long>(h) * D;
        rope_up4<F16>(*reinterpret_cast<const uint2*>(row + a0), x);
        rope_up4<F16>(*reinterpret_cast<const uint2*>(row + a1), x + 4);
      }
    }
    const uint16_t* w = is_q ? p.q_weight : p.k_weight;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
#pragma unroll
    for (int s = 1; s < kLanes; s <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, s);
    uint2 y0, y1;
    if (!is_v) {
      if (w != nullptr) {
        const float inv = rsqrtf(sq * (1.f / D) + p.eps);
        float g[8];
        rope_up4<F16>(*reinterpret_cast<const uint2*>(w + a0), g);
        rope_up4<F16>(*reinterpret_cast<const uint2*>(w + a1), g + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
      }
      float y[8];
      if (!turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
      } else if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
          y[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = x[i] * cs[i] - x[i + 4] * sn[i];
          y[i + 4] = x[i + 4] * cs[i] + x[i] * sn[i];
        }
      }
      if (!known)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7fffffff);
      y0 = rope_down4<F16>(y);
      y1 = rope_down4<F16>(y + 4);
      if (have) {
        uint16_t* o = (is_q ? p.q_out + tok * p.q_out_stride : p.k_out + tok * p.k_out_stride) +
                      static_cast<long long>(h) * D;
        *reinterpret_cast<uint2*>(o + a0) = y0;
        *reinterpret_cast<uint2*>(o + a1) = y1;
      }
    }
    if constexpr (CACHE == kRopeCacheSame) {
      if (have && slot && !is_q) {
        uint16_t* dst = static_cast<uint16_t*>(p.cache) + ((blk * Hkv + h) * p.block_size + off) * 2LL * D;
        if (is_v) {
          reinterpret_cast<uint4*>(dst + D)[c] = q4_pack8<F16>(x);
        } else {
          *reinterpret_cast<uint2*>(dst + a0) = y0;
          *reinterpret_cast<uint2*>(dst + a1) = y1;
        }
      }
    }
    if constexpr (CACHE == kRopeCacheQ4) {
      // ranges of both groups over the row's lanes (every lane takes part)
      float z[8];
      const int d0 = is_v ? 8 * c : a0, d1 = is_v ? 8 * c + 4 : a1;
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = x[i];
      } else {
        rope_up4<F16>(y0, z);
        rope_up4<F16>(y1, z + 4);
      }
      float s[Q4<D>::kGroups], m[Q4<D>::kGroups];
#pragma unroll
      for (int g = 0; g < Q4<D>::kGroups; ++g) {
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((d0 >> 6) == g) q4_range(z[i], lo, hi);
          if ((d1 >> 6) == g) q4_range(z[4 + i], lo, hi);
        }
#pragma unroll
        for (int t = 1; t < kLanes; t <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, t));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, t));
        }
        q4_params<F16>(lo, hi, s[g], m[g]);
      }
      if (have && slot && !is_q) {
        uint8_t* tile = static_cast<uint8_t*>(p.cache) + q4_tile<D>(blk, h, Hkv, p.block_size, off);
        const int j = off % kQ4TileTokens;
        const int g0 = Q4<D>::kGroups == 1 ? 0 : d0 >> 6, g1 = Q4<D>::kGroups == 1 ? 0 : d1 >> 6;
        const float s0 = g0 == 0 ? s[0] : s[Q4<D>::kGroups - 1], m0 = g0 == 0 ? m[0] : m[Q4<D>::kGroups - 1];
        const float s1 = g1 == 0 ? s[0] : s[Q4<D>::kGroups - 1], m1 = g1 == 0 ? m[0] : m[Q4<D>::kGroups - 1];
        if (is_v) {
          q4_store_v<D, F16>(tile, j, c, z, s0, m0);
        } else {
          q4_store_k4<D>(tile, j, d0, z, s0, m0);
          q4_store_k4<D>(tile, j, d1, z + 4, s1, m1);
        }
        if (c < Q4<D>::kGroups) {
          const float sp = c == 0 ? s[0] : s[Q4<D>::kGroups - 1], mp = c == 0 ? m[0] : m[Q4<D>::kGroups - 1];
          q4_store_params<D, F16>(tile, j, is_v ? 1 : 0, c, sp, mp);
        }
      }
    }
  }
}

}  // namespace hcp
