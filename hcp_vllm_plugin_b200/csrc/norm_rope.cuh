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
// token's cos / sin once and go over the token's heads, two rows' loads in flight.
// With few tokens the heads are spread over blocks instead, one round each.  With the
// 4-bit cache further blocks of the same launch take k and v, 16 tokens of one head
// each, so that whole tiles of the cache are built in shared memory (q4_cache.cuh).
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
  long long num_tokens;
  int spread;                  // blocks of a token
  unsigned kv_blocks;          // blocks that take k and v, with the 4-bit cache
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

// This lane's dims of a row: a0 .. a0+3 and a1 .. a1+3, partners where it turns them.
struct RopeLane {
  int a0, a1;
  bool turns;
};
__device__ __forceinline__ RopeLane rope_lane(const NormRopeParams& p, int c) {
  RopeLane r;
  const int pairs = p.rotary / 8;  // lanes that rotate
  r.turns = c < pairs;
  r.a0 = !r.turns ? p.rotary + 8 * (c - pairs) : p.interleaved ? 8 * c : 4 * c;
  r.a1 = r.turns && !p.interleaved ? p.rotary / 2 + 4 * c : r.a0 + 4;
  return r;
}
template <bool F16, bool TAB32>
__device__ __forceinline__ void rope_angles(const NormRopeParams& p, long long pos, int c, float* cs, float* sn) {
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
// Norm and rotation of one row; every lane of the warp takes part.
template <int D, bool F16>
__device__ __forceinline__ void rope_row(const NormRopeParams& p, const RopeLane& r, const uint16_t* w, bool known,
                                         const float* cs, const float* sn, const uint2 (&in)[2], uint2 (&out)[2]) {
  float x[8];
  rope_up4<F16>(in[0], x);
  rope_up4<F16>(in[1], x + 4);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
#pragma unroll
  for (int s = 1; s < D / 8; s <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, s);
  if (w != nullptr) {
    const float inv = rsqrtf(sq * (1.f / D) + p.eps);
    float g[8];
    rope_up4<F16>(*reinterpret_cast<const uint2*>(w + r.a0), g);
    rope_up4<F16>(*reinterpret_cast<const uint2*>(w + r.a1), g + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
  }
  float y[8];
  if (!r.turns) {
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
  if (!known) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7fffffff);
  }
  out[0] = rope_down4<F16>(y);
  out[1] = rope_down4<F16>(y + 4);
}

// k and v of 16 tokens of one head: k normed, rotated and written to k_out, both into the cache.
template <int D, bool F16, bool TAB32>
__device__ __forceinline__ void rope_kv_block(const NormRopeParams& p, int unit, Q4Stage<D>& st) {
  using L = Q4<D>;
  constexpr int kRows = kRopeThreads / L::kLanes;
  const int h = unit % p.num_kv_heads;
  long long t0;
  long long slot = q4_run_slots(p.slot_mapping, p.num_tokens, unit / p.num_kv_heads, t0);
  if (t0 >= p.num_tokens) return;
  if (threadIdx.x < 32) {
    Q4UpdateParams u;
    u.num_blocks = p.num_blocks;
    u.block_size = p.block_size;
    u.bs_shift = p.bs_shift;
    u.num_kv_heads = p.num_kv_heads;
    if (slot >= 0) {
      const long long pos = p.positions[t0 + threadIdx.x];
      if (pos < 0 || pos >= p.table_rows) slot = -1;
    }
    q4_place<D>(st, u, slot, h);
  }
  const int c = threadIdx.x % L::kLanes;
  const RopeLane ln = rope_lane(p, c);
#pragma unroll 2
  for (int row = threadIdx.x / L::kLanes; row < kQ4TileTokens; row += kRows) {
    const long long tok = t0 + row;
    const bool here = tok >= 0 && tok < p.num_tokens;
    const long long pos = here ? p.positions[tok] : -1;
    const bool known = pos < p.table_rows;
    uint2 in[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)}, out[2];
    uint4 vraw = make_uint4(0u, 0u, 0u, 0u);
    float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (here) {
      const uint16_t* k = p.k + tok * p.k_stride + static_cast<long long>(h) * D;
      in[0] = *reinterpret_cast<const uint2*>(k + ln.a0);
      in[1] = *reinterpret_cast<const uint2*>(k + ln.a1);
      vraw = reinterpret_cast<const uint4*>(p.v + tok * p.v_stride + static_cast<long long>(h) * D)[c];
    }
    if (ln.turns && known && pos >= 0) rope_angles<F16, TAB32>(p, pos, c, cs, sn);
    rope_row<D, F16>(p, ln, p.k_weight, known, cs, sn, in, out);
    if (pos >= 0) {
      uint16_t* k = p.k_out + tok * p.k_out_stride + static_cast<long long>(h) * D;
      *reinterpret_cast<uint2*>(k + ln.a0) = out[0];
      *reinterpret_cast<uint2*>(k + ln.a1) = out[1];
    }
    float z[8], x[8];  // the rounded key, the value
    rope_up4<F16>(out[0], z);
    rope_up4<F16>(out[1], z + 4);
    q4_unpack8<F16>(vraw, x);
    // K: ranges of both groups over the row's lanes (a lane may hold dims of both); V: of the lane's group
    constexpr uint32_t kInf = q4_inf2<F16>(), kNegInf = kInf | 0x80008000u;
    uint32_t lo[L::kGroups], hi[L::kGroups];
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) {
      const bool i0 = (ln.a0 >> 6) == g, i1 = (ln.a1 >> 6) == g;
      lo[g] = q4_min2<F16>(i0 ? q4_min2<F16>(out[0].x, out[0].y) : kInf, i1 ? q4_min2<F16>(out[1].x, out[1].y) : kInf);
      hi[g] = q4_max2<F16>(i0 ? q4_max2<F16>(out[0].x, out[0].y) : kNegInf, i1 ? q4_max2<F16>(out[1].x, out[1].y) : kNegInf);
    }
    uint32_t vlo = q4_min2<F16>(q4_min2<F16>(vraw.x, vraw.y), q4_min2<F16>(vraw.z, vraw.w));
    uint32_t vhi = q4_max2<F16>(q4_max2<F16>(vraw.x, vraw.y), q4_max2<F16>(vraw.z, vraw.w));
#pragma unroll
    for (int s = 1; s < L::kLanes; s <<= 1) {
#pragma unroll
      for (int g = 0; g < L::kGroups; ++g) {
        lo[g] = q4_min2<F16>(lo[g], __shfl_xor_sync(0xffffffffu, lo[g], s));
        hi[g] = q4_max2<F16>(hi[g], __shfl_xor_sync(0xffffffffu, hi[g], s));
      }
      if (s < 8) {
        vlo = q4_min2<F16>(vlo, __shfl_xor_sync(0xffffffffu, vlo, s));
        vhi = q4_max2<F16>(vhi, __shfl_xor_sync(0xffffffffu, vhi, s));
      }
    }
    float s[L::kGroups], m[L::kGroups], vs, vm;
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) q4_params<F16>(lo[g], hi[g], s[g], m[g]);
    q4_params<F16>(vlo, vhi, vs, vm);
    constexpr int kLast = L::kGroups - 1;
    const bool u0 = ln.a0 < 64, u1 = ln.a1 < 64;
    q4_stage_k4<D>(st, row, ln.a0, q4_codes<4>(z, u0 ? s[0] : s[kLast], u0 ? m[0] : m[kLast]));
    q4_stage_k4<D>(st, row, ln.a1, q4_codes<4>(z + 4, u1 ? s[0] : s[kLast], u1 ? m[0] : m[kLast]));
    q4_stage_v8<D>(st, row, c, q4_codes<8>(x, vs, vm));
    if (c < L::kGroups) q4_stage_params<D, F16>(st, row, 0, c, c == 0 ? s[0] : s[kLast], c == 0 ? m[0] : m[kLast]);
    if ((c & 7) == 0) q4_stage_params<D, F16>(st, row, 1, c >> 3, vs, vm);
  }
  __syncthreads();
  q4_flush<D>(st, static_cast<uint8_t*>(p.cache));
}

// Blocks 0 .. kv_blocks - 1 (with the 4-bit cache; the longer ones come first): k and v, 16
// tokens of one head each.  The blocks after them: rows of one token each.
template <int D, bool F16, bool TAB32, int CACHE>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const NormRopeParams p) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kRopeThreads / kLanes;   // rows of a round
  const int H = p.num_heads, Hkv = p.num_kv_heads;
  if constexpr (CACHE == kRopeCacheQ4) {
    __shared__ Q4Stage<D> st;
    if (blockIdx.x < p.kv_blocks) {
      rope_kv_block<D, F16, TAB32>(p, static_cast<int>(blockIdx.x), st);
      return;
    }
  }
  const unsigned bid = blockIdx.x - p.kv_blocks;
  const unsigned tok32 = p.spread == 1 ? bid : bid / p.spread;
  const int part = p.spread == 1 ? 0 : bid - tok32 * p.spread;
  const long long tok = tok32;
  const int c = threadIdx.x % kLanes;
  const RopeLane ln = rope_lane(p, c);
  const int rows = CACHE == kRopeCacheQ4 ? H : H + Hkv;
  constexpr int U = 2;
  uint2 in[U][2], out[2];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * p.spread * kRows + threadIdx.x / kLanes;
      in[u][0] = in[u][1] = make_uint2(0u, 0u);
      if (r < rows) {
        const uint16_t* row = r < H ? p.q + tok * p.q_stride + static_cast<long long>(r) * D
                                    : p.k + tok * p.k_stride + static_cast<long long>(r - H) * D;
        in[u][0] = *reinterpret_cast<const uint2*>(row + ln.a0);
        in[u][1] = *reinterpret_cast<const uint2*>(row + ln.a1);
      }
    }
  };
  load(part * kRows);                            // beside the position
  const long long pos = p.positions[tok];
  if (pos < 0) return;                           // padding row: everything stays
  const bool known = pos < p.table_rows;
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (ln.turns && known) rope_angles<F16, TAB32>(p, pos, c, cs, sn);
  long long dst = -1;                            // cache offset of the token's row of head 0
  if constexpr (CACHE == kRopeCacheSame) {
    long long blk;
    int off;
    if (known && slot_block(p.slot_mapping[tok], p.num_blocks, p.block_size, p.bs_shift, blk, off))
      dst = (blk * Hkv * p.block_size + off) * 2LL * D;
  }
  for (int r0 = part * kRows; r0 < rows; r0 += p.spread * kRows * U) {
    if (r0 != part * kRows) load(r0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * p.spread * kRows + threadIdx.x / kLanes;
      if (r0 + u * p.spread * kRows >= rows) break;  // the same for all
      rope_row<D, F16>(p, ln, r < H ? p.q_weight : p.k_weight, known, cs, sn, in[u], out);
      if (r >= rows) continue;
      uint16_t* row = r < H ? p.q_out + tok * p.q_out_stride + static_cast<long long>(r) * D
                            : p.k_out + tok * p.k_out_stride + static_cast<long long>(r - H) * D;
      *reinterpret_cast<uint2*>(row + ln.a0) = out[0];
      *reinterpret_cast<uint2*>(row + ln.a1) = out[1];
      if constexpr (CACHE == kRopeCacheSame) {
        if (r >= H && dst >= 0) {
          uint16_t* to = static_cast<uint16_t*>(p.cache) + dst + static_cast<long long>(r - H) * p.block_size * 2 * D;
          *reinterpret_cast<uint2*>(to + ln.a0) = out[0];
          *reinterpret_cast<uint2*>(to + ln.a1) = out[1];
        }
      }
    }
  }
  if constexpr (CACHE == kRopeCacheSame) {
    if (dst >= 0)
      for (int h = part * kRows + threadIdx.x / kLanes; h < Hkv; h += p.spread * kRows) {
        const uint4 v = reinterpret_cast<const uint4*>(p.v + tok * p.v_stride + static_cast<long long>(h) * D)[c];
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.cache) + dst + static_cast<long long>(h) * p.block_size * 2 * D + D)[c] = v;
      }
  }
}

}  // namespace hcp
