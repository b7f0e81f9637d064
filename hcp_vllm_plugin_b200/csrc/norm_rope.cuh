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
// rotation needs no exchange.  A warp takes one token: its lanes hold the token's
// cos / sin and the weights and go over the token's heads, three rounds of loads in
// flight.  With few tokens a token's rounds are spread over warps.  With the
// 4-bit cache further blocks of the same launch take k and v, 16 tokens of one head
// each, so that whole tiles of the cache are built in shared memory (q4_cache.cuh).
//
// Measured at 16384 tokens of 28/4 heads, D 128, bf16: 54 us (277 MB, 5.1 TB/s, 0.79 of the
// measured copy rate), 62 us with the 16-bit cache, 67 us with the 4-bit one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "q4_cache.cuh"

namespace hcp {

constexpr int kRopeThreads = 128;
constexpr int kRopeBlocks = 8;   // of an SM

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
  int parts;                   // warps of a token
  int rounds;                  // of a warp
  unsigned kv_blocks;          // blocks that take k and v, with the 4-bit cache
};

template <bool F16>
__device__ __forceinline__ void rope_up4(const uint2& v, float* x) {
  const float2 a = q4_up2<F16>(v.x), b = q4_up2<F16>(v.y);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}
template <bool F16>
__device__ __forceinline__ uint2 rope_down4(const float* x) {
  return make_uint2(q4_down2<F16>(x[0], x[1]), q4_down2<F16>(x[2], x[3]));
}

// This lane's dims of a row: a0 .. a0+3 and a1 .. a1+3, partners where it turns them.
struct RopeLane {
  int a0, a1;
  bool turns;
};
template <bool INTER>
__device__ __forceinline__ RopeLane rope_lane(const NormRopeParams& p, int c) {
  RopeLane r;
  const int pairs = p.rotary / 8;  // lanes that rotate
  r.turns = c < pairs;
  r.a0 = !r.turns ? p.rotary + 8 * (c - pairs) : INTER ? 8 * c : 4 * c;
  r.a1 = r.turns && !INTER ? p.rotary / 2 + 4 * c : r.a0 + 4;
  return r;
}
// Cosines and sines of the lane's pairs at a position; 1 and 0 where it turns none.
template <bool F16, bool TAB32>
__device__ __forceinline__ void rope_angles(const NormRopeParams& p, const RopeLane& r, long long pos, int c, float* cs,
                                            float* sn) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (!r.turns || pos < 0 || pos >= p.table_rows) return;
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
// What all rows of a token share that have the same weights.
struct RopeMap {
  float g[8], cs[4], sn[4];
};
template <bool F16>
__device__ __forceinline__ void rope_weights(RopeMap& f, const RopeLane& r, const uint16_t* w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.g[i] = 1.f;
  if (w != nullptr) {
    rope_up4<F16>(*reinterpret_cast<const uint2*>(w + r.a0), f.g);
    rope_up4<F16>(*reinterpret_cast<const uint2*>(w + r.a1), f.g + 4);
  }
}
// Norm and rotation of one row; every lane of the warp takes part.  The products are rounded
// as the formula has them: (x inv) w, then u cos - v sin.  Weights, angles and inv in one map
// would save a third of the multiplications (51 against 54 us at 16384 tokens) and round five
// times as many keys to the other neighbour, each of which may turn a step of the 4-bit cache.
template <int D, bool F16, bool INTER>
__device__ __forceinline__ void rope_row(const RopeLane& r, const RopeMap& f, bool norm, float eps, const uint2 (&in)[2],
                                         uint2 (&out)[2]) {
  float x[8], y[8];
  rope_up4<F16>(in[0], x);
  rope_up4<F16>(in[1], x + 4);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
#pragma unroll
  for (int s = 1; s < D / 8; s <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, s);
  if (norm) {
    const float inv = rsqrtf(fmaf(sq, 1.f / D, eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), f.g[i]);
  }
  if (r.turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = INTER ? 2 * i : i, b = INTER ? 2 * i + 1 : i + 4;
      y[a] = __fsub_rn(__fmul_rn(x[a], f.cs[i]), __fmul_rn(x[b], f.sn[i]));
      y[b] = __fadd_rn(__fmul_rn(x[b], f.cs[i]), __fmul_rn(x[a], f.sn[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  }
  out[0] = rope_down4<F16>(y);
  out[1] = rope_down4<F16>(y + 4);
}

// k and v of 16 tokens of one head: k normed, rotated and written to k_out, both into the cache.
template <int D, bool F16, bool TAB32, bool INTER>
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
  const RopeLane ln = rope_lane<INTER>(p, c);
#pragma unroll 2
  for (int row = threadIdx.x / L::kLanes; row < kQ4TileTokens; row += kRows) {
    const long long tok = t0 + row;
    const bool here = tok >= 0 && tok < p.num_tokens;
    const long long pos = here ? p.positions[tok] : -1;
    uint2 in[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)}, out[2];
    uint4 vraw = make_uint4(0u, 0u, 0u, 0u);
    if (here) {
      const uint16_t* k = p.k + tok * p.k_stride + static_cast<long long>(h) * D;
      in[0] = *reinterpret_cast<const uint2*>(k + ln.a0);
      in[1] = *reinterpret_cast<const uint2*>(k + ln.a1);
      vraw = reinterpret_cast<const uint4*>(p.v + tok * p.v_stride + static_cast<long long>(h) * D)[c];
    }
    RopeMap f;
    rope_angles<F16, TAB32>(p, ln, pos, c, f.cs, f.sn);
    if (pos >= p.table_rows) in[0] = in[1] = make_uint2(0x7fff7fffu, 0x7fff7fffu);  // NaN
    rope_weights<F16>(f, ln, p.k_weight);
    rope_row<D, F16, INTER>(ln, f, p.k_weight != nullptr, p.eps, in, out);
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
    q4_stage_k4<D>(st, row, ln.a0, q4_codes<4, F16>(z, u0 ? s[0] : s[kLast], u0 ? m[0] : m[kLast]));
    q4_stage_k4<D>(st, row, ln.a1, q4_codes<4, F16>(z + 4, u1 ? s[0] : s[kLast], u1 ? m[0] : m[kLast]));
    q4_stage_v8<D>(st, row, c, q4_codes<8, F16>(x, vs, vm));
    if (c < L::kGroups) q4_stage_params<D, F16>(st, row, 0, c, c == 0 ? s[0] : s[kLast], c == 0 ? m[0] : m[kLast]);
    if ((c & 7) == 0) q4_stage_params<D, F16>(st, row, 1, c >> 3, vs, vm);
  }
  __syncthreads();
  q4_flush<D>(st, static_cast<uint8_t*>(p.cache));
}

// Blocks 0 .. kv_blocks - 1 (with the 4-bit cache; the longer ones come first): k and v, 16
// tokens of one head each.  The warps of the blocks after them: `rounds` rounds of one token's
// rows each, 32 / (D/8) rows a round, queries before keys.
template <int D, bool F16, bool TAB32, int CACHE, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  constexpr int kLanes = D / 8;
  constexpr int kWarpRows = 32 / kLanes;         // rows of a round
  constexpr int kAhead = 3;                      // rounds in flight
  ptx::chain_wait();
  ptx::chain_next();
  if constexpr (CACHE == kRopeCacheQ4) {
    __shared__ Q4Stage<D> st;
    if (blockIdx.x < p.kv_blocks) {
      rope_kv_block<D, F16, TAB32, INTER>(p, static_cast<int>(blockIdx.x), st);
      return;
    }
  }
  const int H = p.num_heads, Hkv = p.num_kv_heads;
  const int rows = CACHE == kRopeCacheQ4 ? H : H + Hkv;
  const long long unit = static_cast<long long>(blockIdx.x - p.kv_blocks) * (kRopeThreads / 32) + threadIdx.x / 32;
  const long long tok = p.parts == 1 ? unit : unit / p.parts;
  if (tok >= p.num_tokens) return;
  const int part = p.parts == 1 ? 0 : static_cast<int>(unit - tok * p.parts);
  const int c = threadIdx.x % kLanes, sub = threadIdx.x % 32 / kLanes;
  const RopeLane ln = rope_lane<INTER>(p, c);
  // row r stands at base + r * D, for keys too
  const uint16_t* const qs = p.q + tok * p.q_stride;
  const uint16_t* const ks = p.k + tok * p.k_stride - static_cast<long long>(H) * D;
  const int begin = part * p.rounds * kWarpRows, end = min(rows, begin + p.rounds * kWarpRows);
  uint2 in[kAhead][2], out[2];
  auto load = [&](uint2 (&to)[2], int r) {
    to[0] = to[1] = make_uint2(0u, 0u);
    if (r < end) {
      const uint16_t* src = (r < H ? qs : ks) + r * D;
      to[0] = *reinterpret_cast<const uint2*>(src + ln.a0);
      to[1] = *reinterpret_cast<const uint2*>(src + ln.a1);
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(in[i], begin + i * kWarpRows + sub);  // beside the position
  const long long pos = p.positions[tok];
  if (pos < 0) return;                           // padding row: everything stays
  const bool known = pos < p.table_rows;
  long long dst = -1;                            // cache offset of the token's row of head 0
  if constexpr (CACHE == kRopeCacheSame) {
    long long blk;
    int off;
    if (known && slot_block(p.slot_mapping[tok], p.num_blocks, p.block_size, p.bs_shift, blk, off))
      dst = (blk * Hkv * p.block_size + off) * 2LL * D;
  }
  uint16_t* const qo = p.q_out + tok * p.q_out_stride;
  uint16_t* const ko = p.k_out + tok * p.k_out_stride - static_cast<long long>(H) * D;
  bool keys = begin + sub >= H;                  // rows rise: queries, then keys
  bool norm = (keys ? p.k_weight : p.q_weight) != nullptr;
  RopeMap f;
  rope_angles<F16, TAB32>(p, ln, pos, c, f.cs, f.sn);
  rope_weights<F16>(f, ln, keys ? p.k_weight : p.q_weight);
  for (int r0 = begin; r0 < end; r0 += kAhead * kWarpRows) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = r0 + i * kWarpRows + sub;
      if (r0 + i * kWarpRows >= end) break;      // the same for all lanes
      if (CACHE != kRopeCacheQ4 && !keys && r >= H) {
        keys = true;
        norm = p.k_weight != nullptr;
        rope_weights<F16>(f, ln, p.k_weight);
      }
      if (!known) in[i][0] = in[i][1] = make_uint2(0x7fff7fffu, 0x7fff7fffu);  // NaN
      rope_row<D, F16, INTER>(ln, f, norm, p.eps, in[i], out);
      load(in[i], r + kAhead * kWarpRows);
      if (r >= end) continue;
      uint16_t* to = (r < H ? qo : ko) + r * D;
      *reinterpret_cast<uint2*>(to + ln.a0) = out[0];
      *reinterpret_cast<uint2*>(to + ln.a1) = out[1];
      if constexpr (CACHE == kRopeCacheSame) {
        if (r >= H && dst >= 0) {
          uint16_t* at = static_cast<uint16_t*>(p.cache) + dst + static_cast<long long>(r - H) * p.block_size * 2 * D;
          *reinterpret_cast<uint2*>(at + ln.a0) = out[0];
          *reinterpret_cast<uint2*>(at + ln.a1) = out[1];
          reinterpret_cast<uint4*>(at + D)[c] = reinterpret_cast<const uint4*>(p.v + tok * p.v_stride + (r - H) * D)[c];
        }
      }
    }
  }
}

}  // namespace hcp
