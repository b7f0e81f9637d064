// The 4-bit paged KV cache: its format, the scatter of new rows into it and the
// gather of rows out of it.
//
// A group is 64 dims of one token, KV head and side (K or V).  With lo and hi
// its smallest and largest element:
//   s = round16((hi - lo) / 15),  n_d = round((x_d - lo) / s) clamped to 0..15,
//   x'_d = lo + s n_d
// where round16 rounds to the rows' 16-bit type and round takes ties to even.
// lo is an element of the group, so it is exact.  s = 0 (a constant group, or a
// range that underflows) gives n = 0.  A group with an infinity or NaN, or
// whose range overflows 32 bits, gets s = lo = NaN and reads back as NaN.  All
// of this is done in 32 bits with IEEE division; n and s are the only rounded
// values.  4 bits + (16 + 16) / 64 = 4.5 bits an element against 16.
//
// Layout: uint8 [num_blocks, Hkv, block_size, 9 D / 8]; one (block, head) is
// block_size / 16 tiles of 16 tokens, 18 D bytes each, so a tile is one
// contiguous piece and the attention kernel's lanes find their matrix-instruction
// fragments in whole 16-byte pieces (decode_q4.cuh):
//   [0, 8D)     K: token j at j D/2.  32-bit words of 8 dims; block b of 8 dims
//               is word (b%8)/2 * 2G + b/8 * 2 + b%2 (G = D/64 groups), dim 8b+i
//               in its bits 4i..4i+3
//   [8D, 16D)   V: block b of 8 dims at 64 b; token 4t+i, dims 8b+2m and 8b+2m+1
//               in the low and high half of byte 16t + 4m + i
//   [16D, 18D)  token j at j D/8: (s, lo) of each K group, then of each V group
// A token's bytes are its own (no byte holds two tokens), so rows are written
// without reading.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "cache.cuh"

namespace hcp {

constexpr int kQ4TileTokens = 16;

template <int D>
struct Q4 {
  static constexpr int kGroups = D / 64;
  static constexpr int kLanes = D / 8;       // lanes of one row, 8 dims each
  static constexpr int kTileBytes = 18 * D;
  static constexpr int kVOff = 8 * D;
  static constexpr int kParamOff = 16 * D;
  static constexpr int kTokenParams = D / 8;
  // byte offset of dim block b's word inside a token's K row
  static __host__ __device__ constexpr int k_word(int b) {
    return 4 * (((b & 7) >> 1) * (2 * kGroups) + (b >> 3) * 2 + (b & 1));
  }
};

template <bool F16>
__device__ __forceinline__ float q4_up(uint32_t bits16) {
  if constexpr (F16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
  else return __uint_as_float(bits16 << 16);
}
template <bool F16>
__device__ __forceinline__ uint32_t q4_down(float v) {
  if constexpr (F16) return __half_as_ushort(__float2half_rn(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
template <bool F16>
__device__ __forceinline__ void q4_unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = q4_up<F16>(w[i] & 0xffffu);
    x[2 * i + 1] = q4_up<F16>(w[i] >> 16);
  }
}
template <bool F16>
__device__ __forceinline__ uint4 q4_pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = q4_down<F16>(x[2 * i]) | (q4_down<F16>(x[2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Scale and lowest value of a group from its range over all lanes.  Elements
// that are not finite were entered as the range -inf .. inf.
template <bool F16>
__device__ __forceinline__ void q4_params(float lo, float hi, float& s, float& m) {
  s = q4_up<F16>(q4_down<F16>(__fdiv_rn(hi - lo, 15.f)));
  m = lo;
  if (!(s < INFINITY)) s = m = __int_as_float(0x7fffffff);
}
__device__ __forceinline__ void q4_range(float x, float& lo, float& hi) {
  const bool ok = fabsf(x) < INFINITY;
  lo = fminf(lo, ok ? x : -INFINITY);
  hi = fmaxf(hi, ok ? x : INFINITY);
}
__device__ __forceinline__ uint32_t q4_code(float x, float s, float m) {
  if (!(s > 0.f)) return 0;  // constant group, or NaN
  return static_cast<uint32_t>(fminf(fmaxf(rintf(__fdiv_rn(x - m, s)), 0.f), 15.f));
}

// Address of the tile that holds `off` of (block, head).
template <int D>
__device__ __forceinline__ long long q4_tile(long long blk, int h, int hkv, int bs, int off) {
  return ((blk * hkv + h) * (bs / kQ4TileTokens) + off / kQ4TileTokens) * Q4<D>::kTileBytes;
}

// One lane's 8 dims (block b) of a token's V row into its tile.
template <int D, bool F16>
__device__ __forceinline__ void q4_store_v(uint8_t* tile, int j, int b, const float (&x)[8], float s, float m) {
  uint8_t* at = tile + Q4<D>::kVOff + 64 * b + (j >> 2) * 16 + (j & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    at[4 * i] = static_cast<uint8_t>(q4_code(x[2 * i], s, m) | (q4_code(x[2 * i + 1], s, m) << 4));
}
template <int D, bool F16>
__device__ __forceinline__ void q4_store_params(uint8_t* tile, int j, int side, int group, float s, float m) {
  *reinterpret_cast<uint32_t*>(tile + Q4<D>::kParamOff + j * Q4<D>::kTokenParams +
                               4 * (side * Q4<D>::kGroups + group)) = q4_down<F16>(s) | (q4_down<F16>(m) << 16);
}
// Range over the 8 lanes of a group (lanes of one group are neighbours).
__device__ __forceinline__ void q4_reduce8(float& lo, float& hi) {
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
  }
}

struct Q4UpdateParams {
  const uint16_t* key;
  const uint16_t* value;
  long long key_row_stride;    // elements
  long long value_row_stride;
  const int64_t* slot_mapping;
  uint8_t* cache;
  long long num_blocks;
  long long num_tokens;
  int block_size;
  int bs_shift;
  int num_kv_heads;
};

// D/8 lanes per row, K and V rows of one (token, head) side by side; every lane
// of a warp takes part in the shuffles, the ones without a row with zeros.
template <int D, bool F16>
__global__ void __launch_bounds__(256) q4_update_kernel(const Q4UpdateParams p) {
  using L = Q4<D>;
  constexpr int kPair = 2 * L::kLanes;
  const int h = blockIdx.y;
  const int in = threadIdx.x % kPair;
  const bool is_v = in >= L::kLanes;
  const int b = in % L::kLanes;
  const long long tok = static_cast<long long>(blockIdx.x) * (256 / kPair) + threadIdx.x / kPair;
  long long blk = 0;
  int off = 0;
  const bool live = tok < p.num_tokens &&
                    slot_block(p.slot_mapping[tok], p.num_blocks, p.block_size, p.bs_shift, blk, off);
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  if (live)
    raw = reinterpret_cast<const uint4*>((is_v ? p.value + tok * p.value_row_stride : p.key + tok * p.key_row_stride) +
                                         static_cast<long long>(h) * D)[b];
  float x[8];
  q4_unpack8<F16>(raw, x);
  float lo = INFINITY, hi = -INFINITY, s, m;
#pragma unroll
  for (int i = 0; i < 8; ++i) q4_range(x[i], lo, hi);
  q4_reduce8(lo, hi);
  q4_params<F16>(lo, hi, s, m);
  if (!live) return;
  uint8_t* tile = p.cache + q4_tile<D>(blk, h, p.num_kv_heads, p.block_size, off);
  const int j = off % kQ4TileTokens;
  if (is_v) {
    q4_store_v<D, F16>(tile, j, b, x, s, m);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= q4_code(x[i], s, m) << (4 * i);
    *reinterpret_cast<uint32_t*>(tile + j * (D / 2) + L::k_word(b)) = w;
  }
  if ((b & 7) == 0) q4_store_params<D, F16>(tile, j, is_v ? 1 : 0, b >> 3, s, m);
}

struct Q4GatherParams {
  const uint8_t* cache;
  const int64_t* slot_mapping;
  uint16_t* key;
  uint16_t* value;
  long long key_row_stride;    // elements
  long long value_row_stride;
  long long num_blocks;
  long long num_tokens;
  int block_size;
  int bs_shift;
  int num_kv_heads;
};

template <int D, bool F16>
__global__ void __launch_bounds__(256) q4_gather_kernel(const Q4GatherParams p) {
  using L = Q4<D>;
  constexpr int kPair = 2 * L::kLanes;
  const int h = blockIdx.y;
  const int in = threadIdx.x % kPair;
  const bool is_v = in >= L::kLanes;
  const int b = in % L::kLanes;
  const long long tok = static_cast<long long>(blockIdx.x) * (256 / kPair) + threadIdx.x / kPair;
  if (tok >= p.num_tokens) return;
  long long blk;
  int off;
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (slot_block(p.slot_mapping[tok], p.num_blocks, p.block_size, p.bs_shift, blk, off)) {
    const uint8_t* tile = p.cache + q4_tile<D>(blk, h, p.num_kv_heads, p.block_size, off);
    const int j = off % kQ4TileTokens;
    const uint32_t sm = *reinterpret_cast<const uint32_t*>(tile + L::kParamOff + j * L::kTokenParams +
                                                           4 * ((is_v ? L::kGroups : 0) + (b >> 3)));
    const float s = q4_up<F16>(sm & 0xffffu), m = q4_up<F16>(sm >> 16);
    uint32_t w = 0;
    if (is_v) {
      const uint8_t* at = tile + L::kVOff + 64 * b + (j >> 2) * 16 + (j & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= static_cast<uint32_t>(at[4 * i]) << (8 * i);
    } else {
      w = *reinterpret_cast<const uint32_t*>(tile + j * (D / 2) + L::k_word(b));
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((w >> (4 * i)) & 15u), s, m);
    out = q4_pack8<F16>(x);
  }
  uint16_t* row = (is_v ? p.value + tok * p.value_row_stride : p.key + tok * p.key_row_stride) +
                  static_cast<long long>(h) * D;
  reinterpret_cast<uint4*>(row)[b] = out;
}

}  // namespace hcp
