// The 4-bit paged KV cache: its format, the scatter of new rows into it and the
// gather of rows out of it.
//
// A group is 64 dims of one token, KV head and side (K or V).  With lo and hi
// its smallest and largest element:
//   s = round16((hi - lo) / 15),  n_d = round((x_d - lo) / s) clamped to 0..15,
//   x'_d = lo + s n_d
// where round16 rounds to the rows' 16-bit type and round takes ties to even.
// lo is an element of the group, so it is exact.  s = 0 (a constant group, or a
// range that underflows; s below 2^-126 counts as 0) gives n = 0.  A group with an
// infinity or NaN, or whose range overflows 32 bits, gets s = lo = NaN and reads back
// as NaN.  All of this is done in 32 bits; n and s are the only rounded values.  4 bits + (16 + 16) / 64 = 4.5 bits an element against 16.
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
#include "sm100_ptx.cuh"

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
__device__ __forceinline__ float2 q4_up2(uint32_t w) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <bool F16>
__device__ __forceinline__ uint32_t q4_down2(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool F16>
__device__ __forceinline__ void q4_unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = q4_up2<F16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <bool F16>
__device__ __forceinline__ uint4 q4_pack8(const float (&x)[8]) {
  return make_uint4(q4_down2<F16>(x[0], x[1]), q4_down2<F16>(x[2], x[3]), q4_down2<F16>(x[4], x[5]),
                    q4_down2<F16>(x[6], x[7]));
}

// Packed pairs of the 16-bit type: smallest and largest, NaN wherever one is NaN.
template <bool F16>
__device__ __forceinline__ uint32_t q4_min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (F16) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t q4_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (F16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool F16>
constexpr uint32_t q4_inf2() { return F16 ? 0x7c007c00u : 0x7f807f80u; }

// Scale and lowest value of a group from the packed ranges of its elements at even
// and odd places.  The quotient by 15 is a product corrected by one residual
// (Markstein), which rounds correctly.  An infinity or NaN in the group, or a range
// past 32 bits, leaves the residual NaN or the scale infinite.
template <bool F16>
__device__ __forceinline__ void q4_params(uint32_t lo2, uint32_t hi2, float& s, float& m) {
  lo2 = q4_min2<F16>(lo2, __byte_perm(lo2, lo2, 0x1032));
  hi2 = q4_max2<F16>(hi2, __byte_perm(hi2, hi2, 0x1032));
  m = q4_up<F16>(lo2 & 0xffffu);
  const float d = q4_up<F16>(hi2 & 0xffffu) - m;
  constexpr float r = 1.f / 15.f;
  const float q = d * r;
  s = q4_up<F16>(q4_down<F16>(fmaf(fmaf(-q, 15.f, d), r, q)));
  if (s < 0x1p-126f) s = 0.f;
  if (!(s < INFINITY)) s = m = __int_as_float(0x7fffffff);
}
__device__ __forceinline__ float q4_reciprocal(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return r;
}
// Whole numbers of N elements of one group, element i in bits 4i..4i+3:
// round((x - m) / s), ties to even, 0 where s is 0 or NaN.  The quotient is a product
// with the reciprocal, corrected by one residual (Markstein's step): a quotient that
// is a tie comes out exact whatever the reciprocal's last bits, and one that is not
// keeps its side.  Adding 2^23 rounds to a whole number, whose bits are the sum's
// lowest.  (s is at most 2^128 / 15 and at least 2^-126: its reciprocal is a normal number.)
template <int N, bool F16>
__device__ __forceinline__ uint32_t q4_codes(const float* x, float s, float m) {
  if (!(s > 0.f)) return 0;
  const float r = q4_reciprocal(s);
  const float2 r2 = make_float2(r, r), s2 = make_float2(-s, -s), m2 = make_float2(-m, -m), one = make_float2(8388608.f, 8388608.f);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 d = __fadd2_rn(make_float2(x[i], x[i + 1]), m2);
    const float2 q = __fmul2_rn(d, r2);
    float2 t = __ffma2_rn(__ffma2_rn(q, s2, d), r2, q);
    if (F16) {  // a scale among fp16's smallest numbers may be rounded far down; else t is below 15.5
      t.x = fminf(t.x, 15.f);
      t.y = fminf(t.y, 15.f);
    }
    t = __fadd2_rn(t, one);
    w += __float_as_uint(t.x) << (4 * i);
    w += __float_as_uint(t.y) << (4 * i + 4);
  }
  constexpr uint32_t k2p23 = 0x4b000000u;  // the bits of 2^23, once per element
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) all += k2p23 << (4 * i);
  return w - all;
}

// Address of the tile that holds `off` of (block, head).
template <int D>
__device__ __forceinline__ long long q4_tile(long long blk, int h, int hkv, int bs, int off) {
  return ((blk * hkv + h) * (bs / kQ4TileTokens) + off / kQ4TileTokens) * Q4<D>::kTileBytes;
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

constexpr int kQ4Threads = 128;

// 16 tokens of one head on their way into the cache: their tile as it will stand
// there, and where each token goes.
template <int D>
struct Q4Stage {
  alignas(16) uint8_t tile[Q4<D>::kTileBytes];
  long long dst[kQ4TileTokens];  // cache offset of each token's tile, -1: nowhere
  int at[kQ4TileTokens];         // the token's place in it
  int whole;                     // all 16 tokens are that tile, in order
};

// Tokens are taken in runs of 16 that start where the first slot's tile starts,
// so that a request's chunk falls into whole tiles: run `g` holds tokens
// 16 g - phase .. + 15, phase the first slot's place in its tile.  There is one phase a
// call: in a batch of several chunks those that begin elsewhere in their tiles go token by
// token (16384 rows of 4 heads, D 128: scatter 28.6 us for 12.8, gather 9.5 for 8.0), as
// single tokens of many requests do (64 or 256 of them: 3.7 and 4.6 us, a launch's latency).
__device__ __forceinline__ int q4_phase(const int64_t* slots) {
  const long long s = slots[0];
  return s < 0 ? 0 : static_cast<int>(s & (kQ4TileTokens - 1));
}

// Called by whole warps: slot of token 16 run - phase + lane (lane < 16, -1 where there is
// none), and the run's first token.  Two runs' slots are read beside the first slot, so that
// nothing waits for the phase.
__device__ __forceinline__ long long q4_run_slots(const int64_t* slots, long long num_tokens, long long run,
                                                  long long& t0) {
  const int lane = threadIdx.x & 31;
  const long long at = (run - 1) * kQ4TileTokens + lane;
  const long long s = at >= 0 && at < num_tokens ? slots[at] : -1;
  const int phase = q4_phase(slots);
  t0 = run * kQ4TileTokens - phase;
  const long long mine = __shfl_sync(0xffffffffu, s, (kQ4TileTokens - phase + lane) & 31);
  return lane < kQ4TileTokens ? mine : -1;
}

// Called by the first warp: places of the run's tokens (`slot`: of lane's token, -1 where it stays out).
template <int D>
__device__ __forceinline__ void q4_place(Q4Stage<D>& st, const Q4UpdateParams& p, long long slot, int h) {
  const int lane = threadIdx.x & 31;
  long long blk = 0;
  int off = 0;
  const bool keep = slot_block(slot, p.num_blocks, p.block_size, p.bs_shift, blk, off);
  const long long first = __shfl_sync(0xffffffffu, slot, 0);
  const unsigned in = __ballot_sync(0xffffffffu, keep && slot == first + lane && (first & (kQ4TileTokens - 1)) == 0);
  if (lane < kQ4TileTokens) {
    st.dst[lane] = keep ? q4_tile<D>(blk, h, p.num_kv_heads, p.block_size, off) : -1;
    st.at[lane] = off % kQ4TileTokens;
  }
  if (lane == 0) st.whole = in == 0xffffu;
}

// 4 dims from d (a multiple of 4) of token j's K row, and one block of 8 dims of its V row.
template <int D>
__device__ __forceinline__ void q4_stage_k4(Q4Stage<D>& st, int j, int d, uint32_t codes) {
  *reinterpret_cast<uint16_t*>(st.tile + j * (D / 2) + Q4<D>::k_word(d >> 3) + ((d >> 2) & 1) * 2) =
      static_cast<uint16_t>(codes);
}
template <int D>
__device__ __forceinline__ void q4_stage_k8(Q4Stage<D>& st, int j, int b, uint32_t codes) {
  *reinterpret_cast<uint32_t*>(st.tile + j * (D / 2) + Q4<D>::k_word(b)) = codes;
}
template <int D>
__device__ __forceinline__ void q4_stage_v8(Q4Stage<D>& st, int j, int b, uint32_t codes) {
  uint8_t* at = st.tile + Q4<D>::kVOff + 64 * b + (j >> 2) * 16 + (j & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) at[4 * i] = static_cast<uint8_t>(codes >> (8 * i));
}
template <int D, bool F16>
__device__ __forceinline__ void q4_stage_params(Q4Stage<D>& st, int j, int side, int group, float s, float m) {
  *reinterpret_cast<uint32_t*>(st.tile + Q4<D>::kParamOff + j * Q4<D>::kTokenParams +
                               4 * (side * Q4<D>::kGroups + group)) = q4_down<F16>(s) | (q4_down<F16>(m) << 16);
}

// The staged run into the cache: a whole tile in 16-byte pieces, else token by token.
template <int D>
__device__ __forceinline__ void q4_flush(const Q4Stage<D>& st, uint8_t* cache) {
  using L = Q4<D>;
  if (st.whole) {
    uint4* dst = reinterpret_cast<uint4*>(cache + st.dst[0]);
    for (int i = threadIdx.x; i < L::kTileBytes / 16; i += blockDim.x) dst[i] = reinterpret_cast<const uint4*>(st.tile)[i];
    return;
  }
  constexpr int kWords = D / 8, kItems = 2 * kWords + L::kTokenParams / 4;
  for (int i = threadIdx.x; i < kQ4TileTokens * kItems; i += blockDim.x) {
    const int j = i / kItems, e = i - j * kItems;
    if (st.dst[j] < 0) continue;
    uint8_t* tile = cache + st.dst[j];
    const int to = st.at[j];
    if (e < kWords) {
      *reinterpret_cast<uint32_t*>(tile + to * (D / 2) + 4 * e) = *reinterpret_cast<const uint32_t*>(st.tile + j * (D / 2) + 4 * e);
    } else if (e < 2 * kWords) {
      const int b = L::kVOff + 64 * (e - kWords);
#pragma unroll
      for (int m = 0; m < 4; ++m) tile[b + (to >> 2) * 16 + 4 * m + (to & 3)] = st.tile[b + (j >> 2) * 16 + 4 * m + (j & 3)];
    } else {
      const int b = L::kParamOff + 4 * (e - 2 * kWords);
      *reinterpret_cast<uint32_t*>(tile + b + to * L::kTokenParams) =
          *reinterpret_cast<const uint32_t*>(st.tile + b + j * L::kTokenParams);
    }
  }
}

// A block takes 16 tokens of one head: D/8 lanes a row quantise K and V rows into the
// staged tile, which leaves in 16-byte pieces where it is whole (a chunk of a prefill),
// token by token elsewhere (decodes).  HBM's share is 2 bytes read, 9/16 written an element; what
// bounds it is the quantisation's instructions (77% of the issue slots): 13.3 us for 16384 rows of 4
// heads, D 128, against 6.7 us of bytes; 45 us with byte stores straight to the cache.
template <int D, bool F16>
__global__ void __launch_bounds__(kQ4Threads) q4_update_kernel(const Q4UpdateParams p) {
  using L = Q4<D>;
  __shared__ Q4Stage<D> st;
  ptx::chain_wait();
  ptx::chain_next();
  constexpr int kRows = kQ4Threads / L::kLanes;
  const int h = blockIdx.x % p.num_kv_heads;
  long long t0;
  const long long slot = q4_run_slots(p.slot_mapping, p.num_tokens, blockIdx.x / p.num_kv_heads, t0);
  if (t0 >= p.num_tokens) return;
  if (threadIdx.x < 32) q4_place<D>(st, p, slot, h);
  const int b = threadIdx.x % L::kLanes;
  uint4 raw[2 * kQ4TileTokens / kRows];
#pragma unroll
  for (int i = 0; i < 2 * kQ4TileTokens / kRows; ++i) {
    const int row = i * kRows + threadIdx.x / L::kLanes, j = row % kQ4TileTokens;
    const long long tok = t0 + j;
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tok >= 0 && tok < p.num_tokens)
      raw[i] = reinterpret_cast<const uint4*>((row >= kQ4TileTokens ? p.value + tok * p.value_row_stride
                                                                    : p.key + tok * p.key_row_stride) +
                                              static_cast<long long>(h) * D)[b];
  }
#pragma unroll
  for (int i = 0; i < 2 * kQ4TileTokens / kRows; ++i) {
    const int row = i * kRows + threadIdx.x / L::kLanes, j = row % kQ4TileTokens;
    const bool is_v = row >= kQ4TileTokens;
    float x[8], s, m;
    q4_unpack8<F16>(raw[i], x);
    uint32_t lo = q4_min2<F16>(q4_min2<F16>(raw[i].x, raw[i].y), q4_min2<F16>(raw[i].z, raw[i].w));
    uint32_t hi = q4_max2<F16>(q4_max2<F16>(raw[i].x, raw[i].y), q4_max2<F16>(raw[i].z, raw[i].w));
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) {  // 8 neighbouring lanes hold a group
      lo = q4_min2<F16>(lo, __shfl_xor_sync(0xffffffffu, lo, k));
      hi = q4_max2<F16>(hi, __shfl_xor_sync(0xffffffffu, hi, k));
    }
    q4_params<F16>(lo, hi, s, m);
    const uint32_t codes = q4_codes<8, F16>(x, s, m);
    if (is_v) q4_stage_v8<D>(st, j, b, codes);
    else q4_stage_k8<D>(st, j, b, codes);
    if ((b & 7) == 0) q4_stage_params<D, F16>(st, j, is_v ? 1 : 0, b >> 3, s, m);
  }
  __syncthreads();
  q4_flush<D>(st, p.cache);
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

template <bool F16>
__device__ __forceinline__ uint4 q4_open8(uint32_t w, uint32_t sm) {
  const float s = q4_up<F16>(sm & 0xffffu), m = q4_up<F16>(sm >> 16);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((w >> (4 * i)) & 15u), s, m);
  return q4_pack8<F16>(x);
}

// A warp takes a run of 16 tokens of one head (runs as in the scatter).  Where the run is a
// whole tile, V is read in its 16-byte pieces of 4 tokens x 8 dims; rows leave in full lines
// either way.  Bound by HBM: 9/16 bytes read, 2 written an element.  Measured: 7.8 us for 16384
// rows of 4 heads, D 128 (15.6 us token by token).
template <int D, bool F16>
__global__ void __launch_bounds__(kQ4Threads) q4_gather_kernel(const Q4GatherParams p) {
  using L = Q4<D>;
  constexpr int kRows = 32 / L::kLanes;  // rows of a warp's store
  ptx::chain_wait();
  ptx::chain_next();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * (kQ4Threads / 32) + threadIdx.x / 32;
  const int h = static_cast<int>(unit % p.num_kv_heads);
  // lane j < 16: token j's tile and place
  long long t0, blk = 0, src = -1;
  int off = 0;
  const long long slot = q4_run_slots(p.slot_mapping, p.num_tokens, unit / p.num_kv_heads, t0);
  if (t0 >= p.num_tokens) return;
  if (slot_block(slot, p.num_blocks, p.block_size, p.bs_shift, blk, off))
    src = q4_tile<D>(blk, h, p.num_kv_heads, p.block_size, off);
  const long long first = __shfl_sync(0xffffffffu, slot, 0);
  const bool whole = (__ballot_sync(0xffffffffu, src >= 0 && slot == first + lane && (first & (kQ4TileTokens - 1)) == 0) &
                      0xffffu) == 0xffffu;
  const int b = lane % L::kLanes, sub = lane / L::kLanes;
  uint16_t* const key = p.key + t0 * p.key_row_stride + static_cast<long long>(h) * D + 8 * b;
  uint16_t* const value = p.value + t0 * p.value_row_stride + static_cast<long long>(h) * D + 8 * b;
  if (whole) {
    const uint8_t* tile = p.cache + __shfl_sync(0xffffffffu, src, 0);
    const uint8_t* prm = tile + L::kParamOff + 4 * (b >> 3);
#pragma unroll
    for (int i = 0; i < kQ4TileTokens / kRows; ++i) {
      const int j = i * kRows + sub;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + j * (D / 2) + L::k_word(b));
      const uint32_t sm = *reinterpret_cast<const uint32_t*>(prm + j * L::kTokenParams);
      *reinterpret_cast<uint4*>(key + j * p.key_row_stride) = q4_open8<F16>(w, sm);
    }
#pragma unroll
    for (int i = 0; i < 4 / kRows; ++i) {
      const int t = i * kRows + sub;
      const uint4 v = *reinterpret_cast<const uint4*>(tile + L::kVOff + 64 * b + 16 * t);
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // token 4t + k: byte k of each word
        const int j = 4 * t + k;
        const uint32_t w = __byte_perm(__byte_perm(v.x, v.y, k | ((4 + k) << 4)), __byte_perm(v.z, v.w, k | ((4 + k) << 4)), 0x5410);
        const uint32_t sm = *reinterpret_cast<const uint32_t*>(prm + j * L::kTokenParams + 4 * L::kGroups);
        *reinterpret_cast<uint4*>(value + j * p.value_row_stride) = q4_open8<F16>(w, sm);
      }
    }
    return;
  }
#pragma unroll 4
  for (int i = 0; i < kQ4TileTokens / kRows; ++i) {
    const int j = i * kRows + sub;
    const long long at = __shfl_sync(0xffffffffu, src, j);
    const int place = __shfl_sync(0xffffffffu, off, j) % kQ4TileTokens;
    if (t0 + j < 0 || t0 + j >= p.num_tokens) continue;
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    if (at >= 0) {
      const uint8_t* tile = p.cache + at;
      const uint32_t* prm = reinterpret_cast<const uint32_t*>(tile + L::kParamOff + place * L::kTokenParams) + (b >> 3);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + place * (D / 2) + L::k_word(b));
      const uint8_t* vb = tile + L::kVOff + 64 * b + (place >> 2) * 16 + (place & 3);
      const uint32_t vw = vb[0] | (vb[4] << 8) | (vb[8] << 16) | (static_cast<uint32_t>(vb[12]) << 24);
      k = q4_open8<F16>(kw, prm[0]);
      v = q4_open8<F16>(vw, prm[L::kGroups]);
    }
    *reinterpret_cast<uint4*>(key + j * p.key_row_stride) = k;
    *reinterpret_cast<uint4*>(value + j * p.value_row_stride) = v;
  }
}

}  // namespace hcp
