// Single-token attention over the 4-bit paged cache (q4_cache.cuh) for B200.
//
// For every query row r with its request's pages and n = kv_lens[r] keys, per
// head h of KV head h / G:
//   o = sum_j softmax_j(scale q . k_j) v_j,   k_j, v_j = lo + s n  per 64 dims,
//   lse = log sum_j exp(scale q . k_j).
//
// Bound by HBM: 9/8 D bytes per key and KV head (K and V), against 2 G D
// products.  What has to be kept small is the work per byte.  So:
//   * the whole numbers n are the matrix operands, exact in fp16; scales and lowest
//     values are applied outside in 32 bits, per 64-dim group:
//       q . k  = sum_g  s_g (q_g . (64 + n_g)) + (lo_g - 64 s_g) sum(q_g)
//       o_g    = sum_j (p_j s_j) (n_j - 8)     + sum_j p_j (lo_j + 8 s_j)
//     V is centred, so that sums over many keys stay as small as their own terms; a
//     score's sum is over 64 products, where the offset costs 6 bits of 24 and saves
//     the centring (a ninth of the kernel's instructions);
//   * keys are the rows of the first product (16 keys x 8 heads) and dims those of
//     the second (16 dims x 8 heads), so a group of up to 8 query heads fills the
//     instruction's 8 columns instead of half of 16 rows;
//   * the tile layout gives every lane its fragments of both products in whole
//     16-byte pieces: no transposes but of the 8 x 8 blocks of P between the products
//     (movmatrix);
//   * q and p_j s_j enter the products in fp16, scaled by powers of two: q by its
//     head's largest element (no loss), p_j s_j by the largest of them that the head
//     and group met so far, in weights of the present base: a scale counts by what its
//     key weighs, so a large value that nobody attends takes no bits from the others.
//     Rounding p_j s_j to 11 bits is off by at most 2^-11 of each key's term, and by
//     2^-33 of the largest p s where that is more (fp16's smallest numbers).  The terms'
//     weights sum to one, so this is an eighth of what rounding the result to bf16 may be
//     off, and is left there.  A result of fp16 or 32 bits would show it: for those
//     (REST) what the rounding leaves is multiplied too, which takes each term to 2^-22 for
//     8 matrix instructions more on a tile's 16 (33 ragged rows, D 64, fp16: 17.1 us for 16.5;
//     64 rows x 32768 keys, D 128: 271 us for 239, which bf16 results are spared).
//
// Split: all rows' tiles of 16 keys, heads outermost in a row, form one line that
// the warps cut into equal pieces, so any mix of lengths is even in this kernel (the
// join's form goes by the mean number of parts) and nothing about the lengths has to be
// known on the host.  Every block sums the lengths itself.  A
// warp works alone: its tiles come through a ring of asynchronous copies in shared
// memory, two tiles a step.  A (row, KV head) that lies inside one piece is written
// to out from the warp's registers; one that is cut leaves a partial (O, base, sum)
// per piece in the workspace, and a second kernel, scheduled as the first runs out,
// joins them in order.
//
// Measured (28 heads over 4, D 128, bf16; a replayed graph): 64 rows x 32768 keys 239 us =
// 5.1 TB/s, 0.78 of the measured copy rate (273 us in a long stream of calls, whose power lowers the
// clock); 1 x 131072 keys 26.9 us; 16 rows of up to 300 keys 11.9 us, latencies.  DRAM is half busy and
// the pages' place does not matter (as long with all of them in L2); of the issue slots 57 % are, with
// 293 instructions a tile.  What bounds it is a step's chain of dependent instructions on three warps
// a scheduler (the stalls are fixed latencies and busy pipes).  Four warps a scheduler leave 128
// registers, too few for two tiles a step (20 us more); two cover less latency (20 us more).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "decode.cuh"
#include "q4_cache.cuh"

namespace hcp {

constexpr int kDq4Warps = 4;
constexpr int kDq4Threads = kDq4Warps * 32;
constexpr int kDq4Sms = 148;
constexpr int kDq4MaxCtas = 3 * kDq4Sms;
constexpr int kDq4MaxPieces = kDq4MaxCtas * kDq4Warps;
constexpr int kDq4Stages = 3;    // steps of a warp's ring: one read, the others in flight
constexpr int kDq4Step = 2;      // tiles of a step, and of a piece at least
constexpr int kDq4JoinWarps = 16;
constexpr int kDq4JoinThreads = 256;                          // of a join block where pairs are many
constexpr int kDq4FewParts = 32;                              // of a pair that a warp joins alone
constexpr int kDq4MaxLong = 2 * kDq4MaxPieces / kDq4FewParts; // pairs of more: a piece has parts of two pairs at most
constexpr int kDq4Lookers = 32;                               // blocks a head that look for them
constexpr int kDq4UnitTop = 127 + 118;  // exponent of the finest unit's reciprocal: p_j <= 2^8 times it stays finite
// Blocks of an SM: 168 registers a thread, and twice the sums beyond 8 heads a group.
constexpr int dq4_ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }

struct DecodeQ4Params {
  const void* q;
  long long q_row_stride;
  const uint8_t* cache;
  const int32_t* block_table;
  long long bt_stride;
  long long bt_width;
  long long bt_rows;
  long long num_blocks;
  const int32_t* kv_lens;
  const int32_t* token_req;   // may be null: row r reads table row r
  void* out;
  long long out_row_stride;
  float* lse;                 // may be null
  long long lse_stride;
  int4* desc;                 // [rows][Hkv] {first piece, its slot, pieces, 0}; pieces 0: nothing to join
  float2* part_ml;            // [pieces][2][G] base (log2 units) and sum
  float* part_o;              // [pieces][2][G][D] sums to that base
  int rows;
  int num_heads;
  int num_kv_heads;
  int group;
  int block_size;
  int sub_shift;              // log2(tiles in a block)
  float scale_log2;
  int out_dt;
  int out_vec;                // rows of out take 16-byte stores
};

// 16 bytes, or 16 zeros where `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Whole numbers of a word's nibble pairs (i, i + 4) as n - 8 in fp16, exact, by the
// published method of 4-bit weight kernels: bits put into the mantissa of a power of two.
// With a nibble in mantissa bits 0-3 of 1024 the value is 1024 + n, in bits 4-7 it is
// 1024 + 16 n: two pairs without a shift, the other two after one shift by 8.  The two
// constants come in registers that the compiler cannot see through: as immediates
// they would cost a move at every use (an instruction takes one immediate).
struct Q4Consts {
  uint32_t k1024, k72;  // 1024 twice, -72 twice
};
__device__ __forceinline__ Q4Consts q4_consts() {
  Q4Consts c;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(c.k1024));
  asm volatile("mov.b32 %0, 0xd480d480;" : "=r"(c.k72));
  return c;
}
__device__ __forceinline__ void q4_pairs(uint32_t w, const Q4Consts& c, uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = i == 0 ? w : w >> 8;
    uint32_t a, b;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(a) : "r"(v), "r"(c.k1024));  // (v & mask) | 1024
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(b) : "r"(v), "r"(c.k1024));
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r[2 * i]) : "r"(a), "r"(0xe408e408u));     // - 1032
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[2 * i + 1]) : "r"(b), "r"(0x2c002c00u), "r"(c.k72));  // / 16 - 72
  }
}

__device__ __forceinline__ uint32_t q4_max2_f16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The same pairs as 1024 + 16 n, without the centring: for products whose sums start
// anew in every tile, where 16 (64 + n) costs 6 bits of 24 and the offset's share is
// known (64 times the sum of the other operand).
__device__ __forceinline__ void q4_pairs_raw(uint32_t w, const Q4Consts& c, uint32_t (&r)[4]) {
  const uint32_t v[4] = {w << 4, w, w >> 4, w >> 8};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(r[i]) : "r"(v[i]), "r"(c.k1024));
}

// Tiles of a row (0 for a padding row or an empty one).
__device__ __forceinline__ int dq4_len(const DecodeQ4Params& p, int r, int& req) {
  req = p.token_req != nullptr ? p.token_req[r] : r;
  if (req < 0 || req >= p.bt_rows) return -1;
  const long long n = max(0, p.kv_lens[r]);
  return static_cast<int>(min(n, p.bt_width * p.block_size));
}
__device__ __forceinline__ int dq4_tiles(int len) { return len > 0 ? (len + 15) >> 4 : 0; }

template <int D>
struct Dq4Smem {
  static constexpr int kStepBytes = kDq4Step * Q4<D>::kTileBytes;
  static constexpr int kRing = kDq4Stages * kStepBytes;
  alignas(16) uint8_t ring[kDq4Warps][kRing];
  long long wsum[kDq4Warps];
  long long first_cum[kDq4Warps];  // tiles of the line before the row of each warp's first tile
  int4 first[kDq4Warps];           // that row, its request, its keys
};

__device__ __forceinline__ void dq4_store(const DecodeQ4Params& p, long long row, int head, int D, int d, float v) {
  const long long i = row * p.out_row_stride + static_cast<long long>(head) * D + d;
  if (p.out_dt == HCP_F32) static_cast<float*>(p.out)[i] = v;
  else if (p.out_dt == HCP_F16) static_cast<__half*>(p.out)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}

// 8 neighbouring dims of a head's result.
__device__ __forceinline__ void dq4_store8(const DecodeQ4Params& p, long long row, int head, int D, int d, const float (&v)[8]) {
  if (p.out_vec) {
    const long long i = row * p.out_row_stride + static_cast<long long>(head) * D + d;
    if (p.out_dt == HCP_F32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + i);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i) = p.out_dt == HCP_F16 ? q4_pack8<true>(v) : q4_pack8<false>(v);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) dq4_store(p, row, head, D, d + k, v[k]);
  }
}

template <int D, bool F16, int NT, bool REST>
__global__ void __launch_bounds__(kDq4Threads, dq4_ctas_per_sm(NT))
    decode_q4_kernel(const __grid_constant__ DecodeQ4Params p) {
  using L = Q4<D>;
  using S = Dq4Smem<D>;
  constexpr int NG = L::kGroups;
  constexpr int KW = 2 * NG;           // K words of a lane and token
  constexpr int U = kDq4Step;
  extern __shared__ __align__(16) uint8_t dq4_smem[];
  S& sm = *reinterpret_cast<S*>(dq4_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.group, Hkv = p.num_kv_heads;
  const Q4Consts consts = q4_consts();
  ptx::chain_wait();

  // ---- the line of tiles: sums of every thread's run of rows
  const int run = (p.rows + kDq4Threads - 1) / kDq4Threads;
  long long mine = 0;
  int last_len = 0, last_req = 0;  // of the run's last row: its only one where there are few
  for (int r = tid * run; r < min(p.rows, (tid + 1) * run); ++r) {
    last_len = dq4_len(p, r, last_req);
    mine += dq4_tiles(last_len);
  }
  long long inc = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc, s);
    if (lane >= s) inc += a;
  }
  if (lane == 31) sm.wsum[warp] = inc;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kDq4Warps; ++w) {
    before += w < warp ? sm.wsum[w] : 0;
    all += sm.wsum[w];
  }
  ptx::chain_next();

  // ---- the warps' pieces of the line; the thread whose rows hold a piece's first tile says where
  constexpr int kPieces = kDq4Sms * dq4_ctas_per_sm(NT) * kDq4Warps;
  const long long total = all * Hkv;
  const long long piece = max(1ll, (total + kPieces * U - 1) / (kPieces * U)) * U;
#pragma unroll
  for (int w = 0; w < kDq4Warps; ++w) {
    const long long at = (static_cast<long long>(blockIdx.x) * kDq4Warps + w) * piece;
    long long cum = (before + inc - mine) * Hkv;
    if (at >= cum && at < cum + mine * Hkv) {
      int r = tid * run, req = last_req, n = run == 1 ? last_len : dq4_len(p, r, req);
      while (r + 1 < p.rows && at >= cum + static_cast<long long>(dq4_tiles(n)) * Hkv) {
        cum += static_cast<long long>(dq4_tiles(n)) * Hkv;
        n = dq4_len(p, ++r, req);
      }
      sm.first[w] = make_int4(r, req, n, 0);
      sm.first_cum[w] = cum;
    }
  }
  __syncthreads();
  const int me = blockIdx.x * kDq4Warps + warp;
  const long long f_begin = me * piece, f_end = min(total, f_begin + piece);
  long long f = f_begin, cum = 0;
  int row = 0, req = 0, len = 0;
  if (f < f_end) {
    const int4 first = sm.first[warp];
    row = first.x;
    req = first.y;
    len = first.z;
    cum = sm.first_cum[warp];
  }
  const uint32_t ring = ptx::smem_u32(sm.ring[warp]) + 16 * lane;
  const int sub_mask = (1 << p.sub_shift) - 1;

  while (f < f_end) {
    while (row + 1 < p.rows && f >= cum + static_cast<long long>(dq4_tiles(len)) * Hkv) {
      cum += static_cast<long long>(dq4_tiles(len)) * Hkv;
      len = dq4_len(p, ++row, req);
    }
    const int tiles = dq4_tiles(len);
    if (f >= cum + static_cast<long long>(tiles) * Hkv) break;  // lengths changed under the call
    const uint32_t in_row = static_cast<uint32_t>(f - cum);
    const int kvh = static_cast<int>(in_row / static_cast<uint32_t>(tiles));
    const int t0 = static_cast<int>(in_row - static_cast<uint32_t>(kvh) * static_cast<uint32_t>(tiles));
    const int n = static_cast<int>(min(static_cast<long long>(tiles - t0), f_end - f));
    const int steps = (n + U - 1) / U;

    // ---- tiles t0 .. t0 + n, a step of two at a time through the ring
    const int32_t* bt = p.block_table + req * p.bt_stride;
    // page of tile 32 b + lane; the next 32 are on their way while these are used
    auto pages = [&](int b) {
      int v = -1;
      if (32 * b + lane < n) v = bt[(t0 + 32 * b + lane) >> p.sub_shift];
      return v;  // looked at when it is used
    };
    int page = pages(0), page_next = pages(1);
    uint4 raw[NT][KW];  // q, on its way while the ring fills
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        raw[nt][w] = make_uint4(0u, 0u, 0u, 0u);
        if (nt * 8 + g < G)
          raw[nt][w] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + row * p.q_row_stride +
                                                       static_cast<long long>(kvh * G + nt * 8 + g) * D + 64 * (w >> 1) +
                                                       16 * t + 8 * (w & 1));
      }
    uint32_t held = 0;          // bits 2k, 2k + 1: whether the tiles of the step issued k before the last are there
    int in_at = 0, out_at = 0;  // ring offsets of the next copy and of the next step to read
    auto issue = [&](int st) {
      uint32_t there = 0;
      if (st < steps) {
        if (st > 0 && (st & (32 / U - 1)) == 0) {
          page = page_next;
          page_next = pages(st / (32 / U) + 1);
        }
        const uint8_t* src[U];
        uint32_t bytes[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t blk = static_cast<uint32_t>(__shfl_sync(0xffffffffu, page, (U * st + u) & 31));  // -1 past the last tile too
          const bool in = blk < static_cast<uint32_t>(p.num_blocks);
          there |= in ? 1u << u : 0u;
          bytes[u] = in ? 16u : 0u;
          blk = in ? blk : 0u;
          const uint32_t at = ((blk * Hkv + kvh) << p.sub_shift) + ((t0 + U * st + u) & sub_mask);
          src[u] = p.cache + 16 * lane + static_cast<uint64_t>(at) * L::kTileBytes;
        }
        constexpr int kChunks = L::kTileBytes / 16;
#pragma unroll
        for (int c = 0; c < (U * kChunks + 31) / 32; ++c) {
          // chunk 32 c + lane of the step's two tiles
          const bool second = 32 * c >= kChunks || (32 * c + 31 >= kChunks && 32 * c + lane >= kChunks);
          if (32 * c + 31 < U * kChunks || 32 * c + lane < U * kChunks)
            cp_async16(ring + in_at + 512 * c, (second ? src[1] - L::kTileBytes : src[0]) + 512 * c, second ? bytes[1] : bytes[0]);
        }
      }
      in_at = in_at == (kDq4Stages - 1) * S::kStepBytes ? 0 : in_at + S::kStepBytes;
      held = (held << U) | there;
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kDq4Stages - 1; ++i) issue(i);

    // ---- Q fragments: columns are heads, lane's k index pairs (d, d + 4).  Each head is
    // scaled by a power of two into fp16's range and rounded to it: exact but for elements below
    // 2^-18 of its largest, which are off by at most 2^-29 of that.  (Not to the range's top: sums
    // times large scales have to stay finite.)  The power goes into the head's factor.
    uint32_t qb[NT][2 * KW][2];
    float sq[NT][NG][2];  // 16 times the sums of the scaled q over each group, heads 2t and 2t+1
    float hs[NT][2];      // score in log2 units = hs * 16 (scaled q . k)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        float x[8];
        q4_unpack8<F16>(raw[nt][w], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with top * 2^e in [2^4, 2^5), e at most 126 (and 0 for an empty or infinite head)
      const int ex = static_cast<int>(__float_as_uint(top) >> 23);
      const int e = ex == 0 || ex == 255 ? 0 : min(126, 131 - ex);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      float part[NG];
#pragma unroll
      for (int a = 0; a < NG; ++a) part[a] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        float x[8];
        q4_unpack8<F16>(raw[nt][w], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= up;
          part[w >> 1] += x[i];
        }
        qb[nt][2 * w][0] = pack2<true>(x[0], x[4]);
        qb[nt][2 * w][1] = pack2<true>(x[1], x[5]);
        qb[nt][2 * w + 1][0] = pack2<true>(x[2], x[6]);
        qb[nt][2 * w + 1][1] = pack2<true>(x[3], x[7]);
      }
#pragma unroll
      for (int a = 0; a < NG; ++a) {
        part[a] += __shfl_xor_sync(0xffffffffu, part[a], 1);
        part[a] += __shfl_xor_sync(0xffffffffu, part[a], 2);
        sq[nt][a][0] = 16.f * __shfl_sync(0xffffffffu, part[a], 8 * t);
        sq[nt][a][1] = 16.f * __shfl_sync(0xffffffffu, part[a], 8 * t + 4);
      }
      // at least the smallest number of 32 bits: with 0 an absent key's -inf would be NaN (scores of 2^-22 at most stay)
      const float down = fmaxf(0.0625f * p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - e) << 23), 0x1p-149f);
      hs[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      hs[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
    }
    float o[NT][NG][4][4];
    float vz[NT][NG][2], l_run[NT][2];
    float base[NT][2];   // of the weights: the running maximum or up to 8 below it; 0 before the first key
    float limit[NT][2];  // the score at which the base has to rise: (base + 8) / hs, -inf before the first key
    float vinv[NT][NG][2];  // powers of two that multiply p_j s_j: the sums o are in units of 1 / vinv
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int a = 0; a < NG; ++a) {
        vz[nt][a][0] = vz[nt][a][1] = 0.f;
        vinv[nt][a][0] = vinv[nt][a][1] = __uint_as_float(kDq4UnitTop << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][a][i][0] = o[nt][a][i][1] = o[nt][a][i][2] = o[nt][a][i][3] = 0.f;
      }
      limit[nt][0] = limit[nt][1] = -INFINITY;
      base[nt][0] = base[nt][1] = 0.f;
      l_run[nt][0] = l_run[nt][1] = 0.f;
    }
    for (int st = 0; st < steps; ++st) {
      cp_async_wait<kDq4Stages - 2>();
      __syncwarp();  // every lane's pieces are in, and the step before is read by all
      issue(st + kDq4Stages - 1);
      const uint8_t* step = sm.ring[warp] + out_at;
      out_at = out_at == (kDq4Stages - 1) * S::kStepBytes ? 0 : out_at + S::kStepBytes;
      // keys of the step; where some of its 32 are missing (past the end, or a page outside the cache), masks
      const int left = min(len - 16 * (t0 + U * st), 16 * (n - U * st));
      const uint32_t there = held >> (U * (kDq4Stages - 1));
      const bool whole_step = left >= 16 * U && (there & 3u) == 3u;
      uint32_t prm[U][2][2 * NG];  // of tokens 2g, 2g+1: K (s, lo) of each group, then V
      float sc[U][NT][4];          // scores: rows are tokens 2g (c0, c1) and 2g+1 (c2, c3)
      bool raise = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint8_t* tile = step + u * L::kTileBytes;
        uint32_t kw[2][KW];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint8_t* pp = tile + L::kParamOff + (2 * g + e) * L::kTokenParams;
          const uint8_t* kp = tile + (2 * g + e) * (D / 2) + t * (D / 8);
          if constexpr (NG == 2) {
            const uint4 v = *reinterpret_cast<const uint4*>(pp), w = *reinterpret_cast<const uint4*>(kp);
            prm[u][e][0] = v.x; prm[u][e][1] = v.y; prm[u][e][2] = v.z; prm[u][e][3] = v.w;
            kw[e][0] = w.x; kw[e][1] = w.y; kw[e][2] = w.z; kw[e][3] = w.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(pp), w = *reinterpret_cast<const uint2*>(kp);
            prm[u][e][0] = v.x; prm[u][e][1] = v.y;
            kw[e][0] = w.x; kw[e][1] = w.y;
          }
        }
        if (!whole_step) {  // unwritten bytes may be anything
          const int m = (there >> u) & 1u ? left - 16 * u - 2 * g : 0;
#pragma unroll
          for (int a = 0; a < 2 * NG; ++a) {
            prm[u][0][a] = m > 0 ? prm[u][0][a] : 0u;
            prm[u][1][a] = m > 1 ? prm[u][1][a] : 0u;
          }
        }
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          float acc[NT][4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t x[4], y[4];
            q4_pairs_raw(kw[0][2 * a + e], consts, x);
            q4_pairs_raw(kw[1][2 * a + e], consts, y);
            const uint32_t fa[4] = {x[0], y[0], x[1], y[1]}, fb[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int kk = 2 * (2 * a + e);
              if (e == 0) mma16816_first(acc[nt], fa, qb[nt][kk][0], qb[nt][kk][1]);
              else mma16816<true>(acc[nt], fa, qb[nt][kk][0], qb[nt][kk][1]);
              mma16816<true>(acc[nt], fb, qb[nt][kk + 1][0], qb[nt][kk + 1][1]);
            }
          }
          const float s0 = q4_up<F16>(prm[u][0][a] & 0xffffu), z0 = fmaf(-64.f, s0, q4_up<F16>(prm[u][0][a] >> 16));
          const float s1 = q4_up<F16>(prm[u][1][a] & 0xffffu), z1 = fmaf(-64.f, s1, q4_up<F16>(prm[u][1][a] >> 16));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 zz = make_float2(e == 0 ? z0 : z1, e == 0 ? z0 : z1), ss = make_float2(e == 0 ? s0 : s1, e == 0 ? s0 : s1);
              const float2 qq = make_float2(sq[nt][a][0], sq[nt][a][1]);
              const float2 zq = a == 0 ? __fmul2_rn(zz, qq) : __ffma2_rn(zz, qq, make_float2(sc[u][nt][2 * e], sc[u][nt][2 * e + 1]));
              const float2 r = __ffma2_rn(ss, make_float2(acc[nt][2 * e], acc[nt][2 * e + 1]), zq);
              sc[u][nt][2 * e] = r.x;
              sc[u][nt][2 * e + 1] = r.y;
            }
        }
        if (!whole_step) {
          const int m = (there >> u) & 1u ? left - 16 * u - 2 * g : 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][nt][e] = m > (e >> 1) ? sc[u][nt][e] : -INFINITY;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float m0 = fmaxf(sc[0][nt][0], sc[0][nt][2]), m1 = fmaxf(sc[0][nt][1], sc[0][nt][3]);
#pragma unroll
        for (int u = 1; u < U; ++u) {
          m0 = fmaxf(m0, fmaxf(sc[u][nt][0], sc[u][nt][2]));
          m1 = fmaxf(m1, fmaxf(sc[u][nt][1], sc[u][nt][3]));
        }
        raise = raise || m0 > limit[nt][0] || m1 > limit[nt][1];
      }
      float vs[U][2][NG];
#pragma unroll
      for (int a = 0; a < NG; ++a)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) vs[u][e][a] = q4_up<F16>(prm[u][e][NG + a] & 0xffffu);
      if (__any_sync(0xffffffffu, raise)) {
        // a score above the base by more than 8 raises it (weights <= 2^8)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
#pragma unroll
            for (int u = 1; u < U; ++u) mx = fmaxf(mx, fmaxf(sc[u][nt][e], sc[u][nt][e + 2]));
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
            const float old = limit[nt][e] == -INFINITY ? -INFINITY : base[nt][e];
            const float now = fmaxf(old, mx * hs[nt][e]);
            const float al = now == -INFINITY ? 1.f : ex2_approx(old - now);
            base[nt][e] = now == -INFINITY ? 0.f : now;
            limit[nt][e] = now == -INFINITY ? -INFINITY : __fdividef(now + kRescaleThreshold, hs[nt][e]);
            l_run[nt][e] *= al;
            const int ea = static_cast<int>(__float_as_uint(al) >> 23);
            // scales' exponents of the largest score's key, whose weight is 1 now
            uint32_t top = 0u;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const uint32_t es = (__float_as_uint(vs[u][r][0]) >> 23) | (__float_as_uint(vs[u][r][NG - 1]) >> 23) << 16;
                top = __vmaxu2(top, sc[u][nt][e + 2 * r] == mx ? es : 0u);
              }
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, s));
#pragma unroll
            for (int a = 0; a < NG; ++a) {
              vz[nt][a][e] *= al;
              // the unit falls with the weights it stands for, by al's power of two; the rest of al is the sums'.
              // With the first keys it comes to 2^-8 to 2^-9 of the largest score's s
              const int ev = static_cast<int>(__float_as_uint(vinv[nt][a][e]) >> 23);
              const int es = static_cast<int>(a == 0 ? top & 0xffffu : top >> 16);
              const int to = max(1, min(old < now && old == -INFINITY ? 262 - es : ev + 127 - ea, kDq4UnitTop));
              const float f = ea == 0 ? 0.f : __uint_as_float(__float_as_uint(al) + (static_cast<uint32_t>(to - ev) << 23));
              vinv[nt][a][e] = __uint_as_float(static_cast<uint32_t>(to) << 23);
#pragma unroll
              for (int i2 = 0; i2 < 4; ++i2) {
                o[nt][a][i2][e] *= f;
                o[nt][a][i2][e + 2] *= f;
              }
            }
          }
      }
      float pr[U][NT][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // pairs of heads in packed arithmetic
          const float2 f = make_float2(hs[nt][0], hs[nt][1]), b = make_float2(-base[nt][0], -base[nt][1]);
          // (the product rounded as in the base: the largest score's weight is 1 however large it is)
          const float2 x0 = __fadd2_rn(__fmul2_rn(make_float2(sc[u][nt][0], sc[u][nt][1]), f), b);
          const float2 x1 = __fadd2_rn(__fmul2_rn(make_float2(sc[u][nt][2], sc[u][nt][3]), f), b);
          pr[u][nt][0] = ex2_approx(x0.x);
          pr[u][nt][1] = ex2_approx(x0.y);
          pr[u][nt][2] = ex2_approx(x1.x);
          pr[u][nt][3] = ex2_approx(x1.y);
          const float2 l = __fadd2_rn(make_float2(l_run[nt][0], l_run[nt][1]),
                                      __fadd2_rn(make_float2(pr[u][nt][0], pr[u][nt][1]), make_float2(pr[u][nt][2], pr[u][nt][3])));
          l_run[nt][0] = l.x;
          l_run[nt][1] = l.y;
        }
      // ---- the weights of the second product, p_j s_j in units of 1 / vinv
      uint32_t bp[U][NT][NG][2];
      uint32_t br[REST ? U : 1][NT][NG][2];  // what that rounding leaves
      uint32_t largest;
      auto weigh = [&] {
        largest = 0u;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int a = 0; a < NG; ++a) {
              const float2 unit = make_float2(vinv[nt][a][0], vinv[nt][a][1]);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 y = __fmul2_rn(__fmul2_rn(make_float2(pr[u][nt][2 * e], pr[u][nt][2 * e + 1]), unit),
                                            make_float2(vs[u][e][a], vs[u][e][a]));
                bp[u][nt][a][e] = pack2<true>(y.x, y.y);
                if constexpr (REST) {
                  const float2 h = q4_up2<true>(bp[u][nt][a][e]);
                  br[u][nt][a][e] = pack2<true>(y.x - h.x, y.y - h.y);
                }
                largest = q4_max2_f16(largest, bp[u][nt][a][e]);
              }
            }
      };
      weigh();
      // one at 2^15 or above raises its head's and group's unit, so that the largest is in [2^8, 2^9)
      if (__any_sync(0xffffffffu, ((largest + 0x08000800u) & 0x80008000u) != 0u)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int a = 0; a < NG; ++a) {
            uint32_t top = 0u;  // exponents of 2^-16 times the largest, of both heads (p is at most 2^8, a scale 2^124)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = 0.f;
#pragma unroll
              for (int u = 0; u < U; ++u)
                mx = fmaxf(mx, fmaxf(pr[u][nt][e] * (vs[u][0][a] * 0x1p-16f), pr[u][nt][e + 2] * (vs[u][1][a] * 0x1p-16f)));
              top |= (__float_as_uint(mx) >> 23) << (16 * e);
            }
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, s));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int em = static_cast<int>(e == 0 ? top & 0xffffu : top >> 16);
              const int ev = static_cast<int>(__float_as_uint(vinv[nt][a][e]) >> 23);
              const int to = em + ev >= 253 ? max(246 - em, 1) : ev;  // (2^16 mx vinv >= 2^15)
              const float f = __uint_as_float(static_cast<uint32_t>(max(127 + to - ev, 0)) << 23);
              vinv[nt][a][e] = __uint_as_float(static_cast<uint32_t>(to) << 23);
#pragma unroll
              for (int i2 = 0; i2 < 4; ++i2) {
                o[nt][a][i2][e] *= f;
                o[nt][a][i2][e + 2] *= f;
              }
            }
          }
        weigh();
      }
      // ---- O += V^T P per group
#pragma unroll
      for (int a = 0; a < NG; ++a)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint4 vw = *reinterpret_cast<const uint4*>(step + u * L::kTileBytes + L::kVOff + (a * 8 + g) * 64 + t * 16);
          const uint32_t vwords[4] = {vw.x, vw.y, vw.z, vw.w};
          const float z0 = fmaf(8.f, vs[u][0][a], q4_up<F16>(prm[u][0][NG + a] >> 16));
          const float z1 = fmaf(8.f, vs[u][1][a], q4_up<F16>(prm[u][1][NG + a] >> 16));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 p0 = make_float2(pr[u][nt][0], pr[u][nt][1]), p1 = make_float2(pr[u][nt][2], pr[u][nt][3]);
            const float2 zv = __ffma2_rn(p0, make_float2(z0, z0), __ffma2_rn(p1, make_float2(z1, z1), make_float2(vz[nt][a][0], vz[nt][a][1])));
            vz[nt][a][0] = zv.x;
            vz[nt][a][1] = zv.y;
            bp[u][nt][a][0] = movmatrix_t(bp[u][nt][a][0]);
            bp[u][nt][a][1] = movmatrix_t(bp[u][nt][a][1]);
            if constexpr (REST) {
              br[u][nt][a][0] = movmatrix_t(br[u][nt][a][0]);
              br[u][nt][a][1] = movmatrix_t(br[u][nt][a][1]);
            }
          }
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            uint32_t fa[4];  // dims 2p (row g) and 2p+1 (row g+8) of tokens 4t, 4t+2 and 4t+1, 4t+3
            q4_pairs(vwords[i2], consts, fa);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<true>(o[nt][a][i2], fa, bp[u][nt][a][0], bp[u][nt][a][1]);
              if constexpr (REST) mma16816<true>(o[nt][a][i2], fa, br[u][nt][a][0], br[u][nt][a][1]);
            }
          }
        }
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- the result, or this piece's part of it: lane (g, t) holds dims 8 (8 a + g) .. + 7 of heads 2t, 2t + 1
    const bool whole = n == tiles;
    const int slot = f == f_begin ? 0 : 1;
    const long long part = (static_cast<long long>(me) * 2 + slot) * G;
#pragma unroll
    for (int s = 4; s < 32; s <<= 1)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], s);
#pragma unroll
          for (int a = 0; a < NG; ++a) vz[nt][a][e] += __shfl_xor_sync(0xffffffffu, vz[nt][a][e], s);
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float l = l_run[nt][e];
        const int h = nt * 8 + 2 * t + e;
        if (h >= G) continue;
        const float inv = whole ? (l == 0.f ? 0.f : __fdividef(1.f, l)) : 1.f;
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          float v[8];
          const float unit = __uint_as_float((254u << 23) - __float_as_uint(vinv[nt][a][e]));  // 1 / vinv
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            v[2 * i2] = fmaf(o[nt][a][i2][e], unit, vz[nt][a][e]) * inv;
            v[2 * i2 + 1] = fmaf(o[nt][a][i2][e + 2], unit, vz[nt][a][e]) * inv;
          }
          const int d = 8 * (8 * a + g);
          if (whole) {
            dq4_store8(p, row, kvh * G + h, D, d, v);
          } else {
            float4* dst = reinterpret_cast<float4*>(p.part_o + (part + h) * D + d);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
        if (g == 0) {
          if (!whole) {
            // no key yet: base -inf, but a NaN sum must show
            p.part_ml[part + h] = make_float2(l == 0.f ? -INFINITY : base[nt][e], l);
          } else if (p.lse != nullptr) {
            p.lse[(kvh * G + h) * p.lse_stride + row] = l == 0.f ? -INFINITY : (base[nt][e] + lg2_approx(l)) * 0.69314718055994530942f;
          }
        }
      }
    if (t0 == 0 && lane == 0) {
      int parts = 0;
      if (!whole) {
        const long long end = f - f_begin + tiles - 1;  // its last tile, from this piece's first
        parts = 1 + static_cast<int>(end <= INT_MAX && piece <= INT_MAX ? static_cast<uint32_t>(end) / static_cast<uint32_t>(piece)
                                                                         : end / piece);
      }
      p.desc[static_cast<long long>(row) * Hkv + kvh] = make_int4(me, slot, parts, 0);
    }
    f += n;
  }
  // ---- rows without keys (zeros, lse -inf) and padding rows have nothing to join; the last warps have least to do
  for (int r = kPieces - 1 - me; r < p.rows; r += kPieces) {
    const int n = dq4_len(p, r, req);
    if (n > 0) continue;
    if (n == 0) {
      for (int e = lane; e < p.num_heads * D; e += 32) dq4_store(p, r, e / D, D, e % D, 0.f);
      if (p.lse != nullptr)
        for (int h = lane; h < p.num_heads; h += 32) p.lse[h * p.lse_stride + r] = -INFINITY;
    }
    for (int h = lane; h < Hkv; h += 32) p.desc[static_cast<long long>(r) * Hkv + h] = make_int4(0, 0, 0, 0);
  }
}

// ---- joins of a (row, KV head)'s parts; sums run in a fixed order
// That pair's parts, and whether there are any.
__device__ __forceinline__ bool dq4_parts(const DecodeQ4Params& p, int pair, int4& desc) {
  desc = p.desc[pair];
  return desc.z > 0 && desc.x >= 0 && desc.x + desc.z <= kDq4MaxPieces && (desc.y & ~1) == 0;
}
__device__ __forceinline__ long long dq4_part(const int4& desc, int i, int G, int h) {
  return (static_cast<long long>(desc.x + i) * 2 + (i == 0 ? desc.y : 0)) * G + h;
}
__device__ __forceinline__ float dq4_lse(float M, float ls) {
  return ls == 0.f ? -INFINITY : (M + lg2_approx(ls)) * 0.69314718055994530942f;
}

// A warp takes a head of the pair and all its parts.
template <int D>
__device__ __forceinline__ void dq4_join_few(const DecodeQ4Params& p, const int4 desc, int pair, int h) {
  constexpr int V = D / 32;  // neighbouring dims of a lane
  const int G = p.group, lane = threadIdx.x & 31;
  const int row = pair / p.num_kv_heads, kvh = pair % p.num_kv_heads;
  float M = -INFINITY;
  for (int i = lane; i < desc.z; i += 32) M = fmaxf(M, p.part_ml[dq4_part(desc, i, G, h)].x);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
  float acc[V], ls = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  if (M != -INFINITY) {
#pragma unroll 8
    for (int i = 0; i < desc.z; ++i) {
      const long long at = dq4_part(desc, i, G, h);
      const float2 ml = p.part_ml[at];
      const float x = ex2_approx(ml.x - M);
      ls = fmaf(x, ml.y, ls);
      const float* part = p.part_o + at * D + V * lane;
      if constexpr (V == 4) {
        const float4 o = *reinterpret_cast<const float4*>(part);
        acc[0] = fmaf(x, o.x, acc[0]);
        acc[1] = fmaf(x, o.y, acc[1]);
        acc[2] = fmaf(x, o.z, acc[2]);
        acc[3] = fmaf(x, o.w, acc[3]);
      } else {
        const float2 o = *reinterpret_cast<const float2*>(part);
        acc[0] = fmaf(x, o.x, acc[0]);
        acc[1] = fmaf(x, o.y, acc[1]);
      }
    }
  }
  const int head = kvh * G + h;
#pragma unroll
  for (int v = 0; v < V; ++v) dq4_store(p, row, head, D, V * lane + v, ls == 0.f ? 0.f : acc[v] / ls);
  if (lane == 0 && p.lse != nullptr) p.lse[head * p.lse_stride + row] = dq4_lse(M, ls);
}

// A block takes 32 V dims (blockIdx.z) of one head of a pair and its warps share the parts, P each at a
// time, all loaded before the first weight is known.  The parts were just written by other SMs, so the
// reads' latency is what this costs.
//   Few pairs, each of many parts (LOOK false): a block a pair (blockIdx.x) and head (blockIdx.y).
//   Many pairs, most of few parts (LOOK): the first blocks look through a share of the pairs, one head each,
// for those of more parts than a warp should take alone (one long row among many short ones: 440 parts to a
// pair at 128k keys); the warps of the blocks after them take a head of a pair each.  Measured (28/4 heads,
// D 128, the whole call): one row of 131072 keys among 31 of 300 takes 95 us with a warp for every head and
// pair, 38 us so.
template <int D, int V, int P, bool LOOK>
__global__ void __launch_bounds__(LOOK ? kDq4JoinThreads : kDq4JoinWarps * 32, LOOK ? 4 : 1)
    decode_q4_join_kernel(const __grid_constant__ DecodeQ4Params p) {
  __shared__ float weight[kDq4MaxPieces], red[kDq4JoinWarps], sum[kDq4JoinWarps], so[kDq4JoinWarps][32 * V];
  __shared__ int found, list[LOOK ? kDq4MaxLong : 1];
  ptx::chain_wait();
  ptx::chain_next();
  const int G = p.group, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int h = LOOK ? blockIdx.x % G : blockIdx.y;
  int4 desc;
  if constexpr (LOOK) {
    const int pairs = p.rows * p.num_kv_heads, lookers = kDq4Lookers * G;
    if (blockIdx.x >= lookers) {
      const long long at = static_cast<long long>(blockIdx.x - lookers) * warps + warp;
      const int pair = static_cast<int>(at / G);
      if (pair < pairs && dq4_parts(p, pair, desc) && desc.z <= kDq4FewParts) dq4_join_few<D>(p, desc, pair, static_cast<int>(at % G));
      return;
    }
    if (tid == 0) found = 0;
    __syncthreads();
    for (int i = blockIdx.x / G + kDq4Lookers * tid; i < pairs; i += kDq4Lookers * blockDim.x)
      if (p.desc[i].z > kDq4FewParts) {
        const int at = atomicAdd(&found, 1);  // in any order: each is joined by itself
        if (at < kDq4MaxLong) list[at] = i;
      }
    __syncthreads();
  }
  const int count = LOOK ? min(found, kDq4MaxLong) : 1;
  for (int k = 0; k < count; ++k) {
    const int pair = LOOK ? list[k] : static_cast<int>(blockIdx.x);
    if (!dq4_parts(p, pair, desc)) continue;
    const float* const part = p.part_o + (blockIdx.z * 32 + lane) * V;
    float o[P][V];
    auto load = [&](int i0) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int i = i0 + j * warps;
#pragma unroll
        for (int v = 0; v < V; ++v) o[j][v] = 0.f;
        if (i >= desc.z) continue;
        const float* at = part + dq4_part(desc, i, G, h) * D;
        if constexpr (V == 4) {
          const float4 x = *reinterpret_cast<const float4*>(at);
          o[j][0] = x.x; o[j][1] = x.y; o[j][2] = x.z; o[j][3] = x.w;
        } else if constexpr (V == 2) {
          const float2 x = *reinterpret_cast<const float2*>(at);
          o[j][0] = x.x; o[j][1] = x.y;
        } else {
          o[j][0] = *at;
        }
      }
    };
    load(warp);
    float M = -INFINITY;
    for (int i = tid; i < desc.z; i += blockDim.x) M = fmaxf(M, p.part_ml[dq4_part(desc, i, G, h)].x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
    if (lane == 0) red[warp] = M;
    __syncthreads();
    M = red[0];
    for (int w = 1; w < warps; ++w) M = fmaxf(M, red[w]);
    const float base = M == -INFINITY ? 0.f : M;
    float ls = 0.f;
    for (int i = tid; i < desc.z; i += blockDim.x) {
      const float2 ml = p.part_ml[dq4_part(desc, i, G, h)];
      const float x = ex2_approx(ml.x - base);
      weight[i] = x;
      ls = fmaf(x, ml.y, ls);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, s);
    if (lane == 0) sum[warp] = ls;
    __syncthreads();
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    for (int i0 = warp; i0 < desc.z; i0 += P * warps) {
      if (i0 != warp) load(i0);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (i0 + j * warps >= desc.z) break;
        const float x = weight[i0 + j * warps];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = fmaf(x, o[j][v], acc[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) so[warp][lane * V + v] = acc[v];
    __syncthreads();
    const int row = pair / p.num_kv_heads, head = pair % p.num_kv_heads * G + h;
    ls = 0.f;
    for (int w = 0; w < warps; ++w) ls += sum[w];
    for (int d = tid; d < 32 * V; d += blockDim.x) {
      float v = 0.f;
      for (int w = 0; w < warps; ++w) v += so[w][d];
      dq4_store(p, row, head, D, blockIdx.z * 32 * V + d, ls == 0.f ? 0.f : v / ls);
    }
    if (tid == 0 && blockIdx.z == 0 && p.lse != nullptr) p.lse[head * p.lse_stride + row] = dq4_lse(M, ls);
    if constexpr (LOOK) __syncthreads();
  }
}

}  // namespace hcp
