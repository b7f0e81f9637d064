// Single-token attention over the 4-bit paged cache (q4_cache.cuh) for B200.
//
// For every query row r with its request's pages and n = kv_lens[r] keys, per
// head h of KV head h / G:
//   o = sum_j softmax_j(scale q . k_j) v_j,   k_j, v_j = lo + s n  per 64 dims,
//   lse = log sum_j exp(scale q . k_j).
//
// Bound by HBM: 9/8 D bytes per key and KV head (K and V), against 2 G D
// products.  What has to be kept small is the work per byte.  So:
//   * the whole numbers n - 8 are the matrix operands, exact in fp16; scales and
//     lowest values are applied outside in 32 bits, per 64-dim group:
//       q . k  = sum_g  s_g (q_g . (n_g - 8)) + (lo_g + 8 s_g) sum(q_g)
//       o_g    = sum_j (p_j s_j) (n_j - 8)    + sum_j p_j (lo_j + 8 s_j)
//     (centred, the accumulated sums stay as small as the result's own terms);
//   * keys are the rows of the first product (16 keys x 8 heads) and dims those of
//     the second (16 dims x 8 heads), so a group of up to 8 query heads fills the
//     instruction's 8 columns instead of half of 16 rows;
//   * the tile layout gives every lane its fragments of both products in whole
//     16-byte pieces: no shared memory, no transposes; only the 8 x 8 blocks of P
//     are transposed between the products (movmatrix);
//   * q and p_j s_j enter the products in fp16, scaled by powers of two: q by its
//     head's largest element (no loss), p_j s_j by the largest scale met so far.
//     Rounding p_j s_j to 11 bits is off by at most 2^-11 of each key's term, and the
//     terms' weights sum to one: a quarter of what rounding the result to bf16 may be
//     off.  A second product for the rest costs 8 of the 16 matrix instructions and
//     a tenth of the issue slots of a kernel that is bound by them.
//
// Split: all rows' tiles of 16 keys, heads outermost in a row, form one line that
// the blocks cut into equal pieces, so any mix of lengths is even and nothing
// about the lengths has to be known on the host.  Every block sums the lengths
// itself.  A (row, KV head) that lies inside one piece is written to out by its
// block; one that is cut leaves a partial (O, m, l) per piece in the workspace, and
// a second kernel, already resident when the first ends, joins them in order.
// Inside a piece the four warps take the tiles in turn and join in shared memory.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "decode.cuh"
#include "q4_cache.cuh"

namespace hcp {

constexpr int kDq4Warps = 4;
constexpr int kDq4Threads = kDq4Warps * 32;
constexpr int kDq4CtasPerSm = 4;
constexpr int kDq4Sms = 148;
constexpr int kDq4Ctas = kDq4Sms * kDq4CtasPerSm;
constexpr int kDq4MinTiles = kDq4Warps;  // tiles of a piece at least: one a warp
constexpr int kDq4Stages = 4;            // tiles of a warp's ring: one read, the others in flight

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
  int4* desc;                 // [ctas] {row, kv head, slot of the first part, parts}; row -1: none
  float2* part_ml;            // [ctas][2][G] base (log2 units) and sum
  float* part_o;              // [ctas][2][G][D] sums to that base
  int rows;
  int num_heads;
  int num_kv_heads;
  int group;
  int block_size;
  int sub_shift;              // log2(tiles in a block)
  float scale_log2;
  int out_dt;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Whole numbers of a word's nibbles I and I+4 as a pair n - 8 in fp16, exact.  With a
// nibble in mantissa bits 0-3 of 1024 the value is 1024 + n, in bits 4-7 it is
// 1024 + 16 n: two pairs without a shift, the other two after one shift by 8.
__device__ __forceinline__ void q4_pairs(uint32_t w, uint32_t (&r)[4]) {
  const __half2 c0 = __floats2half2_rn(-1032.f, -1032.f), c1 = __floats2half2_rn(-72.f, -72.f);
  const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = i == 0 ? w : w >> 8;
    const uint32_t a = (v & 0x000f000fu) | 0x64006400u, b = (v & 0x00f000f0u) | 0x64006400u;
    const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&a), c0);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, c1);
    r[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
    r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// Tiles of a row (0 for a padding row or an empty one).
__device__ __forceinline__ int dq4_len(const DecodeQ4Params& p, int r, int& req) {
  req = p.token_req != nullptr ? p.token_req[r] : r;
  if (req < 0 || req >= p.bt_rows) return -1;
  const long long n = max(0, p.kv_lens[r]);
  return static_cast<int>(min(n, p.bt_width * p.block_size));
}
__device__ __forceinline__ int dq4_tiles(int len) { return len > 0 ? (len + 15) >> 4 : 0; }

template <int D, int NT>
struct Dq4Smem {
  static constexpr int kCols = 8 * NT;
  static constexpr int kPitch = D + 4;
  // the warps' rings of tiles; once a piece of a row is through, its sums
  static constexpr int kRing = kDq4Stages * Q4<D>::kTileBytes;
  union {
    alignas(16) uint8_t ring[kDq4Warps][kRing];
    float o[kDq4Warps][kCols][kPitch];
  };
  float m[kDq4Warps][kCols];
  float l[kDq4Warps][kCols];
  long long start[kDq4Threads + 1];
  long long wsum[kDq4Warps];
};

__device__ __forceinline__ void dq4_store(const DecodeQ4Params& p, long long row, int head, int D, int d, float v) {
  const long long i = row * p.out_row_stride + static_cast<long long>(head) * D + d;
  if (p.out_dt == HCP_F32) static_cast<float*>(p.out)[i] = v;
  else if (p.out_dt == HCP_F16) static_cast<__half*>(p.out)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}

template <int D, bool F16, int NT>
__global__ void __launch_bounds__(kDq4Threads, NT == 1 ? kDq4CtasPerSm : 2)
    decode_q4_kernel(const __grid_constant__ DecodeQ4Params p) {
  using L = Q4<D>;
  constexpr int NG = L::kGroups;
  constexpr int KW = 2 * NG;           // K words of a lane and token
  __shared__ Dq4Smem<D, NT> sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.group, Hkv = p.num_kv_heads;
  const uint32_t ring = ptx::smem_u32(sm.ring[warp]);

  // ---- the line of tiles: sums of every thread's run of rows
  const int run = (p.rows + kDq4Threads - 1) / kDq4Threads;
  long long mine = 0;
  for (int r = tid * run; r < min(p.rows, (tid + 1) * run); ++r) {
    int req;
    mine += dq4_tiles(dq4_len(p, r, req));
  }
  long long inc = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc, s);
    if (lane >= s) inc += a;
  }
  if (lane == 31) sm.wsum[warp] = inc;
  __syncthreads();
  long long before = 0;
  for (int w = 0; w < warp; ++w) before += sm.wsum[w];
  sm.start[tid] = before + inc - mine;
  if (tid == kDq4Threads - 1) sm.start[kDq4Threads] = before + inc;
  __syncthreads();
  const long long total = sm.start[kDq4Threads] * Hkv;
  const long long piece = max(static_cast<long long>(kDq4MinTiles), (total + gridDim.x - 1) / gridDim.x);
  long long f = blockIdx.x * piece;
  const long long f_end = min(total, f + piece);
  const long long f_begin = f;

  // rows without keys: zeros, lse -inf
  for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
    int req;
    if (dq4_len(p, r, req) != 0) continue;
    for (int e = tid; e < p.num_heads * D; e += kDq4Threads) dq4_store(p, r, e / D, D, e % D, 0.f);
    if (p.lse != nullptr)
      for (int h = tid; h < p.num_heads; h += kDq4Threads) p.lse[h * p.lse_stride + r] = -INFINITY;
  }
  int4 desc = make_int4(-1, 0, 0, 0);
  if (f < f_end) {
    // the row that holds tile f
    int lo = 0, hi = kDq4Threads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sm.start[mid] * Hkv <= f) lo = mid; else hi = mid - 1;
    }
    int row = lo * run, req;
    long long cum = sm.start[lo] * Hkv;
    int len = dq4_len(p, row, req);
    while (f < f_end) {
      while (row + 1 < p.rows && f >= cum + static_cast<long long>(dq4_tiles(len)) * Hkv) {
        cum += static_cast<long long>(dq4_tiles(len)) * Hkv;
        len = dq4_len(p, ++row, req);
      }
      if (f >= cum + static_cast<long long>(dq4_tiles(len)) * Hkv) break;  // lengths changed under the call
      const int tiles = dq4_tiles(len);
      const int kvh = static_cast<int>((f - cum) / tiles);
      const int t0 = static_cast<int>((f - cum) - static_cast<long long>(kvh) * tiles);
      const int n = static_cast<int>(min(static_cast<long long>(tiles - t0), f_end - f));

      // ---- Q fragments: columns are heads, lane's k index pairs (d, d + 4).  Each head is
      // scaled by a power of two to the top of fp16's range and rounded to it: exact down to
      // 2^-29 of its largest element for 11-bit elements.  The power goes into the head's factor.
      uint32_t qb[NT][2 * KW][2];
      float sq[NT][NG][2];  // sums of the scaled q over each group, heads 2t and 2t+1
      float hs[NT][2];      // score = hs * (scaled q . k), in log2 units
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int hc = nt * 8 + g;
        const uint16_t* qh = static_cast<const uint16_t*>(p.q) + row * p.q_row_stride +
                             static_cast<long long>(kvh * G + hc) * D;
        uint4 raw[KW];
        float top = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          raw[w] = make_uint4(0u, 0u, 0u, 0u);
          if (hc < G) raw[w] = *reinterpret_cast<const uint4*>(qh + 64 * (w >> 1) + 16 * t + 8 * (w & 1));
          float x[8];
          q4_unpack8<F16>(raw[w], x);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e with top * 2^e in [2^14, 2^15), e at most 126 (and 0 for an empty or infinite head)
        const int ex = static_cast<int>(__float_as_uint(top) >> 23);
        const int e = ex == 0 || ex == 255 ? 0 : min(126, 141 - ex);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        float part[NG];
#pragma unroll
        for (int a = 0; a < NG; ++a) part[a] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          float x[8];
          q4_unpack8<F16>(raw[w], x);
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
          sq[nt][a][0] = __shfl_sync(0xffffffffu, part[a], 8 * t);
          sq[nt][a][1] = __shfl_sync(0xffffffffu, part[a], 8 * t + 4);
        }
        const float down = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        hs[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        hs[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
      float o[NT][NG][4][4];
      float vz[NT][NG][2], l_run[NT][2];
      float base[NT][2];   // of the weights: the running maximum or up to 8 below it; -inf before the first key
      float limit[NT][2];  // the score / hs at which the base has to rise: (base + 8) / hs
      float vref[NG];      // powers of two: the sums o are in units of vref, 1 / vref multiplies V's scales
      float vinv[NG], vlim[NG];
#pragma unroll
      for (int a = 0; a < NG; ++a) {
        vref[a] = 0.f;
        vinv[a] = 0.f;
        vlim[a] = 0.f;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          vz[nt][a][0] = vz[nt][a][1] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][a][i][0] = o[nt][a][i][1] = o[nt][a][i][2] = o[nt][a][i][3] = 0.f;
        }
        limit[nt][0] = limit[nt][1] = base[nt][0] = base[nt][1] = -INFINITY;
        l_run[nt][0] = l_run[nt][1] = 0.f;
      }

      // ---- this warp's tiles t0 + warp + 4 i, i < cnt, through its ring
      const int cnt = n > warp ? (n - warp + kDq4Warps - 1) / kDq4Warps : 0;
      const int32_t* bt = p.block_table + req * p.bt_stride;
      const int sub_mask = (1 << p.sub_shift) - 1;
      const int first = t0 + warp;
      // page of tile 32 b + lane; the next 32 are on their way while these are used
      auto pages = [&](int b) {
        int v = -1;
        if (32 * b + lane < cnt) v = __ldg(bt + ((first + kDq4Warps * (32 * b + lane)) >> p.sub_shift));
        return v < p.num_blocks ? v : -1;
      };
      int page = pages(0), page_next = pages(1);
      uint32_t held = 0;  // bit k: the tile issued k before the last one has a page
      auto issue = [&](int i) {
        int blk = -1;
        if (i < cnt) {
          if (i > 0 && (i & 31) == 0) {
            page = page_next;
            page_next = pages((i >> 5) + 1);
          }
          blk = __shfl_sync(0xffffffffu, page, i & 31);
          if (blk >= 0) {
            const int ti = first + kDq4Warps * i;
            const uint8_t* src = p.cache + (((static_cast<long long>(blk) * Hkv + kvh) << p.sub_shift) + (ti & sub_mask)) *
                                               L::kTileBytes + 16 * lane;
            const uint32_t dst = ring + (i % kDq4Stages) * L::kTileBytes + 16 * lane;
#pragma unroll
            for (int c = 0; c < L::kTileBytes / 512; ++c) cp_async16(dst + 512 * c, src + 512 * c);
            constexpr int kRest = L::kTileBytes % 512 / 16;
            if (lane < kRest) cp_async16(dst + L::kTileBytes / 512 * 512, src + L::kTileBytes / 512 * 512);
          }
        }
        held = (held << 1) | (blk >= 0 ? 1u : 0u);
        cp_async_commit();
      };
#pragma unroll
      for (int i = 0; i < kDq4Stages - 1; ++i) issue(i);
      for (int i = 0; i < cnt; ++i) {
        cp_async_wait<kDq4Stages - 2>();
        __syncwarp();  // every lane's pieces are in, and the tile before is read by all
        issue(i + kDq4Stages - 1);
        if (((held >> (kDq4Stages - 1)) & 1u) == 0) continue;  // a page outside the cache holds no keys
        const uint8_t* tile = sm.ring[warp] + (i % kDq4Stages) * L::kTileBytes;
        const int left = len - 16 * (first + kDq4Warps * i);
        uint32_t prm[2][2 * NG];  // of tokens 2g, 2g+1: K (s, lo) of each group, then V
        uint32_t kw[2][KW];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint8_t* pp = tile + L::kParamOff + (2 * g + e) * L::kTokenParams;
          const uint8_t* kp = tile + (2 * g + e) * (D / 2) + t * (D / 8);
          if constexpr (NG == 2) {
            const uint4 v = *reinterpret_cast<const uint4*>(pp), u = *reinterpret_cast<const uint4*>(kp);
            prm[e][0] = v.x; prm[e][1] = v.y; prm[e][2] = v.z; prm[e][3] = v.w;
            kw[e][0] = u.x; kw[e][1] = u.y; kw[e][2] = u.z; kw[e][3] = u.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(pp), u = *reinterpret_cast<const uint2*>(kp);
            prm[e][0] = v.x; prm[e][1] = v.y;
            kw[e][0] = u.x; kw[e][1] = u.y;
          }
        }
        if (left < 16) {  // keys past the end: unwritten bytes may be anything
#pragma unroll
          for (int a = 0; a < 2 * NG; ++a) {
            prm[0][a] = 2 * g < left ? prm[0][a] : 0u;
            prm[1][a] = 2 * g + 1 < left ? prm[1][a] : 0u;
          }
        }
        // ---- scores: rows are tokens 2g (c0, c1) and 2g+1 (c2, c3)
        float sc[NT][4];
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t x[4], y[4];
            q4_pairs(kw[0][2 * a + e], x);
            q4_pairs(kw[1][2 * a + e], y);
            const uint32_t fa[4] = {x[0], y[0], x[1], y[1]}, fb[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<true>(acc[nt], fa, qb[nt][2 * (2 * a + e)][0], qb[nt][2 * (2 * a + e)][1]);
              mma16816<true>(acc[nt], fb, qb[nt][2 * (2 * a + e) + 1][0], qb[nt][2 * (2 * a + e) + 1][1]);
            }
          }
          const float s0 = q4_up<F16>(prm[0][a] & 0xffffu), z0 = fmaf(8.f, s0, q4_up<F16>(prm[0][a] >> 16));
          const float s1 = q4_up<F16>(prm[1][a] & 0xffffu), z1 = fmaf(8.f, s1, q4_up<F16>(prm[1][a] >> 16));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[nt][e] = fmaf(e < 2 ? z0 : z1, sq[nt][a][e & 1], fmaf(e < 2 ? s0 : s1, acc[nt][e], a == 0 ? 0.f : sc[nt][e]));
          }
        }
        if (left < 16) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[nt][e] = 2 * g + (e >> 1) < left ? sc[nt][e] : -INFINITY;
        }
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          raise = raise || fmaxf(sc[nt][0], sc[nt][2]) > limit[nt][0] || fmaxf(sc[nt][1], sc[nt][3]) > limit[nt][1];
        float vs[2][NG];
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          vs[0][a] = q4_up<F16>(prm[0][NG + a] & 0xffffu);
          vs[1][a] = q4_up<F16>(prm[1][NG + a] & 0xffffu);
          raise = raise || fmaxf(vs[0][a], vs[1][a]) > vlim[a];
        }
        if (__any_sync(0xffffffffu, raise)) {
          // a score above the base by more than 8 raises it (weights <= 2^8)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(sc[nt][e], sc[nt][e + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float now = fmaxf(base[nt][e], mx * hs[nt][e]);
              const float al = now == -INFINITY ? 1.f : ex2_approx(base[nt][e] - now);
              base[nt][e] = now;
              limit[nt][e] = now == -INFINITY ? -INFINITY : __fdividef(now + kRescaleThreshold, hs[nt][e]);
              l_run[nt][e] *= al;
#pragma unroll
              for (int a = 0; a < NG; ++a) {
                vz[nt][a][e] *= al;
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                  o[nt][a][i2][e] *= al;
                  o[nt][a][i2][e + 2] *= al;
                }
              }
            }
          // a scale above 2^7 vref raises vref: weight times scale stays below 2^15 in fp16
#pragma unroll
          for (int a = 0; a < NG; ++a) {
            float mx = fmaxf(vs[0][a], vs[1][a]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (mx > vlim[a]) {
              // 2^6 vref <= mx < 2^7 vref now (vref and 1 / vref stay normal numbers)
              const int ex = max(static_cast<int>(__float_as_uint(mx) >> 23) - 6, 1);
              const float now = __uint_as_float(static_cast<uint32_t>(ex) << 23);
              const float al = vref[a] * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
              vref[a] = now;
              vinv[a] = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
              vlim[a] = now * 128.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[nt][a][i2][e] *= al;
            }
          }
        }
        float pr[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float b0 = base[nt][0] == -INFINITY ? 0.f : base[nt][0], b1 = base[nt][1] == -INFINITY ? 0.f : base[nt][1];
          pr[nt][0] = ex2_approx(fmaf(sc[nt][0], hs[nt][0], -b0));
          pr[nt][1] = ex2_approx(fmaf(sc[nt][1], hs[nt][1], -b1));
          pr[nt][2] = ex2_approx(fmaf(sc[nt][2], hs[nt][0], -b0));
          pr[nt][3] = ex2_approx(fmaf(sc[nt][3], hs[nt][1], -b1));
          l_run[nt][0] += pr[nt][0] + pr[nt][2];
          l_run[nt][1] += pr[nt][1] + pr[nt][3];
        }
        // ---- O += V^T P per group
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          const uint4 vw = *reinterpret_cast<const uint4*>(tile + L::kVOff + (a * 8 + g) * 64 + t * 16);
          const uint32_t vwords[4] = {vw.x, vw.y, vw.z, vw.w};
          const float z0 = fmaf(8.f, vs[0][a], q4_up<F16>(prm[0][NG + a] >> 16));
          const float z1 = fmaf(8.f, vs[1][a], q4_up<F16>(prm[1][NG + a] >> 16));
          const float s0 = vs[0][a] * vinv[a], s1 = vs[1][a] * vinv[a];
          uint32_t bp[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            vz[nt][a][0] = fmaf(pr[nt][0], z0, fmaf(pr[nt][2], z1, vz[nt][a][0]));
            vz[nt][a][1] = fmaf(pr[nt][1], z0, fmaf(pr[nt][3], z1, vz[nt][a][1]));
            bp[nt][0] = movmatrix_t(pack2<true>(pr[nt][0] * s0, pr[nt][1] * s0));
            bp[nt][1] = movmatrix_t(pack2<true>(pr[nt][2] * s1, pr[nt][3] * s1));
          }
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            uint32_t fa[4];  // dims 2p (row g) and 2p+1 (row g+8) of tokens 4t, 4t+2 and 4t+1, 4t+3
            q4_pairs(vwords[i2], fa);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<true>(o[nt][a][i2], fa, bp[nt][0], bp[nt][1]);
          }
        }
      }
      cp_async_wait<0>();
      __syncthreads();  // the rings are read: their memory takes the sums

      // ---- join the warps: sums over the lanes' tokens first
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = l_run[nt][e];
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
          const int col = nt * 8 + 2 * t + e;
          if (g == 0) {
            sm.m[warp][col] = l != l ? 0.f : base[nt][e];  // a NaN sum must not hide behind an empty base
            sm.l[warp][col] = l;
          }
#pragma unroll
          for (int a = 0; a < NG; ++a) {
            float z = vz[nt][a][e];
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) z += __shfl_xor_sync(0xffffffffu, z, s);
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
              const float2 v = make_float2(fmaf(o[nt][a][i2][e], vref[a], z), fmaf(o[nt][a][i2][e + 2], vref[a], z));
              *reinterpret_cast<float2*>(&sm.o[warp][col][8 * (8 * a + g) + 2 * i2]) = v;
            }
          }
        }
      __syncthreads();
      const bool whole = n == tiles;
      const int slot = f == f_begin ? 0 : 1;
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + slot) * G;
      for (int e = tid; e < G * D; e += kDq4Threads) {
        const int h = e / D, d = e % D;
        float M = sm.m[0][h];
#pragma unroll
        for (int w = 1; w < kDq4Warps; ++w) M = fmaxf(M, sm.m[w][h]);
        float acc = 0.f, ls = 0.f;
        if (M != -INFINITY) {
#pragma unroll
          for (int w = 0; w < kDq4Warps; ++w) {
            const float x = ex2_approx(sm.m[w][h] - M);
            acc = fmaf(x, sm.o[w][h][d], acc);
            ls = fmaf(x, sm.l[w][h], ls);
          }
        }
        if (whole) {
          const int head = kvh * G + h;
          dq4_store(p, row, head, D, d, ls == 0.f ? 0.f : acc / ls);
          if (d == 0 && p.lse != nullptr)
            p.lse[head * p.lse_stride + row] = ls == 0.f ? -INFINITY : (M + lg2_approx(ls)) * 0.69314718055994530942f;
        } else {
          p.part_o[(part + h) * D + d] = acc;
          if (d == 0) p.part_ml[part + h] = make_float2(M, ls);
        }
      }
      if (!whole && t0 == 0) {
        const long long last = (f + tiles - 1) / piece;
        desc = make_int4(row, kvh, slot, static_cast<int>(last - blockIdx.x) + 1);
      }
      __syncthreads();
      f += n;
    }
  }
  if (tid == 0) p.desc[blockIdx.x] = desc;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Joins the parts of the (row, KV head) whose first part lies in block
// blockIdx.x, for head blockIdx.y of the group: parts in order, warps by turns.
template <int D>
__global__ void __launch_bounds__(128) decode_q4_join_kernel(const __grid_constant__ DecodeQ4Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 desc = p.desc[blockIdx.x];
  if (desc.x < 0) return;
  constexpr int V = D / 32;
  __shared__ float so[4][D], sml[4][2];
  const int G = p.group, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto index = [&](int i) {
    return (static_cast<long long>(blockIdx.x + i) * 2 + (i == 0 ? desc.z : 0)) * G + h;
  };
  float M = -INFINITY;
  for (int i = lane; i < desc.w; i += 32) M = fmaxf(M, p.part_ml[index(i)].x);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
  float acc[V], ls = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (M != -INFINITY) {
#pragma unroll 4
    for (int i = warp; i < desc.w; i += 4) {
      const long long at = index(i);
      const float2 ml = p.part_ml[at];
      const float x = ex2_approx(ml.x - M);
      ls = fmaf(x, ml.y, ls);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(x, p.part_o[at * D + v * 32 + lane], acc[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) so[warp][v * 32 + lane] = acc[v];
  if (lane == 0) sml[warp][0] = ls;
  __syncthreads();
  ls = sml[0][0] + sml[1][0] + sml[2][0] + sml[3][0];
  const int head = desc.y * G + h;
  for (int d = threadIdx.x; d < D; d += 128) {
    const float v = so[0][d] + so[1][d] + so[2][d] + so[3][d];
    dq4_store(p, desc.x, head, D, d, ls == 0.f ? 0.f : v / ls);
  }
  if (threadIdx.x == 0 && p.lse != nullptr)
    p.lse[head * p.lse_stride + desc.x] = ls == 0.f ? -INFINITY : (M + lg2_approx(ls)) * 0.69314718055994530942f;
}

}  // namespace hcp
