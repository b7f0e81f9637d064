// One engine step's cache plan, built on the GPU from the requests' lengths.
//
// For request i holding c_i = context_lens[i] tokens and getting n_i new ones,
// with block size bs and table width W (negative lengths count as 0):
//   have_i  = ceil(c_i / bs)
//   need_i  = max(0, min(W, ceil((c_i + n_i) / bs)) - have_i)
//   first_i = free_head + sum_{j<i} need_j
//   block_table[i, have_i + k] = free_blocks[first_i + k], k < need_i
//                                (-1 past the end of the free list)
//   start_i = sum_{j<i} n_j
//   token t = start_i + u of request i: p = c_i + u, position pos_base_i + p,
//   slot block_table[i, p / bs] * bs + p % bs, visible keys p + 1.
//
// The data are a few hundred KB at most: a call costs its launch and one chain
// of dependent reads.  So it is one launch without anything between its
// blocks: each block sums all requests' lengths itself (256 threads, each a run
// of consecutive requests, then one scan of 256 pairs) and works on its share
// of the tokens and of the new table entries.  A token that falls into a new
// block reads its id from the free list and not from the table, which another
// block may be writing; the entries below have_i are only read.  Measured: 2.7 us for
// 8 requests, 4.7 us for 1024 (7.0 with 64-bit divisions by the block size), 4.0 us for 257
// requests with 20000 token rows.
#pragma once

#include <climits>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace hcp {

constexpr int kPlanThreads = 256;

struct StepPlanParams {
  const int32_t* context_lens;
  const int32_t* new_lens;
  const int32_t* pos_base;     // may be null: 0
  int32_t* block_table;
  long long bt_stride;
  long long bt_width;
  const int32_t* free_blocks;
  long long num_free;
  const int32_t* free_head;
  int32_t* query_start;        // [R + 1]
  int32_t* seq_lens;           // [R]
  int64_t* positions;          // [T]
  int64_t* slot_mapping;       // [T]
  int32_t* token_req;          // [T]
  int32_t* kv_lens;            // [T]
  int32_t* free_head_out;      // [1]
  int32_t* missing;            // [1]
  int num_reqs;
  long long num_tokens;
  int block_size;
  int bs_shift;                // log2(block_size) when it is a power of two, else -1
};

// n / block_size for n >= 0 (a 64-bit division costs more than the rest of a request)
__device__ __forceinline__ long long plan_blocks(const StepPlanParams& p, long long n) {
  return p.bs_shift >= 0 ? n >> p.bs_shift : n / p.block_size;
}

struct PlanReq {
  long long ctx, add, have, want, need;
};

__device__ __forceinline__ int plan_i32(long long v) {
  return static_cast<int>(v > INT_MAX ? INT_MAX : v);
}

__device__ __forceinline__ PlanReq plan_req(const StepPlanParams& p, int r) {
  PlanReq q;
  q.ctx = max(0, p.context_lens[r]);
  q.add = max(0, p.new_lens[r]);
  q.have = plan_blocks(p, q.ctx + p.block_size - 1);
  q.want = plan_blocks(p, q.ctx + q.add + p.block_size - 1);
  q.need = max(0ll, min(q.want, p.bt_width) - q.have);
  return q;
}

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(const StepPlanParams p) {
  // starts of every thread's run of requests: tokens, new blocks
  __shared__ long long s_tok[kPlanThreads + 1], s_blk[kPlanThreads + 1];
  __shared__ long long w_tok[kPlanThreads / 32], w_blk[kPlanThreads / 32], w_want[kPlanThreads / 32];
  ptx::chain_wait();
  ptx::chain_next();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (p.num_reqs + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(p.num_reqs, tid * run), r1 = min(p.num_reqs, r0 + run);
  long long tok = 0, blk = 0, wanted = 0;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    const PlanReq q = plan_req(p, r);
    tok += q.add;
    blk += q.need;
    wanted += q.want - q.have;
  }
  long long it = tok, ib = blk;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, it, s), b = __shfl_up_sync(0xffffffffu, ib, s);
    if (lane >= s) {
      it += a;
      ib += b;
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) wanted += __shfl_xor_sync(0xffffffffu, wanted, s);
  if (lane == 31) {
    w_tok[warp] = it;
    w_blk[warp] = ib;
    w_want[warp] = wanted;
  }
  __syncthreads();
  long long bt = 0, bb = 0, total_want = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) {
      bt += w_tok[w];
      bb += w_blk[w];
    }
    total_want += w_want[w];
  }
  const long long my_tok = bt + it - tok, my_blk = bb + ib - blk;
  s_tok[tid] = my_tok;
  s_blk[tid] = my_blk;
  if (tid == kPlanThreads - 1) {
    s_tok[kPlanThreads] = my_tok + tok;
    s_blk[kPlanThreads] = my_blk + blk;
  }
  __syncthreads();
  const long long total_tok = s_tok[kPlanThreads], total_blk = s_blk[kPlanThreads];
  const long long head = min(max(0ll, static_cast<long long>(*p.free_head)), p.num_free);

  if (blockIdx.x == 0) {
    long long at = my_tok;
    for (int r = r0; r < r1; ++r) {
      const PlanReq q = plan_req(p, r);
      p.query_start[r] = plan_i32(at);
      p.seq_lens[r] = plan_i32(q.ctx + q.add);
      at += q.add;
    }
    if (tid == 0) {
      const long long end = min(head + total_blk, p.num_free);
      p.query_start[p.num_reqs] = plan_i32(total_tok);
      *p.free_head_out = plan_i32(end);
      *p.missing = plan_i32(total_want - (end - head));
    }
  }

  const long long step = static_cast<long long>(gridDim.x) * kPlanThreads;
  const long long first = static_cast<long long>(blockIdx.x) * kPlanThreads + tid;
  // new table entries
  for (long long e = first; e < total_blk; e += step) {
    int lo = 0, hi = kPlanThreads - 1;  // last run that starts at or before e
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_blk[mid] <= e) lo = mid; else hi = mid - 1;
    }
    int r = lo * run;
    long long base = s_blk[lo];
    PlanReq q = plan_req(p, r);
    while (e >= base + q.need) {
      base += q.need;
      q = plan_req(p, ++r);
    }
    const long long at = head + e;
    p.block_table[r * p.bt_stride + q.have + (e - base)] = at < p.num_free ? p.free_blocks[at] : -1;
  }
  // tokens
  for (long long t = first; t < p.num_tokens; t += step) {
    if (t >= total_tok) {  // padding
      p.positions[t] = -1;
      p.slot_mapping[t] = -1;
      p.token_req[t] = -1;
      p.kv_lens[t] = 0;
      continue;
    }
    int lo = 0, hi = kPlanThreads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_tok[mid] <= t) lo = mid; else hi = mid - 1;
    }
    int r = lo * run;
    long long base = s_tok[lo], blocks = s_blk[lo];
    PlanReq q = plan_req(p, r);
    while (t >= base + q.add) {
      base += q.add;
      blocks += q.need;
      q = plan_req(p, ++r);
    }
    const long long pos = q.ctx + (t - base);
    const long long idx = plan_blocks(p, pos);
    int page = -1;
    if (idx < p.bt_width) {
      if (idx < q.have) {
        page = p.block_table[r * p.bt_stride + idx];
      } else {
        const long long at = head + blocks + (idx - q.have);
        if (at < p.num_free) page = p.free_blocks[at];
      }
    }
    p.positions[t] = pos + (p.pos_base != nullptr ? p.pos_base[r] : 0);
    p.slot_mapping[t] = page >= 0 ? static_cast<long long>(page) * p.block_size + (pos - idx * p.block_size) : -1;
    p.token_req[t] = r;
    p.kv_lens[t] = plan_i32(pos + 1);
  }
}

}  // namespace hcp
