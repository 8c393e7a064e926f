// cache_plan.cuh — page lists and slot maps of a paged key/value cache, built
// on the GPU from the requests' lengths (attn_cache_plan).
//
// Three exclusive prefix sums over the requests decide everything: new tokens
// n_b, pages taken A_b and pages given back R_b.  The stack of free pages with
// the given-back pages on top is never written out whole: its k-th popped
// entry is index F + R - 1 - k, read from free_pages below F and from the
// shrinking requests' table rows above.  Reads touch free_pages[0, F), table
// entries that exist and entries given back; writes touch free_pages[F, ..)
// and the new entries of growing rows: disjoint, so the blocks need no order
// between them, except for lengths and free_count, which may be updated in
// place: one cluster barrier separates their reads from their writes.
//
// A step of latency: one launch of one cluster of 1 to 8 blocks (each repeats
// the scan of at most 8192 requests and writes a share of the outputs).  64
// decoding requests 3.8 us, 500 requests with 65536 prompt tokens 11.9.
#pragma once

#include <cooperative_groups.h>

#include <cstdint>

#include "../../include/attn_rt.h"

namespace cache_plan {

constexpr int kMaxRequests = 8192;
constexpr int kMaxWarps = 32;
constexpr int kRun = 4;  // tokens that a thread takes at once

struct Params {
  int B, W, page_shift;
  int num_pages, tokens;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* targets;
  int32_t* table;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lengths_out;
  int32_t* free_count_out;
  int32_t* starts;
  int32_t* positions;
  int64_t* slots;
  int32_t* status;
};

struct Sums {
  int64_t tokens;
  int grown, dropped;
};

__device__ __forceinline__ Sums warp_scan(Sums v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, v.tokens, d);
    const int g = __shfl_up_sync(0xffffffffu, v.grown, d);
    const int r = __shfl_up_sync(0xffffffffu, v.dropped, d);
    if (lane >= d) {
      v.tokens += t;
      v.grown += g;
      v.dropped += r;
    }
  }
  return v;
}

// The request whose span [pre[b], pre[b+1]) holds i < pre[B].
__device__ __forceinline__ int owner(const int* pre, int B, int i) {
  int lo = 0, hi = B - 1;  // first b with pre[b + 1] > i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid + 1] > i) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(1024) plan_kernel(const Params p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int sm[];
  int* const held = sm;                   // [B]
  int* const tok_pre = held + p.B;        // [B + 1]
  int* const grow_pre = tok_pre + p.B + 1;
  int* const drop_pre = grow_pre + p.B + 1;
  int* const keeps = drop_pre + p.B + 1;  // [B] pages after the call
  __shared__ Sums warp_sums[kMaxWarps];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int threads = blockDim.x, warps = threads >> 5;
  const int F = *p.free_count;
  const int round_up = (1 << p.page_shift) - 1;
  const int most = p.W << p.page_shift;  // < 2^31: checked by the host
  bool bad = F < 0 || F > p.num_pages, wide = false;
  Sums run{0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += threads) {
    const int b = b0 + tid;
    Sums v{0, 0, 0};
    if (b < p.B) {
      int L = p.lengths[b], G = p.targets[b];
      held[b] = L;  // as it came: repeated in lengths_out if the call is refused
      if (L < 0 || L > most || G < 0) {
        bad = true;
        L = G = 0;
      } else if (G > most) {
        wide = true;
        G = L;
      }
      const int old_pages = (L + round_up) >> p.page_shift;
      const int new_pages = (G + round_up) >> p.page_shift;
      keeps[b] = new_pages;
      v.tokens = max(0, G - L);
      v.grown = max(0, new_pages - old_pages);
      v.dropped = max(0, old_pages - new_pages);
    }
    const Sums inc = warp_scan(v, lane);
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      const Sums s = warp_scan(lane < warps ? warp_sums[lane] : Sums{0, 0, 0}, lane);
      if (lane < warps) warp_sums[lane] = s;
    }
    __syncthreads();
    Sums before = run;
    if (warp > 0) {
      const Sums s = warp_sums[warp - 1];
      before.tokens += s.tokens, before.grown += s.grown, before.dropped += s.dropped;
    }
    const Sums all = warp_sums[warps - 1];
    run.tokens += all.tokens, run.grown += all.grown, run.dropped += all.dropped;
    if (b < p.B) {
      // Saturated: a total past `tokens` refuses the whole call below.
      tok_pre[b] = static_cast<int>(min(before.tokens + inc.tokens - v.tokens, int64_t{0x7fffffff}));
      grow_pre[b] = before.grown + inc.grown - v.grown;
      drop_pre[b] = before.dropped + inc.dropped - v.dropped;
    }
    __syncthreads();
  }
  bad = __syncthreads_or(bad);
  wide = __syncthreads_or(wide);
  const int A = run.grown, R = run.dropped;
  bad = bad || R > p.num_pages - F;  // more pages come back than ever went out
  const bool small = wide || A > F + R || run.tokens > p.tokens;
  const bool ok = !bad && !small;
  const int total = ok ? static_cast<int>(run.tokens) : 0;
  if (tid == 0) {
    tok_pre[p.B] = static_cast<int>(min(run.tokens, int64_t{0x7fffffff}));
    grow_pre[p.B] = A;
    drop_pre[p.B] = R;
  }
  // Every block has read lengths and free_count (and its own shared arrays
  // are complete) before one of them is written.
  cluster.sync();
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t step = threads * static_cast<int>(cluster.num_blocks());  // past 2^31 a step may lead
  const int first = rank * threads + tid;

  // Index x of the given-back pages: a table entry past its request's new end.
  auto given_back = [&](int x) {
    const int b = owner(drop_pre, p.B, x);
    return p.table[b * p.table_stride + keeps[b] + (x - drop_pre[b])];
  };
  // k-th page taken from the stack.
  auto popped = [&](int k) {
    const int i = F + R - 1 - k;
    return i < F ? p.free_pages[i] : given_back(i - F);
  };

  // Runs of consecutive tokens: one search for the request, one page id for
  // the tokens that share it, 16-byte stores.
  const int per = p.tokens > step ? kRun : 1;
  const bool aligned = per == kRun && (reinterpret_cast<uintptr_t>(p.slots) & 15u) == 0 &&
                    (reinterpret_cast<uintptr_t>(p.positions) & 15u) == 0;
  for (int64_t i0 = first * per; i0 < p.tokens; i0 += step * per) {
    int64_t slot[kRun];
    int position[kRun];
    int b = -1, page = 0, have = 0;
    const int32_t* row = nullptr;
#pragma unroll
    for (int x = 0; x < kRun; ++x) {
      slot[x] = -1, position[x] = 0;
      if (x >= per || i0 + x >= total) continue;
      const int i = static_cast<int>(i0) + x;
      const bool next = b < 0 || i >= tok_pre[b + 1];
      if (next) {
        if (b < 0) b = owner(tok_pre, p.B, i);
        else while (i >= tok_pre[b + 1]) ++b;
        have = (held[b] + round_up) >> p.page_shift;
        row = p.table + b * p.table_stride;
      }
      const int pos = held[b] + (i - tok_pre[b]);
      if (next || (pos & round_up) == 0) {
        const int j = pos >> p.page_shift;
        page = j < have ? row[j] : popped(grow_pre[b] + j - have);
      }
      position[x] = pos;
      slot[x] = (static_cast<int64_t>(page) << p.page_shift) + (pos & round_up);
    }
    if (aligned && i0 + kRun <= p.tokens) {
#pragma unroll
      for (int x = 0; x < kRun; x += 2)
        *reinterpret_cast<longlong2*>(p.slots + i0 + x) = make_longlong2(slot[x], slot[x + 1]);
      if (p.positions)
        *reinterpret_cast<int4*>(p.positions + i0) = make_int4(position[0], position[1], position[2], position[3]);
    } else {
#pragma unroll
      for (int x = 0; x < kRun; ++x) {
        if (x >= per || i0 + x >= p.tokens) continue;
        p.slots[i0 + x] = slot[x];
        if (p.positions) p.positions[i0 + x] = position[x];
      }
    }
  }
  for (int64_t b = first; b <= p.B; b += step) p.starts[b] = ok ? tok_pre[b] : 0;
  if (ok) {
    for (int64_t k = first; k < A; k += step) {
      const int b = owner(grow_pre, p.B, static_cast<int>(k));
      const int have = (held[b] + round_up) >> p.page_shift;
      p.table[b * p.table_stride + have + (k - grow_pre[b])] = popped(static_cast<int>(k));
    }
    for (int64_t i = int64_t{F} + first; i < F + R - A; i += step) p.free_pages[i] = given_back(static_cast<int>(i) - F);
  }
  // In place where the caller gave the same arrays.  targets may be
  // lengths_out too: then it holds what is written.
  for (int64_t b = first; b < p.B; b += step) p.lengths_out[b] = ok ? p.targets[b] : held[b];
  if (first == 0) {
    *p.free_count_out = ok ? F + R - A : F;
    if (!ok) atomicCAS(p.status, 0, bad ? ATTN_ERR_INVALID : ATTN_ERR_CAPACITY);
  }
}

}  // namespace cache_plan
