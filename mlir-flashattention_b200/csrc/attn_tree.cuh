// attn_tree.cuh — attention of new tokens over a paged cache (attn_tree_fwd).
//
// For token t of request b and q-head h (kv-head h / g):
//   O = sum_j softmax(scale * q . k_j) v_j
// over the cached keys j < lengths[b] and the request's new keys that the mask
// leaves visible, by the online recurrence with a running maximum m, sum l and
// accumulator in 32 bits.
//
// This header: what the kernels share - operands, the requests as the device
// arrays give them, the split of the work, and values that are no numbers.
// attn_tree_mma.cuh holds the kernel for few query rows and the join of its
// split items, attn_tree_tc.cuh those for many rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

#include "../../include/attn_rt.h"

namespace attn_tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr uint64_t kWaitLimitNs = 1000000000ull;  // 1 s per wait

struct Params {
  int B, T, Hq, Hkv, group;
  int W, num_pages, page_shift;
  int max_new;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  int64_t table_stride, mask_stride;
  int mask_align;  // bytes that every row of the mask is aligned to
  const void* q;
  const void* k_new;
  const void* v_new;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  const uint8_t* mask;
  const float* k_descale_heads;
  const float* v_descale_heads;
  float scale, k_descale, v_descale;
  int32_t* status;
};

struct Request {
  int held, first, count;  // cached tokens, first row and number of new tokens
};

// What the device arrays say of request b, cut to what can be read: a length
// past the table or rows past q would leave the buffers.  Plain loads, here and
// wherever a kernel reads what the one before it in the stream may write: these
// kernels begin before that one ends, so to them such memory is not constant,
// and a load through the read-only path might be moved above the wait.
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.held = p.lengths[b];
  r.first = p.starts[b];
  r.count = p.starts[b + 1] - r.first;
  const int most = p.W << p.page_shift;
  if (r.held < 0 || r.held > most || r.count < 0 || r.count > p.max_new || r.first < 0 ||
      r.first > p.T - r.count) {
    atomicCAS(p.status, 0, ATTN_ERR_INVALID);
    r.held = r.first = r.count = 0;
  }
  return r;
}

// ----------------------------------------------------------------- the work
// An item is one tile of query rows of one request and kv-head: row r of the
// request is its token r / group with the kv-head's q-head r % group, so that
// the heads that share keys share the tile.  Its units are tiles of keys: the
// cached ones in order, then the new ones it can see.  The units of all items,
// one after another, are cut into equal shares, one for each block (or half of
// a block), whatever the requests' lengths; a share may begin and end inside an
// item.  A block meets its share as pieces; one that is not a whole item goes
// to scratch, and the join (a second kernel) adds up the pieces of each cut
// item in order.
struct Split {
  int rows;        // query rows of a tile
  int keys_shift;  // cached keys of a tile, log2
  int new_shift;   // new keys of a tile, log2
};

struct Piece {
  int b, h, rt;       // request, kv-head, row tile
  int k0, k1, tiles;  // units [k0, k1) of the item's `tiles`
  int cached;         // how many of the item's tiles are cached keys
  Request r;
};

// The new-key tiles that row tile rt of a request sees.
__device__ __forceinline__ int new_tiles(const Params& p, const Split& s, const Request& r, int rt) {
  int keys = r.count;
  if (p.mask == nullptr) keys = min(keys, (rt * s.rows + s.rows - 1) / p.group + 1);
  return (keys + (1 << s.new_shift) - 1) >> s.new_shift;
}

__device__ __forceinline__ int cached_tiles(const Split& s, const Request& r) {
  return static_cast<int>((static_cast<uint32_t>(r.held) + (1u << s.keys_shift) - 1) >> s.keys_shift);  // may pass 2^31
}

__device__ __forceinline__ int row_tiles(const Params& p, const Split& s, const Request& r) {
  return static_cast<int>((static_cast<int64_t>(r.count) * p.group + s.rows - 1) / s.rows);
}

// Units of one kv-head of a request.
__device__ __forceinline__ int64_t head_units(const Params& p, const Split& s, const Request& r) {
  const int rts = row_tiles(p, s, r);
  if (rts == 0) return 0;
  int64_t u = static_cast<int64_t>(rts) * cached_tiles(s, r);
  if (p.mask || rts == 1) return u + static_cast<int64_t>(rts) * new_tiles(p, s, r, rts - 1);
  for (int rt = 0; rt < rts; ++rt) u += new_tiles(p, s, r, rt);
  return u;
}

// Where a block's share begins, found by the whole block (blockDim.x threads,
// a multiple of 32, at most 1024).  Up to 32 requests every warp finds it for
// itself, without a barrier: the step of latency that a small call can spare.
struct Share {
  int64_t lo, hi;  // units still to do
  int64_t off;     // units of request b before lo
  int64_t head;    // units of one of its kv-heads
  int b;           // request that holds unit lo
  Request r;
  int64_t total;   // units of all blocks with a share, and their number
  int blocks;
};

// Units [lo, hi) of block c of `blocks`.
__device__ __forceinline__ void share_bounds(int64_t total, int blocks, int c, int64_t& lo, int64_t& hi) {
  if (total < (int64_t{1} << 20) && blocks <= 2048) {  // products below 2^31: no 64-bit division
    const uint32_t t = static_cast<uint32_t>(total), n = static_cast<uint32_t>(blocks);
    lo = t * static_cast<uint32_t>(c) / n, hi = t * static_cast<uint32_t>(c + 1) / n;
  } else {
    lo = total * c / blocks, hi = total * (c + 1) / blocks;
  }
}

__device__ __forceinline__ int64_t scan_warp(int64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += t;
  }
  return v;
}

// TEAMS: shares of a block; a thread gets the share of `team`.  Shares are
// numbered TEAMS * block + team.
template <int TEAMS>
__device__ __forceinline__ Share find_share(const Params& p, const Split& s, int min_units, int team) {
  __shared__ int64_t warp_sum[32];
  __shared__ Share found[TEAMS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  auto blocks_for = [&](int64_t total) {
    return static_cast<int>(min(static_cast<int64_t>(gridDim.x) * TEAMS, (total + min_units - 1) / min_units));
  };
  if (p.B <= 32) {
    const int c = static_cast<int>(blockIdx.x) * TEAMS + team;
    Share r{};
    if (lane < p.B) {
      r.r = request(p, lane);
      r.head = head_units(p, s, r.r);
    }
    const int64_t units = r.head * p.Hkv, end = scan_warp(units, lane);
    r.total = __shfl_sync(0xffffffffu, end, 31);
    r.blocks = blocks_for(r.total);
    if (c < r.blocks) share_bounds(r.total, r.blocks, c, r.lo, r.hi);
    r.off = r.lo - (end - units);
    const unsigned has = __ballot_sync(0xffffffffu, r.off >= 0 && r.lo < end);
    const int src = has ? __ffs(has) - 1 : 0;
    r.b = src;
    r.off = __shfl_sync(0xffffffffu, r.off, src);
    r.head = __shfl_sync(0xffffffffu, r.head, src);
    r.r.held = __shfl_sync(0xffffffffu, r.r.held, src);
    r.r.first = __shfl_sync(0xffffffffu, r.r.first, src);
    r.r.count = __shfl_sync(0xffffffffu, r.r.count, src);
    return r;
  }
  // A thread sums requests tid, tid + threads, ..; with more requests than
  // threads a second pass finds the one that holds the share's first unit.
  const int chunks = (p.B + blockDim.x - 1) / blockDim.x;
  int64_t mine = 0, head = 0;
  Request r{};
  for (int b = tid; b < p.B; b += blockDim.x) {
    r = request(p, b);
    head = head_units(p, s, r);
    mine += head * p.Hkv;
  }
  int64_t inc = scan_warp(mine, lane);
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int64_t total = 0, before = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int blocks = blocks_for(total);
  int64_t lo[TEAMS], hi[TEAMS];
#pragma unroll
  for (int t = 0; t < TEAMS; ++t) {
    const int c = static_cast<int>(blockIdx.x) * TEAMS + t;
    lo[t] = hi[t] = -1;
    if (c < blocks) share_bounds(total, blocks, c, lo[t], hi[t]);
    else if (tid == 0) found[t] = Share{};
  }
  auto offer = [&](int b, int64_t end, int64_t units) {
#pragma unroll
    for (int t = 0; t < TEAMS; ++t)
      if (lo[t] >= 0 && end - units <= lo[t] && lo[t] < end)
        found[t] = Share{lo[t], hi[t], lo[t] - (end - units), head, b, r, total, blocks};
  };
  if (chunks == 1) {
    offer(tid, before + inc, mine);
  } else {
    int64_t run = 0;
    for (int ch = 0; ch < chunks; ++ch) {
      const int b = ch * blockDim.x + tid;
      head = 0;
      if (b < p.B) {
        r = request(p, b);
        head = head_units(p, s, r);
      }
      inc = scan_warp(head * p.Hkv, lane);
      __syncthreads();
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      int64_t pre = run;
      for (int w = 0; w < warps; ++w) {
        if (w < warp) pre += warp_sum[w];
        run += warp_sum[w];
      }
      offer(b, pre + inc, head * p.Hkv);
    }
  }
  __syncthreads();
  return found[team];
}

// The number of the share that holds unit u.
__device__ __forceinline__ int share_of(const Share& sh, int64_t u) {
  return static_cast<int>(((u + 1) * sh.blocks - 1) / sh.total);
}

// The next piece of a share; moves past it.  False at its end.
__device__ __forceinline__ bool next_piece(const Params& p, const Split& s, Share& sh, Piece& out) {
  if (sh.lo >= sh.hi) return false;
  while (sh.off >= sh.head * p.Hkv) {
    sh.off -= sh.head * p.Hkv;
    if (++sh.b >= p.B) return false;  // lengths changed under the call
    sh.r = request(p, sh.b);
    sh.head = head_units(p, s, sh.r);
  }
  const Request& r = sh.r;
  int64_t off = sh.off;
  out.b = sh.b;
  out.r = r;
  out.h = 0;
  if (off >= sh.head) {
    out.h = (off | sh.head) >> 31 ? static_cast<int>(off / sh.head)
                                  : static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(sh.head));
    off -= out.h * sh.head;
  }
  out.cached = cached_tiles(s, r);
  const int rts = row_tiles(p, s, r);
  out.rt = 0;
  if (p.mask || rts == 1) {
    out.tiles = out.cached + new_tiles(p, s, r, rts - 1);
    if (rts > 1) {
      out.rt = static_cast<int>(off / out.tiles);
      off -= static_cast<int64_t>(out.rt) * out.tiles;
    }
  } else {
    for (;; ++out.rt) {
      out.tiles = out.cached + new_tiles(p, s, r, out.rt);
      if (off < out.tiles) break;
      off -= out.tiles;
    }
  }
  out.k0 = static_cast<int>(off);
  out.k1 = static_cast<int>(min(static_cast<int64_t>(out.tiles), off + (sh.hi - sh.lo)));
  sh.lo += out.k1 - out.k0;
  sh.off += out.k1 - out.k0;
  return true;
}

// Scratch of the pieces that are not whole items: share c's first piece goes
// to slot 2 c, its last to 2 c + 1.  The share that holds an item's first
// piece leaves what the join needs to know.
struct alignas(32) Record {
  int pieces;  // 0: no cut item begins in this share
  int slot;    // of the first piece; the others are the first ones of the shares that follow
  int first;   // first row of q of the request
  int row;     // first query row of the item in the request
  int rows;
  int h;
  int held, count;  // of the request
};

struct Scratch {
  Record* record;  // [shares]
  float* m;        // [2 shares][rows] running maximum, log2 units
  float* l;        // [2 shares][rows]
  float4* o;       // [2 shares], in the kernel's own order, relative to m, not divided by l
};

// Of share c, which has already moved past the piece.
__device__ __forceinline__ Record make_record(const Params& p, const Split& s, const Share& sh, const Piece& pc, int c,
                                              int slot) {
  Record r;
  const int64_t end = sh.lo + (pc.tiles - pc.k1);  // the item's end
  r.pieces = share_of(sh, end - 1) - c + 1;
  r.slot = slot;
  r.first = pc.r.first;
  r.row = pc.rt * s.rows;
  r.rows = static_cast<int>(min(static_cast<int64_t>(s.rows), static_cast<int64_t>(pc.r.count) * p.group -
                                                                  static_cast<int64_t>(pc.rt) * s.rows));
  r.h = pc.h;
  r.held = pc.r.held;
  r.count = pc.r.count;
  return r;
}

// What a row's sum of values is divided by, as a factor.  The sum of weights is
// 0 where every score was -inf: 0 for a row that sees no key, else 0 / 0.  (A
// sum that is not a number passes through, and the maximum with it stays -inf
// if all scores were none: pieces are joined relative to base_of.)
__device__ __forceinline__ float over(const Params& p, float sum, int held, int first, int count, int token) {
  if (sum != 0.f) return 1.f / sum;
  bool sees = held > 0 || p.mask == nullptr;
  if (!sees) {
    const uint8_t* const row = p.mask + static_cast<int64_t>(first + token) * p.mask_stride;
#pragma unroll 1
    for (int j = 0; j < count && !sees; ++j) sees = row[j] == 0;
  }
  return sees ? __int_as_float(0x7fc00000) : 0.f;
}

// What weights are taken relative to: a maximum of -inf stands for no key yet.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// A weight of 0 hides a key whose value is infinite or not a number no better
// than 0 * inf does.  Every row sees all cached keys, so this can only happen
// among a request's new ones, and only where a row may be hidden from one.
// There the attention reads a copy of the new values in which such values are
// 0 (clean_values), and in the end the rows that do see them get them back,
// where they decide the sum whatever their weights (whole_values).  Two small
// launches, 8 us of a call and a copy of V (64 drafted tokens for each of 8
// requests with 16384 keys: 114 -> 122 us; 2048 for each of 2: 470 -> 484); in the
// attention's own loops, whose registers are all taken, the same cost 9 to 120 us.
constexpr int kValueThreads = 256;

// odd[block]: whether the block met such a value.
template <typename T, int D>
__global__ void __launch_bounds__(kValueThreads)
    clean_values(const __grid_constant__ Params p, uint4* out, int* odd) {
  constexpr uint32_t kExponent = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
  constexpr int kPacks = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t live = p.starts[p.B];  // rows behind them may hold anything
  const int64_t n = static_cast<int64_t>(p.T) * p.Hkv * kPacks;
  uint32_t met = 0;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kValueThreads) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kValueThreads) {
    const int64_t row = i / kPacks;
    const T* const v = static_cast<const T*>(p.v_new) + row / p.Hkv * p.v_st + row % p.Hkv * p.v_sh;
    uint4 w = reinterpret_cast<const uint4*>(v)[i % kPacks];
    uint32_t* const x = &w.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t m = __vcmpeq2(x[k] & kExponent, kExponent);
      x[k] &= ~m;
      if (row / p.Hkv < live) met |= m;
    }
    out[i] = w;
  }
  const int any = __syncthreads_or(met != 0);
  if (threadIdx.x == 0) odd[blockIdx.x] = any;
}

// A block takes rows_each rows of one request and K/V head, a thread a column and
// every lanes-th row, so that no two change the same result.  What a row adds
// goes by which of +inf, -inf and NaN it sees: without a mask by where each
// comes first in the column, with one by a walk along the row's keys that ends
// when nothing that comes can change it.  2 requests of 2048 tokens, 8 K/V
// heads of 128, whose values are all NaN: 0.3 ms beside the attention's 0.2, under
// a mask 0.4 beside 0.5.
template <typename T, int D>
__global__ void __launch_bounds__(kValueThreads)
    whole_values(const __grid_constant__ Params p, const int* odd, const int flags, const int rows_each,
                 const int splits) {
  constexpr int kLanes = kValueThreads / D, kNever = 0x7fffffff;
  __shared__ int first[3][D];  // of +inf, -inf, NaN: the first row of the column
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int met = 0;
  for (int i = threadIdx.x; i < flags; i += kValueThreads) met |= odd[i];
  if (!__syncthreads_or(met)) return;
  const int col = threadIdx.x % D, lane = threadIdx.x / D;
  const int64_t items = static_cast<int64_t>(p.B) * p.Hkv * splits;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t bh = it / splits;
    const int h = static_cast<int>(bh % p.Hkv);
    const Request r = request(p, static_cast<int>(bh / p.Hkv));
    const int lo = static_cast<int>(it % splits) * rows_each, hi = min(r.count, lo + rows_each);
    if (lo >= hi) continue;  // for the whole block
    const int end = p.mask ? r.count : hi;  // keys that these rows may see
    const T* const v = static_cast<const T*>(p.v_new) + r.first * p.v_st + h * p.v_sh + col;
    if (lane == 0) first[0][col] = first[1][col] = first[2][col] = kNever;
    __syncthreads();
    int f[3] = {kNever, kNever, kNever};
#pragma unroll 8
    for (int j = lane; j < end; j += kLanes) {
      const float y = static_cast<float>(v[j * p.v_st]);
      if (y == INFINITY) f[0] = min(f[0], j);
      if (y == -INFINITY) f[1] = min(f[1], j);
      if (y != y) f[2] = min(f[2], j);
    }
#pragma unroll
    for (int x = 0; x < 3; ++x)
      if (f[x] != kNever) atomicMin(&first[x][col], f[x]);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 3; ++x) f[x] = first[x][col];
    const int start = min(min(f[0], f[1]), f[2]);
    const unsigned kinds = (f[0] < kNever ? 1u : 0u) | (f[1] < kNever ? 2u : 0u) | (f[2] < kNever ? 4u : 0u);
    for (int i = lo + lane; i < hi && kinds; i += kLanes) {
      unsigned seen = 0;
      if (p.mask) {
        const uint8_t* const row = p.mask + (r.first + i) * p.mask_stride;
        for (int j = start; j < end && seen != kinds && !(seen & 4u); ++j) {
          if (row[j]) continue;
          const float y = static_cast<float>(v[j * p.v_st]);
          seen |= (y == INFINITY ? 1u : 0u) | (y == -INFINITY ? 2u : 0u) | (y != y ? 4u : 0u);
        }
      } else {
        seen = (i >= f[0] ? 1u : 0u) | (i >= f[1] ? 2u : 0u) | (i >= f[2] ? 4u : 0u);
      }
      if (!seen) continue;
      const float y = seen == 1u ? INFINITY : seen == 2u ? -INFINITY : __int_as_float(0x7fc00000);
      T* const o = static_cast<T*>(p.o) + (r.first + i) * p.o_st + h * p.group * p.o_sh + col;
      for (int x = 0; x < p.group; ++x) o[x * p.o_sh] = from_f<T>(static_cast<float>(o[x * p.o_sh]) + y);
    }
    __syncthreads();
  }
}

}  // namespace attn_tree
