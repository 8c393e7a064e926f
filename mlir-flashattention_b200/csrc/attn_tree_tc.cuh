// attn_tree_tc.cuh — attn_tree_fwd for many query rows per kv-head (drafted
// trees with grouped heads, chunks of prompts), on tcgen05.
//
// From 64 query rows on, a key's 4 * rows * D operations for its 4 * D bytes
// approach what the GPU computes per byte it reads, and past some 250 rows the
// tensor cores bound the kernel: S = Q K^T and O += P V run as 128-row
// tcgen05.mma with accumulators in tensor memory.  One block per SM:
//   warp 8       TMA producer: Q, then K and V tiles of 128 keys, page segment
//                by page segment, through a ring of shared-memory tiles
//   warp 9       MMA issuer (converged warp, one elected lane issues)
//   warps 0-3    softmax of accumulator 0: one thread per query row
//   warps 4-7    softmax of accumulator 1
//   warps 10-11  idle (they complete warpgroup 2 for the register split)
// In the tiles at the end of the cached and of the new keys the softmax also
// makes the value rows that do not exist 0 in shared memory: their weights are
// 0, but what lies in memory there need not be a number.
// An item is up to two row tiles of one request and kv-head.  With two, each
// has an accumulator and every key tile serves both.  With one ("alone": a
// small tree), the two accumulators take its key tiles in turn, with maxima
// and sums of their own, so that one group's softmax overlaps the other's
// products; thread r of either group then sees row r of both accumulators in
// its lane of tensor memory, and the two are joined in registers, half of the
// columns by each group.
//
// P of a tile overwrites its S columns, so the next S product of that
// accumulator waits until the P V product has read it.  The running maximum
// moves only when a row grows past it by 2^kLazy, which skips most rescalings
// of O in tensor memory.  In bf16 a weight is rounded to 2^-9: as large an
// error as the result's own rounding, taken for half the P V work.
#pragma once

#include "attn_tree_mma.cuh"

namespace attn_tree {

namespace tc {

using namespace attn_sm100;

constexpr int kThreads = 384;
constexpr int kRegsSoftmax = 224, kRegsOther = 56;
constexpr int kRegPool = 256 * kRegsSoftmax + 128 * kRegsOther;
constexpr int kTileRows = 128, kTileKeys = 128;

template <typename T, int D>
struct Cfg {
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static constexpr int kHalves = D / 64;               // 128-byte column blocks
  static constexpr int kBox = kTileKeys * 128;         // one column block of a tile
  static constexpr int kTile = kHalves * kBox;
  static constexpr int kStages = D == 128 ? 5 : 12;    // K and V tiles in the ring
  static constexpr int kBars = 2 + 2 * kStages + 2 + 2 + 2 + 1 + 1;
  static constexpr size_t kSmem = 1024 + (2 + kStages) * kTile + kBars * 8 + 16;
  static constexpr float kShift = F16 ? 8.f : 0.f;     // weights are kept times 2^kShift
  static constexpr float kLazy = F16 ? 6.f : 8.f;      // below 2^(kShift + kLazy): 2^14 in f16
  static_assert(kSmem <= 232448, "shared memory budget");
};

// Waits for this block's own copies and products in flight, abort or not.
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, int* status) {
  int never = 0;
  mbar_wait_bounded(bar, parity, &never, status, kWaitLimitNs);
}

struct Tiles {
  int rows;  // query rows of one accumulator's tile; Split::rows is twice that
  int box;   // tokens of a Q box
};

// How the two accumulators share a piece.
struct Plan {
  bool alone;
  int end[2];  // first key tile that accumulator t does not need (of the item)

  // Accumulator t takes key tile k of a piece that begins at k0.
  __device__ __forceinline__ bool takes(int t, int k, int k0) const {
    return alone ? ((k - k0) & 1) == t : k < end[t];
  }
  __device__ __forceinline__ int first(int t, int k0) const { return alone ? k0 + t : k0; }
  __device__ __forceinline__ int step() const { return alone ? 2 : 1; }
  // End of accumulator t's tiles in a piece that ends at k1.
  __device__ __forceinline__ int stop(int t, int k1) const { return min(end[t], k1); }
};

__device__ __forceinline__ Plan make_plan(const Params& p, const Split& s, const Tiles& tl, const Piece& pc) {
  Plan r;
  const int64_t rows = static_cast<int64_t>(pc.r.count) * p.group - static_cast<int64_t>(pc.rt) * s.rows;
  r.alone = rows <= tl.rows;
  r.end[0] = r.end[1] = pc.tiles;
  if (!r.alone && p.mask == nullptr) {
    const int keys = min(pc.r.count, (pc.rt * s.rows + tl.rows - 1) / p.group + 1);
    r.end[0] = pc.cached + ((keys + (1 << s.new_shift) - 1) >> s.new_shift);
  }
  return r;
}

// Keys that exist in tile k of a piece.
__device__ __forceinline__ int keys_here(const Split& s, const Piece& pc, int k) {
  return k < pc.cached ? min(kTileKeys, pc.r.held - (k << s.keys_shift))
                       : min(1 << s.new_shift, pc.r.count - ((k - pc.cached) << s.new_shift));
}

// Bits of one row of the mask for keys [first, first + here) of its request's
// new ones: the warp reads each row of its 32 query rows' tokens together.
__device__ __forceinline__ void mask_bits(const Params& p, const Piece& pc, int token, int t_lo, int t_hi,
                                          int first, int here, int lane, uint32_t (&bits)[4]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) bits[w] = 0xffffffffu;
  const uint8_t* const m = p.mask + static_cast<int64_t>(pc.r.first) * p.mask_stride + first;
  for (int t0 = t_lo; t0 <= t_hi; t0 += 4) {
    uint32_t b[4][4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        b[x][w] = 1;
        if (t0 + x <= t_hi && 32 * w + lane < here)
          b[x][w] = m[static_cast<int64_t>(t0 + x) * p.mask_stride + 32 * w + lane];
      }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v = __ballot_sync(0xffffffffu, b[x][w] != 0);
        if (token == t0 + x) bits[w] = v;
      }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kc,
                   const __grid_constant__ CUtensorMap map_vc, const __grid_constant__ CUtensorMap map_kn,
                   const __grid_constant__ CUtensorMap map_vn, const __grid_constant__ Params p, const Split split,
                   const Tiles tiles, const Scratch scratch, const int min_units) {
  using C = Cfg<T, D>;
  constexpr bool F16 = C::F16;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  uint8_t* const sQ = smem;
  uint8_t* const sKV = smem + 2 * C::kTile;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(sKV + C::kStages * C::kTile);
  uint64_t* const q_full = bars;
  uint64_t* const q_empty = bars + 1;
  uint64_t* const kv_full = bars + 2;
  uint64_t* const kv_empty = kv_full + C::kStages;
  uint64_t* const s_full = kv_empty + C::kStages;
  uint64_t* const p_ready = s_full + 2;
  uint64_t* const pv_done = p_ready + 2;
  uint64_t* const o_free = pv_done + 2;  // both accumulators of a piece have been read
  uint64_t* const drain = o_free + 1;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_ready[t], 4);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(o_free, 256);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (tid < 2) scratch.record[2 * blockIdx.x + tid].b = -1;
  tc_fence_before();
  Share share = find_share(p, split, min_units);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t share_lo = share.lo;
  Piece pc;
  auto slot = [](int pos) { return pos % C::kStages; };
  auto par = [](int pos) { return static_cast<uint32_t>((pos / C::kStages) & 1); };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, kWaitLimitNs));
  };

  if (warp >= 8) {
    setmaxnreg_dec<kRegsOther>();
    if (warp == 8) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_kc);
        prefetch_tmap(&map_vc);
        prefetch_tmap(&map_kn);
        prefetch_tmap(&map_vn);
      }
      const int seg_shift = min(p.page_shift, split.keys_shift);  // rows of a page segment, log2
      int pos = 0, qi = 0;
      bool ok = true;
      while (ok && next_piece(p, split, share, pc)) {
        const Plan plan = make_plan(p, split, tiles, pc);
        const int32_t* const row = p.table + pc.b * p.table_stride;
        for (int k = pc.k0; k < pc.k1 && ok; ++k) {
          const bool cached = k < pc.cached;
          const int first = cached ? k << split.keys_shift : (k - pc.cached) << split.new_shift;
          int segs = 1, page = 0, at = 0;
          if (cached) {
            segs = (keys_here(split, pc, k) + (1 << seg_shift) - 1) >> seg_shift;
            if (lane < segs) {
              const int key = first + (lane << seg_shift);
              page = __ldg(row + (key >> p.page_shift));
              at = key & ((1 << p.page_shift) - 1);
              if (page < 0 || page >= p.num_pages) {
                atomicCAS(p.status, 0, ATTN_ERR_INVALID);
                page = max(p.num_pages, 1);  // outside the map: zeros
              }
            }
          }
          for (int v = 0; v < 2 && ok; ++v, ++pos) {
            const int s = slot(pos);
            ok = wait(&kv_empty[s], par(pos) ^ 1u);
            if (!ok) break;
            const int seg = cached ? 128 << seg_shift : 128 << split.new_shift;
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], segs * seg * C::kHalves);
            __syncwarp();
            if (lane < segs) {
              const uint32_t dst = smem_u32(sKV + s * C::kTile) + lane * seg;
#pragma unroll
              for (int c = 0; c < C::kHalves; ++c) {
                if (cached)
                  tma_load_5d(dst + c * C::kBox, v ? &map_vc : &map_kc, &kv_full[s], 0, at, c, pc.h, page);
                else
                  tma_load_5d(dst + c * C::kBox, v ? &map_vn : &map_kn, &kv_full[s], 0, pc.r.first + first, c, pc.h, 0);
              }
            }
          }
          if (k == pc.k0 && ok) {
            // Q behind the piece's first keys, which need no wait for the
            // last S product of the piece before.
            ok = wait(q_empty, static_cast<uint32_t>(qi & 1) ^ 1u);
            if (!ok) break;
            if (lane == 0) {
              const int n = plan.alone ? 1 : 2;
              mbar_arrive_expect_tx(q_full, n * C::kHalves * tiles.rows * 128);
              for (int t = 0; t < n; ++t)
                for (int c = 0; c < C::kHalves; ++c)
                  tma_load_5d(smem_u32(sQ + t * C::kTile + c * C::kBox), &map_q, q_full, 0, 0,
                              pc.r.first + pc.rt * (2 * tiles.box) + t * tiles.box, c, pc.h);
            }
            ++qi;
            __syncwarp();
          }
        }
      }
      // Every copy that was started lands before the block may end.
      if (lane == 0) {
        if (qi > 0) drain_wait(q_full, static_cast<uint32_t>((qi - 1) & 1), p.status);
        for (int s = 0; s < C::kStages && s < pos; ++s)
          drain_wait(&kv_full[s], static_cast<uint32_t>(((pos - 1 - s) / C::kStages) & 1), p.status);
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer
      constexpr uint32_t fmt = F16 ? 0u : 1u;
      constexpr uint32_t idS = make_idesc(128, kTileKeys, fmt, false);
      constexpr uint32_t idO = make_idesc(128, D, fmt, true);
      const uint64_t dQ0 = make_sdesc(smem_u32(sQ), 16, 1024);
      const uint64_t dK0 = make_sdesc(smem_u32(sKV), 16, 1024);
      const uint64_t dV0 = make_sdesc(smem_u32(sKV), C::kBox, 1024);
      const uint32_t lead = elect_one();
      int base = 0, qi = 0;
      int s_cnt[2] = {0, 0}, pv_cnt[2] = {0, 0}, items = 0;
      bool ok = true;
      while (ok && next_piece(p, split, share, pc)) {
        const Plan plan = make_plan(p, split, tiles, pc);
        auto kpos = [&](int k) { return base + 2 * (k - pc.k0); };
        int left = 0;  // S products still to issue from this Q
        for (int t = 0; t < 2; ++t) {
          const int f = plan.first(t, pc.k0), e = plan.stop(t, pc.k1);
          if (f < e) left += (e - f + plan.step() - 1) / plan.step();
        }
        int k_seen = pc.k0 - 1;  // last key tile whose K has arrived
        auto issue_S = [&](int t, int k) {
          if (k > k_seen) {
            if (!wait(&kv_full[slot(kpos(k))], par(kpos(k)))) return false;
            k_seen = k;
          }
          // The S columns hold P of this accumulator's last tile: the product
          // that reads it has to be complete, as the two do not share an
          // accumulator and so are not ordered by their issue.
          if (pv_cnt[t] > 0 && !wait(&pv_done[t], static_cast<uint32_t>((pv_cnt[t] - 1) & 1))) return false;
          tc_fence_after();
          const uint64_t a0 = dQ0 + static_cast<uint64_t>(((plan.alone ? 0 : t) * C::kTile) >> 4);
          const uint64_t b0 = dK0 + static_cast<uint64_t>((slot(kpos(k)) * C::kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk * 32) / 128) * C::kBox + ((kk * 32) % 128);
            mma_ss_lead<0>(lead, tmem + t * 128, a0 + (off >> 4), b0 + (off >> 4), idS, kk > 0 ? 1u : 0u);
          }
          mma_commit_lead(lead, &s_full[t]);
          ++s_cnt[t];
          // K is free after its last S product (accumulator 1's, of two).
          if (plan.alone || t == 1) mma_commit_lead(lead, &kv_empty[slot(kpos(k))]);
          if (--left == 0) mma_commit_lead(lead, q_empty);
          return true;
        };
        ok = wait(q_full, static_cast<uint32_t>(qi & 1));
        for (int t = 0; t < 2 && ok; ++t) {
          const int f = plan.first(t, pc.k0);
          if (f < plan.stop(t, pc.k1)) ok = issue_S(t, f);
        }
        bool first_pv[2] = {true, true}, waited = items == 0;
        for (int k = pc.k0; k < pc.k1 && ok; ++k) {
          const int vp = kpos(k) + 1;
          ok = wait(&kv_full[slot(vp)], par(vp));
          for (int t = 0; t < 2 && ok; ++t) {
            if (!plan.takes(t, k, pc.k0)) continue;
            ok = wait(&p_ready[t], static_cast<uint32_t>(pv_cnt[t] & 1));
            if (ok && !waited) {  // O of the piece before has been read
              ok = wait(o_free, static_cast<uint32_t>((items - 1) & 1));
              waited = true;
            }
            if (!ok) break;
            tc_fence_after();
            const uint64_t b0 = dV0 + static_cast<uint64_t>((slot(vp) * C::kTile) >> 4);
#pragma unroll
            for (int kk = 0; kk < kTileKeys / 16; ++kk)
              mma_ts_lead<0>(lead, tmem + 256 + t * D, tmem + t * 128 + kk * 8,
                             b0 + static_cast<uint64_t>((kk * 16 * 128) >> 4), idO, (!first_pv[t] || kk > 0) ? 1u : 0u);
            first_pv[t] = false;
            mma_commit_lead(lead, &pv_done[t]);
            ++pv_cnt[t];
            const int next = k + plan.step();
            if (next < plan.stop(t, pc.k1)) ok = issue_S(t, next);
          }
          if (ok) mma_commit_lead(lead, &kv_empty[slot(vp)]);  // V free after its P V products
        }
        base += 2 * (pc.k1 - pc.k0);
        ++qi;
        ++items;
      }
      mma_commit_lead(lead, drain);
      if (lane == 0) drain_wait(drain, 0, p.status);
      __syncwarp();
    }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ---------------------------------------------------------------- softmax
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + t * 128;
    const uint32_t tO = tmem + lane_off + 256 + t * D;
    float sl2 = p.scale * kLog2e;
    if (sl2 == 0.f) sl2 = 1e-30f;  // a scale of 0: even weights without 0 * inf
    const bool pos = sl2 >= 0.f;
    const float hidden = pos ? -INFINITY : INFINITY;
    int steps = 0;  // S tiles of this accumulator so far
    int base = 0;   // ring position of the piece's first K
    bool ok = true;
    while (next_piece(p, split, share, pc)) {
      const Plan plan = make_plan(p, split, tiles, pc);
      const int64_t item_rows = static_cast<int64_t>(pc.r.count) * p.group - static_cast<int64_t>(pc.rt) * split.rows;
      const int row0 = plan.alone ? 0 : t * tiles.rows;             // of the item
      const int rows = static_cast<int>(min(static_cast<int64_t>(tiles.rows), item_rows - row0));
      const int at = pc.rt * split.rows + row0 + min(r, max(rows, 1) - 1);
      const int token = at / p.group, head = pc.h * p.group + at % p.group;
      const bool busy = (warp & 3) * 32 < rows;  // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f;
      bool first = true;
      const int stop = plan.stop(t, pc.k1);
      // Mask bits of the first new tile, read while its keys are on their way.
      uint32_t bits[4] = {0, 0, 0, 0};
      const int t_lo = __shfl_sync(0xffffffffu, token, 0), t_hi = __shfl_sync(0xffffffffu, token, 31);
      int bits_of = -1;
      if (p.mask && busy && stop > pc.cached) {
        const int f = plan.first(t, pc.k0);
        const int k = max(pc.cached, f) + (plan.alone && pc.cached > f ? ((pc.cached - f) & 1) : 0);
        if (k < stop) {
          mask_bits(p, pc, token, t_lo, t_hi, (k - pc.cached) << split.new_shift, keys_here(split, pc, k), lane, bits);
          bits_of = k;
        }
      }
      for (int k = plan.first(t, pc.k0); k < stop; k += plan.step(), ++steps) {
        const bool cached = k < pc.cached;
        const int here = keys_here(split, pc, k);
        if (!cached && p.mask && busy && bits_of != k) {
          mask_bits(p, pc, token, t_lo, t_hi, (k - pc.cached) << split.new_shift, here, lane, bits);
          bits_of = k;
        }
        if (ok) ok = wait(&s_full[t], static_cast<uint32_t>(steps & 1));
        tc_fence_after();
        if (here < kTileKeys && (t == 0 || !plan.takes(0, k, pc.k0))) {
          // Accumulator 0's products of a tile come first.  The tile before in
          // V's slot has been used (S of this one is complete), so the phase
          // waited for is the slot's next.
          const int vp = base + 2 * (k - pc.k0) + 1;
          if (ok) ok = wait(&kv_full[slot(vp)], par(vp));
          if (r >= here) {
            uint8_t* const v = sKV + slot(vp) * C::kTile + r * 128;
#pragma unroll
            for (int c = 0; c < C::kHalves; ++c)
#pragma unroll
              for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(v + c * C::kBox + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (busy) {
          float s[128];
          {
            uint32_t r0[32], r1[32], r2[32], r3[32];
            tmem_ld32(tS + 0, r0);
            tmem_ld32(tS + 32, r1);
            tmem_ld32(tS + 64, r2);
            tmem_ld32(tS + 96, r3);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s[i] = __uint_as_float(r0[i]);
              s[32 + i] = __uint_as_float(r1[i]);
              s[64 + i] = __uint_as_float(r2[i]);
              s[96 + i] = __uint_as_float(r3[i]);
            }
          }
          int lim = here;  // keys below it are seen
          if (!cached) {
            if (p.mask) {
#pragma unroll
              for (int c = 0; c < 128; ++c)
                if ((bits[c >> 5] >> (c & 31)) & 1u) s[c] = hidden;
            } else {
              lim = min(here, token - ((k - pc.cached) << split.new_shift) + 1);
            }
          }
          if (__any_sync(0xffffffffu, lim < 128)) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c >= lim) s[c] = hidden;
          }
          float red;
          if (pos) {
            float a0 = max3(s[0], s[1], s[2]), a1 = max3(s[3], s[4], s[5]);
#pragma unroll
            for (int c = 6; c < 126; c += 4) {
              a0 = max3(a0, s[c], s[c + 1]);
              a1 = max3(a1, s[c + 2], s[c + 3]);
            }
            red = max3(a0, a1, fmaxf(s[126], s[127]));
          } else {
            float a0 = min3(s[0], s[1], s[2]), a1 = min3(s[3], s[4], s[5]);
#pragma unroll
            for (int c = 6; c < 126; c += 4) {
              a0 = min3(a0, s[c], s[c + 1]);
              a1 = min3(a1, s[c + 2], s[c + 3]);
            }
            red = min3(a0, a1, fminf(s[126], s[127]));
          }
          const float top = red * sl2;
          float alpha = 1.f;
          if (top > m + C::kLazy) {  // from -inf: any finite maximum
            alpha = ex2(m - top);
            m = top;
          }
          if (__any_sync(0xffffffffu, !first && alpha != 1.f)) {
            // The P V product before this S product is complete (see issue_S).
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(tO + c * 32, o);
            }
          }
          first = false;
          const float sub = m == -INFINITY ? 0.f : C::kShift - m;
          const uint64_t sl2x2 = f2_pack(sl2, sl2), subx2 = f2_pack(sub, sub);
          uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const int cc = 32 * h + c;
              float x0, x1;
              f2_unpack(f2_fma(f2_pack(s[2 * cc], s[2 * cc + 1]), sl2x2, subx2), x0, x1);
              const float e0 = ex2(x0), e1 = ex2(x1);
              const uint64_t pr = f2_pack(e0, e1);
              if (c & 1) sum1 = f2_add(sum1, pr); else sum0 = f2_add(sum0, pr);
              pk[c] = pack2<F16>(e0, e1);
            }
            tmem_st32(tS + 32 * h, pk);
          }
          float q0, q1;
          f2_unpack(f2_add(sum0, sum1), q0, q1);
          l = l * alpha + (q0 + q1);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
      }
      base += 2 * (pc.k1 - pc.k0);
      // ------------------------------------------------------------ a piece ends
      const bool has = plan.first(t, pc.k0) < stop;
      if (has && ok) ok = wait(&pv_done[t], static_cast<uint32_t>((steps - 1) & 1));
      tc_fence_after();
      const bool whole = pc.k0 == 0 && pc.k1 == pc.tiles;
      const int rec = 2 * blockIdx.x + (share.lo - (pc.k1 - pc.k0) == share_lo ? 0 : 1);
      // Alone: columns [D/2 t, D/2 t + D/2) of both accumulators; else all of its own.
      float f0 = 1.f, f1 = 0.f, mm = m, ll = l;
      bool has0 = has, has1 = false;
      if (plan.alone) {
        // Both groups' maxima and sums meet in this piece's scratch slot (shared
        // memory is full).
        scratch.m[rec * 256 + t * 128 + r] = m;
        scratch.l[rec * 256 + t * 128 + r] = l;
        __threadfence();  // read past L1
        tc_fence_before();
        __syncwarp();
        asm volatile("barrier.sync 2, 256;" ::: "memory");
        tc_fence_after();
        has0 = true, has1 = pc.k1 - pc.k0 > 1;
        const float m0 = __ldcg(scratch.m + rec * 256 + r), m1 = __ldcg(scratch.m + rec * 256 + 128 + r);
        mm = fmaxf(m0, m1);
        f0 = mm == -INFINITY ? 0.f : ex2(m0 - mm);
        f1 = mm == -INFINITY ? 0.f : ex2(m1 - mm);
        ll = f0 * __ldcg(scratch.l + rec * 256 + r) + f1 * __ldcg(scratch.l + rec * 256 + 128 + r);
      }
      const bool live = r < rows && busy;
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      const bool none = ll == 0.f;  // nothing seen: 0 whatever the accumulator holds
      const float w0 = whole ? f0 * inv : f0, w1 = whole ? f1 * inv : f1;
      T* const orow = static_cast<T*>(p.o) + static_cast<int64_t>(pc.r.first + token) * p.o_st + head * p.o_sh;
      float* const srow = scratch.o + (static_cast<int64_t>(rec) * 256 + row0 + r) * D;
      const uint32_t tA = tmem + lane_off + 256 + (plan.alone ? 0 : t * D), tB = tmem + lane_off + 256 + D;
      const int c_lo = plan.alone ? t * (D / 2) : 0, c_hi = plan.alone ? c_lo + D / 2 : D;
      if (busy) {
        for (int c = c_lo; c < c_hi; c += 32) {
          uint32_t a[32];
          if (has0) {
            tmem_ld32(tA + c, a);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 32; ++i)
            a[i] = has0 && !none ? __float_as_uint(__uint_as_float(a[i]) * w0) : 0u;
          if (has1 && plan.alone) {
            uint32_t b[32];
            tmem_ld32(tB + c, b);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!none) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), w1, __uint_as_float(a[i])));
          }
          if (live) {
            if (whole) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                reinterpret_cast<uint4*>(orow + c)[i] =
                    make_uint4(pack2<F16>(__uint_as_float(a[8 * i]), __uint_as_float(a[8 * i + 1])),
                               pack2<F16>(__uint_as_float(a[8 * i + 2]), __uint_as_float(a[8 * i + 3])),
                               pack2<F16>(__uint_as_float(a[8 * i + 4]), __uint_as_float(a[8 * i + 5])),
                               pack2<F16>(__uint_as_float(a[8 * i + 6]), __uint_as_float(a[8 * i + 7])));
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(srow + c)[i] = make_uint4(a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(o_free);
      if (plan.alone) {  // both groups have read the slot
        __syncwarp();
        asm volatile("barrier.sync 2, 256;" ::: "memory");
      }
      if (live && (!plan.alone || t == 0)) {
        if (!whole) {
          scratch.m[rec * 256 + row0 + r] = mm;
          scratch.l[rec * 256 + row0 + r] = ll;
        } else if (p.lse) {
          p.lse[static_cast<int64_t>(pc.r.first + token) * p.Hq + head] =
              ll == 0.f ? -INFINITY : (mm - C::kShift + log2f(ll)) * kLn2;
        }
      }
      if (!whole && tid == 0)
        scratch.record[rec] = Record{pc.b, pc.h, pc.rt, (pc.k0 == 0 ? 1 : 0) | (pc.k1 == pc.tiles ? 2 : 0)};
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace tc

}  // namespace attn_tree
