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
//   warp 10      cuts the block's share into pieces, ahead of the others, and
//                hands them out through a short queue in shared memory
//   warp 11      with a mask, turns the mask's bytes into bits in shared memory
//                ahead of the softmax (else idle)
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
// of O in tensor memory.  In bf16 a weight is rounded to 2^-8: as large an
// error as the result's own rounding, taken for half the P V work.
//
// What bounds it is the chain of a tile: S read, maximum, exponentials, P
// written, P V, about 3,850 clocks a pair of tiles while the tensor cores need
// half: 2048 new tokens on 8192 keys, 32 heads on 8, 2 requests: 470 us, 0.9
// PFLOP/s; 484 for the whole call with clean_values and whole_values.  64 drafted
// tokens on 16384 keys, 8 requests: 114 us with the mask's bits (122 the whole
// call), 73 us without a mask.  With a mask the kernel spills 164 bytes a thread,
// without one 12.
#pragma once

#include "attn_tree_mma.cuh"

namespace attn_tree {

namespace tc {

using namespace attn_sm100;

constexpr int kThreads = 384;
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
constexpr int kRegPool = 256 * kRegsSoftmax + 128 * kRegsOther;
constexpr int kTileRows = 128, kTileKeys = 128;

template <typename T, int D, bool MASK, bool ALONE>
struct Cfg {
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static constexpr int kHalves = D / 64;               // 128-byte column blocks
  static constexpr int kBox = kTileKeys * 128;         // one column block of a tile
  static constexpr int kTile = kHalves * kBox;
  // K and V tiles in the ring.  Mask bits take the room of one; a second Q tile
  // that no item has leaves one.
  static constexpr int kQTiles = ALONE ? 1 : 2;
  static constexpr int kStages = (D == 128 ? 7 : 14) - kQTiles - (MASK ? 1 : 0);
  static constexpr int kBits = MASK ? 256 : 0;         // 16-byte rows of mask bits, twice
  static constexpr int kQueue = 4;                     // pieces handed out ahead
  static constexpr int kBars = 2 + 2 * kStages + 2 + 4 + 2 + 3 + 2 * kQueue + 4;
  static constexpr size_t kSmem = 1024 + (kQTiles + kStages) * kTile + 2 * kBits * 16 + kBars * 8 + 16 + kQueue * 64;
  static constexpr float kShift = F16 ? 8.f : 0.f;     // weights are kept times 2^kShift
  static constexpr float kLazy = F16 ? 6.f : 8.f;      // below 2^(kShift + kLazy): 2^14 in f16
  static_assert(kSmem + 512 <= 232448, "shared memory budget");
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

// A piece as the block's warps need it.
struct Job {
  int b, h, rt;            // b = -1: no more
  int k0, k1, cached;      // key tiles [k0, k1) of the item; tiles below `cached` are cached keys
  int held, first, count;  // of the request
  int alone;               // one row tile, whose key tiles both accumulators take in turn
  int end0, end1;          // first key tile that accumulator 0 / 1 does not need
  int rec;                 // scratch slot
  int whole;               // all of its item's key tiles
  int rows;                // query rows of the item

  // Accumulator t takes key tile k.
  __device__ __forceinline__ bool takes(int t, int k) const {
    return alone ? ((k - k0) & 1) == t : k < (t ? end1 : end0);
  }
  __device__ __forceinline__ int from(int t) const { return alone ? k0 + t : k0; }
  __device__ __forceinline__ int step() const { return alone ? 2 : 1; }
  __device__ __forceinline__ int stop(int t) const { return min(t ? end1 : end0, k1); }
  // Places in the ring, from the piece's first on: K, V of each tile in turn, or
  // (early: ALONE, where two tiles are in work) K_0, K_1, V_0, K_2, V_1, .., the
  // order of use, so that no slot is held for a V that is two products away.
  template <bool EARLY>
  __device__ __forceinline__ int k_place(int k) const {
    const int i = k - k0;
    return EARLY ? max(2 * i - 1, 0) : 2 * i;
  }
  template <bool EARLY>
  __device__ __forceinline__ int v_place(int k) const {
    const int i = k - k0;
    return EARLY && k + 1 < k1 ? 2 * i + 2 : 2 * i + 1;
  }
  // Keys that exist in tile k.
  __device__ __forceinline__ int here(const Split& s, int k) const {
    return k < cached ? min(kTileKeys, held - (k << s.keys_shift))
                      : min(1 << s.new_shift, count - ((k - cached) << s.new_shift));
  }
};
static_assert(sizeof(Job) <= 64, "a queue entry");

__device__ __forceinline__ Job make_job(const Params& p, const Split& s, const Tiles& tl, const Piece& pc, int rec) {
  Job j;
  j.b = pc.b, j.h = pc.h, j.rt = pc.rt;
  j.k0 = pc.k0, j.k1 = pc.k1, j.cached = pc.cached;
  j.held = pc.r.held, j.first = pc.r.first, j.count = pc.r.count;
  j.rows = static_cast<int>(min(static_cast<int64_t>(s.rows), static_cast<int64_t>(pc.r.count) * p.group -
                                                                   static_cast<int64_t>(pc.rt) * s.rows));
  j.alone = j.rows <= tl.rows;
  j.end0 = j.end1 = pc.tiles;
  if (!j.alone && p.mask == nullptr) {
    const int keys = min(pc.r.count, (pc.rt * s.rows + tl.rows - 1) / p.group + 1);
    j.end0 = pc.cached + ((keys + (1 << s.new_shift) - 1) >> s.new_shift);
  }
  j.rec = rec;
  j.whole = pc.k0 == 0 && pc.k1 == pc.tiles;
  return j;
}

// Bits of one row of the mask for `here` <= 128 new keys (1: masked, or no
// such key), from V bytes at a time; the row is aligned to V.
template <int V>
__device__ __forceinline__ void mask_row(const uint8_t* row, int here, uint32_t (&bits)[4]) {
  using W = typename std::conditional<V == 16, uint4, typename std::conditional<V == 4, uint32_t, uint8_t>::type>::type;
  auto nibble = [](uint32_t w) { return ((__vcmpne4(w, 0u) & 0x08040201u) * 0x01010101u) >> 24; };
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t b = 0;
    if (32 * q < here) {
      constexpr int kLoads = 32 / V;
      W w[kLoads];
#pragma unroll
      for (int x = 0; x < kLoads; ++x)
        if (32 * q + (x + 1) * V <= here) w[x] = *reinterpret_cast<const W*>(row + 32 * q + x * V);
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        if (32 * q + (x + 1) * V <= here) {
          if constexpr (V == 16)
            b |= (nibble(w[x].x) | nibble(w[x].y) << 4 | nibble(w[x].z) << 8 | nibble(w[x].w) << 12) << (16 * x);
          else if constexpr (V == 4)
            b |= nibble(w[x]) << (4 * x);
          else
            b |= (w[x] != 0 ? 1u : 0u) << x;
        } else {
          for (int e = 0; e < V; ++e) {
            const int j = x * V + e;
            if (32 * q + j < here && row[32 * q + j] != 0) b |= 1u << j;
          }
        }
      }
      if (32 * q + 32 > here) b |= 0xffffffffu << (here - 32 * q);
    } else {
      b = 0xffffffffu;
    }
    bits[q] = b;
  }
}

// ALONE: no request has more rows than one tile, so that every item is alone.
template <typename T, int D, bool MASK, bool ALONE>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kc,
                   const __grid_constant__ CUtensorMap map_vc, const __grid_constant__ CUtensorMap map_kn,
                   const __grid_constant__ CUtensorMap map_vn, const __grid_constant__ Params p, const Split split,
                   const Tiles tiles, const Scratch scratch, const int min_units) {
  using C = Cfg<T, D, MASK, ALONE>;
  constexpr bool F16 = C::F16;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  uint8_t* const sQ = smem;
  uint8_t* const sKV = smem + C::kQTiles * C::kTile;
  uint4* const s_bits = reinterpret_cast<uint4*>(sKV + C::kStages * C::kTile);  // [2][tokens of an item]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_bits + 2 * C::kBits);
  uint64_t* const q_full = bars;
  uint64_t* const q_empty = bars + 1;
  uint64_t* const kv_full = bars + 2;
  uint64_t* const kv_empty = kv_full + C::kStages;
  uint64_t* const s_full = kv_empty + C::kStages;
  uint64_t* const p_ready = s_full + 2;    // [half of P][accumulator]
  uint64_t* const pv_done = p_ready + 4;
  uint64_t* const o_free = pv_done + 2;    // both accumulators of a piece have been read
  uint64_t* const met = o_free + 1;        // alone: both groups are at one point
  uint64_t* const drain = met + 1;
  uint64_t* const job_full = drain + 1;
  uint64_t* const job_empty = job_full + C::kQueue;
  uint64_t* const bits_full = job_empty + C::kQueue;
  uint64_t* const bits_empty = bits_full + 2;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bits_empty + 2);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Job* const jobs = reinterpret_cast<Job*>(tmem_slot + 4);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
      mbar_init(&p_ready[2 + t], 4);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(o_free, 256);
    mbar_init(met, 256);
    mbar_init(drain, 1);
    for (int i = 0; i < C::kQueue; ++i) {
      mbar_init(&job_full[i], 1);
      mbar_init(&job_empty[i], MASK ? 11 : 10);  // producer, issuer, eight softmax warps, warp 11
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bits_full[i], 1);
      mbar_init(&bits_empty[i], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_wait();
  grid_release();
  if (tid == 0) scratch.record[blockIdx.x].pieces = 0;
  tc_fence_before();
  Share share = find_share<1>(p, split, min_units, 0);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto slot = [](int pos) { return pos % C::kStages; };
  auto par = [](int pos) { return static_cast<uint32_t>((pos / C::kStages) & 1); };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, kWaitLimitNs));
  };
  // The n-th piece; false when there is none (or the block gives up).
  auto take_job = [&](int n, Job& j) {
    const int i = n % C::kQueue;
    if (!wait(&job_full[i], static_cast<uint32_t>((n / C::kQueue) & 1))) return false;
    j = jobs[i];
    return j.b >= 0;
  };
  auto leave_job = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&job_empty[n % C::kQueue]);
  };

  if (warp >= 8) {
    setmaxnreg_dec<kRegsOther>();
    if (warp == 8) {
      // ---------------------------------------------------------- producer
      const int seg_shift = min(p.page_shift, split.keys_shift);  // rows of a page segment, log2
      int pos = 0, n = 0;
      bool ok = true;
      Job j;
      for (; ok && take_job(n, j); ++n) {
        leave_job(n);
        const int32_t* const row = p.table + j.b * p.table_stride;
        auto segments = [&](int k) { return (j.here(split, k) + (1 << seg_shift) - 1) >> seg_shift; };
        auto page_of = [&](int k) {  // of this lane's segment
          if (k >= min(j.cached, j.k1) || lane >= segments(k)) return 0;
          return row[((k << split.keys_shift) + (lane << seg_shift)) >> p.page_shift];
        };
        // K and V of a tile share its page ids, which are read a tile ahead.
        constexpr int kLag = ALONE ? 1 : 0;
        int page_next = page_of(j.k0), page_last = 0;
        for (int k = j.k0; k < j.k1 + kLag && ok; ++k) {
          const int page_here = page_next;
          page_next = page_of(k + 1);
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int kk = v ? k - kLag : k;
            if (kk < j.k0 || kk >= j.k1) continue;
            const bool cached = kk < j.cached;
            const int segs = cached ? segments(kk) : 1;
            int page = v && ALONE ? page_last : page_here, at = 0;
            if (cached && lane < segs) {
              at = ((kk << split.keys_shift) + (lane << seg_shift)) & ((1 << p.page_shift) - 1);
              if (page < 0 || page >= p.num_pages) {
                atomicCAS(p.status, 0, ATTN_ERR_INVALID);
                page = max(p.num_pages, 1);  // outside the map: zeros
              }
            }
            const int s = slot(pos);
            ok = wait(&kv_empty[s], par(pos) ^ 1u);
            if (!ok) break;
            ++pos;
            const int seg = 128 << (cached ? seg_shift : split.new_shift);
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], segs * seg * C::kHalves);
            __syncwarp();
            if (lane < segs) {
              const uint32_t dst = smem_u32(sKV + s * C::kTile) + lane * seg;
#pragma unroll
              for (int c = 0; c < C::kHalves; ++c) {
                if (cached)
                  tma_load_5d(dst + c * C::kBox, v ? &map_vc : &map_kc, &kv_full[s], 0, at, c, j.h, page);
                else
                  tma_load_5d(dst + c * C::kBox, v ? &map_vn : &map_kn, &kv_full[s], 0,
                              j.first + ((kk - j.cached) << split.new_shift), c, j.h, 0);
              }
            }
          }
          page_last = page_here;
          if (k == j.k0 && ok) {
            // Q behind the piece's first keys, which need not wait for the
            // last S product of the piece before.
            ok = wait(q_empty, static_cast<uint32_t>(n & 1) ^ 1u);
            if (!ok) break;
            if (lane == 0) {
              const int m = ALONE || j.alone ? 1 : 2;
              mbar_arrive_expect_tx(q_full, m * C::kHalves * tiles.rows * 128);
              for (int t = 0; t < m; ++t)
                for (int c = 0; c < C::kHalves; ++c)
                  tma_load_5d(smem_u32(sQ + t * C::kTile + c * C::kBox), &map_q, q_full, 0, 0,
                              j.first + j.rt * (2 * tiles.box) + t * tiles.box, c, j.h);
            }
            __syncwarp();
          }
        }
      }
      // Every copy that was started lands before the block may end.  (n counts
      // the pieces whose Q was asked for; after a wait that gave up, q_full may
      // be one phase behind, which this wait then also gives up on.)
      if (lane == 0) {
        if (n > 0) drain_wait(q_full, static_cast<uint32_t>((n - 1) & 1), p.status);
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
      int base = 0, n = 0;
      int pv_cnt[2] = {0, 0};
      bool ok = true;
      Job j;
      for (; ok && take_job(n, j); ++n) {
        leave_job(n);
        auto kpos = [&](int k) { return base + j.template k_place<ALONE>(k); };
        int left = 0;  // S products still to issue from this Q
        for (int t = 0; t < 2; ++t) {
          const int f = j.from(t), e = j.stop(t);
          if (f < e) left += (e - f + j.step() - 1) / j.step();
        }
        int k_seen = j.k0 - 1;  // last key tile whose K has arrived
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
          const uint64_t a0 = dQ0 + static_cast<uint64_t>(((j.alone ? 0 : t) * C::kTile) >> 4);
          const uint64_t b0 = dK0 + static_cast<uint64_t>((slot(kpos(k)) * C::kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk * 32) / 128) * C::kBox + ((kk * 32) % 128);
            mma_ss_lead<0>(lead, tmem + t * 128, a0 + (off >> 4), b0 + (off >> 4), idS, kk > 0 ? 1u : 0u);
          }
          mma_commit_lead(lead, &s_full[t]);
          // K is free after its last S product (accumulator 1's, of two).
          if (j.alone || t == 1) mma_commit_lead(lead, &kv_empty[slot(kpos(k))]);
          if (--left == 0) mma_commit_lead(lead, q_empty);
          return true;
        };
        ok = wait(q_full, static_cast<uint32_t>(n & 1));
        for (int t = 0; t < 2 && ok; ++t)
          if (j.from(t) < j.stop(t)) ok = issue_S(t, j.from(t));
        bool first_pv[2] = {true, true}, waited = n == 0;
        for (int k = j.k0; k < j.k1 && ok; ++k) {
          const int vp = base + j.template v_place<ALONE>(k);
          ok = wait(&kv_full[slot(vp)], par(vp));
          for (int t = 0; t < 2 && ok; ++t) {
            if (!j.takes(t, k)) continue;
            ok = wait(&p_ready[t], static_cast<uint32_t>(pv_cnt[t] & 1));
            if (ok && !waited) {  // O of the piece before has been read
              ok = wait(o_free, static_cast<uint32_t>((n - 1) & 1));
              waited = true;
            }
            if (!ok) break;
            tc_fence_after();
            const uint64_t b0 = dV0 + static_cast<uint64_t>((slot(vp) * C::kTile) >> 4);
            // P V of keys 0-63 while the softmax stores the weights of 64-127.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h == 1) {
                ok = wait(&p_ready[2 + t], static_cast<uint32_t>(pv_cnt[t] & 1));
                if (!ok) break;
                tc_fence_after();
              }
#pragma unroll
              for (int kk = h * (kTileKeys / 32); kk < (h + 1) * (kTileKeys / 32); ++kk)
                mma_ts_lead<0>(lead, tmem + 256 + t * D, tmem + t * 128 + kk * 8,
                               b0 + static_cast<uint64_t>((kk * 16 * 128) >> 4), idO,
                               (!first_pv[t] || kk > 0) ? 1u : 0u);
            }
            if (!ok) break;
            first_pv[t] = false;
            mma_commit_lead(lead, &pv_done[t]);
            ++pv_cnt[t];
            const int next = k + j.step();
            if (next < j.stop(t)) ok = issue_S(t, next);
          }
          if (ok) mma_commit_lead(lead, &kv_empty[slot(vp)]);  // V free after its P V products
        }
        base += 2 * (j.k1 - j.k0);
      }
      mma_commit_lead(lead, drain);
      if (lane == 0) drain_wait(drain, 0, p.status);
      __syncwarp();
    } else if (warp == 10) {
      // ---------------------------------------------------------- pieces
      const int64_t share_lo = share.lo;
      Piece pc;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int i = n % C::kQueue;
        const int64_t lo = share.lo;
        const bool more = next_piece(p, split, share, pc);
        ok = wait(&job_empty[i], static_cast<uint32_t>((n / C::kQueue) & 1) ^ 1u);
        if (!ok) break;
        if (lane == 0) {
          const int rec = 2 * blockIdx.x + (lo == share_lo ? 0 : 1);
          if (more && pc.k0 == 0 && pc.k1 < pc.tiles)
            scratch.record[blockIdx.x] = make_record(p, split, share, pc, blockIdx.x, rec);
          if (more) jobs[i] = make_job(p, split, tiles, pc, rec);
          else jobs[i].b = -1;
          mbar_arrive(&job_full[i]);
        }
        if (!more) break;
      }
      __syncwarp();
    } else if constexpr (MASK) {
      // ---------------------------------------------------- mask bits (warp 11)
      int turn = 0;  // new tiles so far
      bool ok = true;
      Job j;
      for (int n = 0; ok && take_job(n, j); ++n) {
        leave_job(n);
        const int tokens = (j.rows + p.group - 1) / p.group;
        const int64_t row0 = j.first + j.rt * split.rows / p.group;
        for (int k = max(j.k0, j.cached); k < j.k1 && ok; ++k, ++turn) {
          const int buf = turn & 1, here = j.here(split, k);
          ok = wait(&bits_empty[buf], static_cast<uint32_t>((turn >> 1) & 1) ^ 1u);
          if (!ok) break;
          for (int i = lane; i < tokens; i += 32) {
            const uint8_t* const row = p.mask + (row0 + i) * p.mask_stride + ((k - j.cached) << split.new_shift);
            uint32_t b[4];
            if (p.mask_align >= 16) mask_row<16>(row, here, b);
            else if (p.mask_align >= 4) mask_row<4>(row, here, b);
            else mask_row<1>(row, here, b);
            s_bits[buf * C::kBits + i] = make_uint4(b[0], b[1], b[2], b[3]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bits_full[buf]);
        }
      }
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
    int meets = 0;  // phases of `met` so far
    int turns = 0;  // new tiles of the pieces before
    bool ok = true;
    for (int n = 0; ok; ++n) {
      ok = wait(&job_full[n % C::kQueue], static_cast<uint32_t>((n / C::kQueue) & 1));
      if (!ok) break;
      // Read in place: only what every tile needs stays in registers.
      const Job& j = jobs[n % C::kQueue];
      if (j.b < 0) break;
      const int k0 = j.k0, cached_end = j.cached, held = j.held, count = j.count;
      const bool alone = j.alone;
      const int row0 = alone ? 0 : t * tiles.rows;  // of the item
      const int rows = min(tiles.rows, j.rows - row0);
      const int at = j.rt * split.rows + row0 + min(r, max(rows, 1) - 1);
      const int token = at / p.group;
      const bool busy = (warp & 3) * 32 < rows;  // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f;
      const int from = j.from(t), stop = j.stop(t);
      for (int k = from; k < stop && ok; k += alone ? 2 : 1, ++steps) {
        const bool cached = k < cached_end;
        const int here = cached ? min(kTileKeys, held - (k << split.keys_shift))
                                : min(1 << split.new_shift, count - ((k - cached_end) << split.new_shift));
        ok = wait(&s_full[t], static_cast<uint32_t>(steps & 1));
        if (!ok) break;
        tc_fence_after();
        if (__builtin_expect(here < kTileKeys, 0) && (t == 0 || !j.takes(0, k))) {
          // Accumulator 0's products of a tile come first.  The tile before in
          // V's slot has been used (S of this one is complete), so the phase
          // waited for is the slot's next.
          const int vp = base + j.template v_place<ALONE>(k);
          ok = wait(&kv_full[slot(vp)], par(vp));
          if (!ok) break;
          if (r >= here) {
            uint8_t* const v = sKV + slot(vp) * C::kTile + r * 128;
#pragma unroll
            for (int c = 0; c < C::kHalves; ++c)
#pragma unroll
              for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(v + c * C::kBox + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        int buf = 0;
        if constexpr (MASK) {
          if (!cached) {
            // The turn of this tile among the block's new tiles.
            const int turn = turns + k - max(k0, cached_end);
            buf = turn & 1;
            ok = wait(&bits_full[buf], static_cast<uint32_t>((turn >> 1) & 1));
            if (!ok) break;
          }
        }
        float s[128];
        if (busy) {
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
          // Bits of the keys that this row does not see.
          uint32_t hide[4] = {0, 0, 0, 0};
          const int lim = cached || MASK ? here : min(here, token - ((k - cached_end) << split.new_shift) + 1);
          if (lim < kTileKeys) {
#pragma unroll
            for (int w = 0; w < 4; ++w) hide[w] = lim >= 32 * w + 32 ? 0u : 0xffffffffu << max(lim - 32 * w, 0);
          }
          if constexpr (MASK) {
            if (!cached) {
              const uint4 b = s_bits[buf * C::kBits + (row0 + min(r, max(rows, 1) - 1)) / p.group];
              hide[0] |= b.x, hide[1] |= b.y, hide[2] |= b.z, hide[3] |= b.w;
            }
          }
          if (__builtin_expect(__any_sync(0xffffffffu, (hide[0] | hide[1] | hide[2] | hide[3]) != 0), 0)) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if ((hide[c >> 5] >> (c & 31)) & 1u) s[c] = hidden;
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
          if (__builtin_expect(__any_sync(0xffffffffu, k != from && alpha != 1.f), 0)) {
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
          l *= alpha;
        }
        if constexpr (MASK) {
          if (!cached) {  // alone: the other group does not read this tile's bits
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&bits_empty[buf]);
              if (alone) mbar_arrive(&bits_empty[buf]);
            }
          }
        }
        // Weights in two halves, each published as it is stored.
        const float sub = m == -INFINITY ? 0.f : C::kShift - m;
        const uint64_t sl2x2 = f2_pack(sl2, sl2), subx2 = f2_pack(sub, sub);
        uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (busy) {
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
            tmem_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * h + t]);
        }
        float q0, q1;
        f2_unpack(f2_add(sum0, sum1), q0, q1);
        l += q0 + q1;
      }
      if (!ok) break;
      base += 2 * (j.k1 - j.k0);
      turns += max(0, j.k1 - max(j.k0, j.cached));
      // ------------------------------------------------------------ a piece ends
      const bool has = from < stop, whole = j.whole;
      if (has && !wait(&pv_done[t], static_cast<uint32_t>((steps - 1) & 1))) break;
      tc_fence_after();
      // Alone: columns [D/2 t, D/2 t + D/2) of both accumulators; else all of its own.
      float f0 = 1.f, f1 = 0.f, mm = m, ll = l;
      if (j.alone) {
        // Both groups' maxima and sums meet in this piece's scratch slot (shared
        // memory is full).
        scratch.m[j.rec * 256 + t * 128 + r] = m;
        scratch.l[j.rec * 256 + t * 128 + r] = l;
        __threadfence();  // read past L1
        tc_fence_before();
        mbar_arrive(met);
        if (!wait(met, static_cast<uint32_t>(meets++ & 1))) break;
        tc_fence_after();
        const float m0 = __ldcg(scratch.m + j.rec * 256 + r), m1 = __ldcg(scratch.m + j.rec * 256 + 128 + r);
        mm = fmaxf(m0, m1);
        f0 = mm == -INFINITY ? 0.f : ex2(m0 - mm);
        f1 = mm == -INFINITY ? 0.f : ex2(m1 - mm);
        ll = f0 * __ldcg(scratch.l + j.rec * 256 + r) + f1 * __ldcg(scratch.l + j.rec * 256 + 128 + r);
        mbar_arrive(met);  // both groups have read the slot
        if (!wait(met, static_cast<uint32_t>(meets++ & 1))) break;
      }
      const bool live = r < rows;
      const bool none = ll == 0.f;  // no weight: 0 or 0 / 0 whatever the accumulator holds
      const float inv = whole && live ? over(p, ll, j.held, j.first, j.count, token) : 1.f;
      const float w0 = f0 * inv, w1 = f1 * inv, nothing = whole && none ? inv : 0.f;
      const int head = j.h * p.group + at % p.group;
      T* const orow = static_cast<T*>(p.o) + static_cast<int64_t>(j.first + token) * p.o_st + head * p.o_sh;
      float4* const srow = scratch.o + static_cast<int64_t>(j.rec) * (D / 4) * 256 + row0 + r;
      const uint32_t tA = j.alone ? tmem + lane_off + 256 : tO;
      const bool two = j.alone && j.k1 - j.k0 > 1, any = j.alone || has;
      const int c_lo = j.alone ? t * (D / 2) : 0, c_hi = j.alone ? c_lo + D / 2 : D;
      if (busy) {
        for (int c = c_lo; c < c_hi; c += 32) {
          uint32_t a[32];
          tmem_ld32(tA + c, a);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            a[i] = any && !none ? __float_as_uint(__uint_as_float(a[i]) * w0) : __float_as_uint(nothing);
          if (two) {
            uint32_t b[32];
            tmem_ld32(tA + D + c, b);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!none) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), w1, __uint_as_float(a[i])));
          }
          if (live && whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(orow + c)[i] =
                  make_uint4(pack2<F16>(__uint_as_float(a[8 * i]), __uint_as_float(a[8 * i + 1])),
                             pack2<F16>(__uint_as_float(a[8 * i + 2]), __uint_as_float(a[8 * i + 3])),
                             pack2<F16>(__uint_as_float(a[8 * i + 4]), __uint_as_float(a[8 * i + 5])),
                             pack2<F16>(__uint_as_float(a[8 * i + 6]), __uint_as_float(a[8 * i + 7])));
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              srow[(c / 4 + i) * 256] = make_float4(__uint_as_float(a[4 * i]), __uint_as_float(a[4 * i + 1]),
                                                    __uint_as_float(a[4 * i + 2]), __uint_as_float(a[4 * i + 3]));
          }
        }
      }
      tc_fence_before();
      mbar_arrive(o_free);
      if (live && (!j.alone || t == 0)) {
        if (!whole) {
          scratch.m[j.rec * 256 + row0 + r] = mm;
          scratch.l[j.rec * 256 + row0 + r] = ll;
        } else if (p.lse) {
          p.lse[static_cast<int64_t>(j.first + token) * p.Hq + head] =
              none ? -INFINITY : (mm - C::kShift + log2f(ll)) * kLn2;
        }
      }
      leave_job(n);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// The join of this kernel's cut items: block (c, y) takes 32 query rows of the
// cut item that begins in block c of the first kernel, if any.  A lane is a
// row (as the first kernel stores them), a warp has D / 4 / 16 times four
// columns; an item has few pieces (all of them only where a single item fills
// the GPU), so a thread reads four of each column at once and adds in order.
constexpr int kJoinThreads = 512, kJoinRows = 32;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    tree_tc_join(const __grid_constant__ Params p, const Scratch scratch) {
  using C = Cfg<T, D, false, false>;
  constexpr int kCols = D / 4 / (kJoinThreads / 32);
  grid_wait();
  grid_release();
  const int c = blockIdx.x, lane = threadIdx.x & 31, col = (threadIdx.x >> 5) * kCols;
  const Record rec = scratch.record[c];
  const int row = blockIdx.y * kJoinRows + lane;
  if (rec.pieces == 0 || row >= rec.rows) return;
  const int n = rec.pieces;
  float top = -INFINITY, sum = 0.f;
  float4 a[kCols] = {};
  for (int i0 = 0; i0 < n; i0 += 4) {
    float m[4], l[4];
    float4 y[4][kCols];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
      for (int k = 0; k < kCols; ++k) y[x][k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + x < n) {
        const int64_t s = i0 + x == 0 ? rec.slot : 2 * (c + i0 + x);
        m[x] = scratch.m[s * 256 + row];
        l[x] = scratch.l[s * 256 + row];
#pragma unroll
        for (int k = 0; k < kCols; ++k) y[x][k] = scratch.o[(s * (D / 4) + col + k) * 256 + row];
      }
    }
    const float high = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
    const float base = base_of(high), f = ex2(top - base);
    top = high;
    sum *= f;
#pragma unroll
    for (int k = 0; k < kCols; ++k) a[k].x *= f, a[k].y *= f, a[k].z *= f, a[k].w *= f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float w = ex2(m[x] - base);
      sum += w * l[x];
#pragma unroll
      for (int k = 0; k < kCols; ++k)
        a[k].x += w * y[x][k].x, a[k].y += w * y[x][k].y, a[k].z += w * y[x][k].z, a[k].w += w * y[x][k].w;
    }
  }
  const int at = rec.row + row;
  const float inv = over(p, sum, rec.held, rec.first, rec.count, at / p.group);
  const int token = rec.first + at / p.group, head = rec.h * p.group + at % p.group;
  T* const out = static_cast<T*>(p.o) + token * p.o_st + head * p.o_sh + 4 * col;
#pragma unroll
  for (int k = 0; k < kCols; ++k)
    reinterpret_cast<uint2*>(out)[k] =
        make_uint2(pack2<C::F16>(a[k].x * inv, a[k].y * inv), pack2<C::F16>(a[k].z * inv, a[k].w * inv));
  if (col == 0 && p.lse)
    p.lse[static_cast<int64_t>(token) * p.Hq + head] =
        sum == 0.f ? -INFINITY : (top - C::kShift + log2f(sum)) * kLn2;
}

}  // namespace tc

}  // namespace attn_tree
