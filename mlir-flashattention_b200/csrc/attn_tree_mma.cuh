// attn_tree_mma.cuh — attn_tree_fwd for few query rows per kv-head (decode,
// small drafts), and the join of items cut between blocks.
//
// With 16 query rows a cached key of D values costs 4 * 16 * D operations for
// 4 * D bytes: 16 a byte against the 250 a byte that this GPU can do per byte
// it reads, so the kernel is bound by the cache's bytes and everything here
// serves to keep loads in flight: a team is one warp that issues TMA loads of
// page segments into a ring of tiles (16 KB of K and of V each, 128-byte
// swizzle) and four warps that each take a quarter of a tile's keys, with their
// own running maxima, sums and accumulators, and meet only when a piece ends.
// A block is two teams and fills an SM; its registers are divided so that the
// reading warps have 224 (setmaxnreg).  Tensor cores by mma.sync m16n8k16:
// operands go from shared memory to registers, so 16 rows cost 16 rows (a
// 128-row accumulator in tensor memory would be 1/8 used and its softmax one
// warp's work).  MT = 1, 2 or (D = 64) 3 16-row tiles share every key that is
// read; more rows are more items.  From there on the warps' own instructions
// bound it (64 rows at D = 64 and 8000 keys: 219 us, 212 us in attn_tree_tc.cuh;
// 128 rows 378 and 214).  64 requests with 8192 keys, 8 kv-heads, bf16: 197 to
// 201 us from one GPU to another, 6.0 to 6.1 TB/s.
//
// An e4m3 cache is met in f16: e4m3 values are f16 values, and a bf16 row of q
// is scaled by the power of two that brings its largest value to 2^14..2^15:
// its 8 bits are then exact in f16 down to 2^-31 of that value, and below that
// the row is rounded to f16's smallest step, off by at most 2^-39 of it.  New keys and values are 16-bit
// and met in their own type.  A tile is twice as many keys, so a warp has two
// groups of 16 at once (MT = 1): the conversions' latency, not their number,
// was the bound.  100 requests with 8192 keys: 205 us, 4.4 TB/s; the loads
// alone take 162 us, the readers' instructions are the rest.
//
// Weights are rounded to the operands' type for P V.  In bf16 a rounding by
// 2^-8 would double the error of the result, whose own rounding is the same
// size: for one row tile P goes in as two bf16 parts, p and p - bf16(p), for
// twice the small product's work.
#pragma once

#include <type_traits>

#include "attn_tree.cuh"
#include "sm100_ptx.cuh"

namespace attn_tree {

constexpr int kMmaWarps = 4, kMmaTeams = 2;
constexpr int kMmaThreads = 384;  // two teams of readers; warps 8 and 9 load, 10 and 11 idle
constexpr int kMmaRegsRead = 224, kMmaRegsLoad = 56;
constexpr int kMmaRegPool = 256 * kMmaRegsRead + 128 * kMmaRegsLoad;

template <typename T, typename TC, int D, int MT>
struct MmaCfg {
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static constexpr bool FP8 = sizeof(TC) == 1;
  static constexpr int kRows = 16 * MT;
  static constexpr int kKeysShift = FP8 ? 7 : 6;       // cached keys of a tile, log2
  static constexpr int kGroups = (1 << kKeysShift) / (16 * kMmaWarps);  // of 16 keys, a warp
  static constexpr int kAtOnce = MT == 1 ? kGroups : 1;
  static constexpr int kRowBytes = D * static_cast<int>(sizeof(TC));
  static constexpr int kNewRowBytes = D * 2;
  static constexpr int kTile = kRowBytes << kKeysShift;  // K or V of a stage
  static constexpr int kStages = 98304 / (2 * kTile);
  static constexpr int kNewShift = 6;                  // most new keys of a tile, log2
  static constexpr int kJoinCols = MT == 1 ? 32 : 16;  // columns that the warps join at a time
  static constexpr int kJoin = kMmaWarps * 16 * kJoinCols * 4;
  // Weights are kept times 2^kShift: in f16 they stay normal down to 2^-22.
  static constexpr float kShift = (FP8 || F16) ? 8.f : 0.f;
  static constexpr bool kTwoParts = !F16 && !FP8 && MT == 1;  // P as two bf16 parts
  static constexpr int kTeam = kStages * 2 * kTile + kRows * D * 2 + kJoin;
  static constexpr size_t kSmem = 1024 + kMmaTeams * kTeam;
  static_assert(kTeam % 1024 == 0, "the rings start on swizzle periods");
  static_assert(kSmem + 4096 <= 232448, "shared memory budget");
  static_assert((kNewRowBytes << kNewShift) <= kTile, "new keys of a stage");
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 values (low byte first) as two f16 values: exact.
__device__ __forceinline__ uint32_t f16_of_e4m3(uint32_t two) {
  uint32_t r;
  const uint16_t h = static_cast<uint16_t>(two);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  return r;
}

// Two weights as the A operand's pair, and what the rounding left of them.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  return F16 ? attn_sm100::pack_f16(x, y) : attn_sm100::pack_bf16(x, y);
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x,
                                            int y, int z, int w, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v),
      "r"(attn_sm100::smem_u32(bar))
      : "memory");
}

// Programmatic launches: what the kernel before in the stream wrote may be
// read after grid_wait; the kernel behind may be set up after grid_release (it
// waits in turn for this one's end).
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The four reading warps of a team meet.
__device__ __forceinline__ void readers_sync(int team) {
  __syncwarp();
  asm volatile("barrier.sync %0, 128;" ::"r"(team + 1) : "memory");
}

template <typename T, typename TC, int D, int MT>
__global__ void __launch_bounds__(kMmaThreads, 1)
    tree_mma_kernel(const __grid_constant__ CUtensorMap map_kc, const __grid_constant__ CUtensorMap map_vc,
                    const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_vn,
                    const __grid_constant__ Params p, const Split split, const Scratch scratch,
                    const int min_units) {
  using C = MmaCfg<T, TC, D, MT>;
  constexpr bool F16 = C::F16, FP8 = C::FP8;
  constexpr int NG = C::kAtOnce;
  constexpr int kSteps = D / 16;    // k-steps of Q K
  constexpr int kTilesD = D / 8;    // n-tiles of P V
  constexpr bool kHoldQ = MT == 1;  // q's fragments stay in registers
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t sh_full[kMmaTeams][C::kStages], sh_empty[kMmaTeams][C::kStages];
  __shared__ volatile int abort_flag;
  __shared__ float sh_m[kMmaTeams][kMmaWarps][C::kRows], sh_l[kMmaTeams][kMmaWarps][C::kRows];
  __shared__ float sh_unit[kMmaTeams][C::kRows];

  const int lane = threadIdx.x & 31, block_warp = threadIdx.x >> 5;
  const int team = block_warp < 8 ? block_warp >> 2 : block_warp & 1;
  const int tid = threadIdx.x & 127, warp = tid >> 5;  // of a reader in its team
  const int sid = kMmaTeams * blockIdx.x + team;       // this team's share
  uint64_t* const full = sh_full[team];
  uint64_t* const empty = sh_empty[team];
  float (*const warp_m)[C::kRows] = sh_m[team];
  float (*const warp_l)[C::kRows] = sh_l[team];
  float* const q_unit = sh_unit[team];  // e4m3: the power of two that a row of q was divided by
  uint8_t* smem = raw + ((1024u - (attn_sm100::smem_u32(raw) & 1023u)) & 1023u) + team * C::kTeam;
  const uint32_t s_ring = attn_sm100::smem_u32(smem);
  uint8_t* const s_q = smem + C::kStages * 2 * C::kTile;  // [rows][D] of T, chunks swizzled
  float* const s_join = reinterpret_cast<float*>(s_q + C::kRows * D * 2);

  if (threadIdx.x == 0) {
    for (int t = 0; t < kMmaTeams; ++t)
      for (int s = 0; s < C::kStages; ++s) {
        attn_sm100::mbar_init(&sh_full[t][s], 1);
        attn_sm100::mbar_init(&sh_empty[t][s], kMmaWarps);
      }
    abort_flag = 0;
    attn_sm100::fence_mbar_init();
    attn_sm100::fence_proxy_async_smem();
  }
  grid_wait();
  grid_release();
  if (threadIdx.x < kMmaTeams) scratch.record[kMmaTeams * blockIdx.x + threadIdx.x].pieces = 0;
  Share share = find_share<kMmaTeams>(p, split, min_units, team);
  __syncthreads();
  const int64_t share_lo = share.lo;
  Piece pc;

  if (block_warp >= 8) {
    attn_sm100::setmaxnreg_dec<kMmaRegsLoad>();
    if (block_warp >= 10) return;
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      attn_sm100::prefetch_tmap(&map_kc);
      attn_sm100::prefetch_tmap(&map_vc);
      attn_sm100::prefetch_tmap(&map_kn);
      attn_sm100::prefetch_tmap(&map_vn);
    }
    const int seg_shift = min(p.page_shift, split.keys_shift);  // rows of a page segment, log2
    const int seg_bytes = C::kRowBytes << seg_shift;
    int n = 0;  // stages filled
    bool ok = true;
    while (ok && next_piece(p, split, share, pc)) {
      const int32_t* const row = p.table + pc.b * p.table_stride;
      auto segments = [&](int k) {
        return (min(1 << split.keys_shift, pc.r.held - (k << split.keys_shift)) + (1 << seg_shift) - 1) >> seg_shift;
      };
      auto page_of = [&](int k) {  // of this lane's segment
        if (k >= min(pc.cached, pc.k1) || lane >= segments(k)) return 0;
        return row[((k << split.keys_shift) + (lane << seg_shift)) >> p.page_shift];
      };
      int page_next = page_of(pc.k0);
      for (int k = pc.k0; k < pc.k1 && ok; ++k, ++n) {
        const int s = n % C::kStages;
        const uint32_t u = static_cast<uint32_t>(n / C::kStages);
        const bool cached = k < pc.cached;
        const int first = cached ? k << split.keys_shift : (k - pc.cached) << split.new_shift;
        const int segs = cached ? segments(k) : 1;
        int page = page_next, at = 0;
        page_next = page_of(k + 1);  // a tile ahead of its use
        if (cached && lane < segs) {
          at = (first + (lane << seg_shift)) & ((1 << p.page_shift) - 1);
          if (page < 0 || page >= p.num_pages) {
            atomicCAS(p.status, 0, ATTN_ERR_INVALID);
            page = max(p.num_pages, 1);  // outside the map: zeros
          }
        }
        ok = __all_sync(0xffffffffu, attn_sm100::mbar_wait_bounded(&empty[s], (u & 1u) ^ 1u, &abort_flag,
                                                                  p.status, kWaitLimitNs));
        if (!ok) break;
        const uint32_t kd = s_ring + s * 2 * C::kTile, vd = kd + C::kTile;
        if (lane == 0)
          attn_sm100::mbar_arrive_expect_tx(
              &full[s], 2 * (cached ? segs * seg_bytes : C::kNewRowBytes << split.new_shift));
        __syncwarp();
        if (lane < segs) {
          if (cached) {
            tma_load_5d(kd + lane * seg_bytes, &map_kc, &full[s], 0, at, 0, pc.h, page);
            tma_load_5d(vd + lane * seg_bytes, &map_vc, &full[s], 0, at, 0, pc.h, page);
          } else {
            tma_load_5d(kd, &map_kn, &full[s], 0, pc.r.first + first, 0, pc.h, 0);
            tma_load_5d(vd, &map_vn, &full[s], 0, pc.r.first + first, 0, pc.h, 0);
          }
        }
      }
    }
    if (!ok && lane == 0) {  // every copy in flight lands before the block may end
      for (int s = 0; s < C::kStages && s < n; ++s) {
        int never = 0;
        const uint32_t armed = static_cast<uint32_t>((n - 1 - s) / C::kStages);
        attn_sm100::mbar_wait_bounded(&full[s], armed & 1u, &never, p.status, kWaitLimitNs);
      }
    }
    return;
  }

  attn_sm100::setmaxnreg_inc<kMmaRegsRead>();
  // ------------------------------------------------------------- four readers
  const int quad = lane & 3, grp = lane >> 2;
  const uint32_t s_q32 = attn_sm100::smem_u32(s_q);
  const float scale2 = p.scale * kLog2e;
  // Where a lane reads in a group of 16 keys: e4m3 keys (row grp, chunk quad),
  // e4m3 values (rows 2 quad and 2 quad + 1, chunk grp), and the addresses that
  // it gives ldmatrix for 16-bit keys and values.
  const uint32_t lane_k = grp * 128 + ((quad ^ grp) * 16);
  const uint32_t lane_v0 = 2 * quad * 128 + ((grp ^ (2 * quad)) * 16);
  const uint32_t lane_v1 = (2 * quad + 1) * 128 + ((grp ^ (2 * quad + 1)) * 16);
  const uint32_t lane_k16 = ((lane & 7) + 8 * (lane >> 4)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) * 16);
  const uint32_t lane_v16 = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);
  int n = 0;
  bool ok = true;
  while (next_piece(p, split, share, pc)) {
    const int row0 = pc.rt * C::kRows;  // the item's first row in the request
    const int rows = static_cast<int>(
        min(static_cast<int64_t>(C::kRows), static_cast<int64_t>(pc.r.count) * p.group - row0));
    // q rows to shared memory (rows behind the last: zeros), 8 threads a row; all
    // loads before the first store.
    uint4 q_in[MT][D / 64];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = 16 * mt + (tid >> 3), at = row0 + r;
      const T* const src = static_cast<const T*>(p.q) + static_cast<int64_t>(pc.r.first + at / p.group) * p.q_st +
                           (pc.h * p.group + at % p.group) * p.q_sh;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        q_in[mt][c] = make_uint4(0, 0, 0, 0);
        if (r < rows) q_in[mt][c] = reinterpret_cast<const uint4*>(src)[(tid & 7) + 8 * c];
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = 16 * mt + (tid >> 3);
      const uint4 (&v)[D / 64] = q_in[mt];
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<uint4*>(s_q + r * D * 2 + ((((tid & 7) + 8 * c) ^ (r & 7)) * 16)) = v[c];
      if constexpr (FP8 && !F16) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
        }
        for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // The power of two of the row's largest value over 2^14; 1 for a row
        // of zeros, and at most 2^113 (an infinite value stays infinite).
        int e = static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 14;
        e = top == 0.f ? 127 : min(max(e, 1), 240);
        if ((tid & 7) == 0) q_unit[r] = __uint_as_float(static_cast<uint32_t>(e) << 23);
      }
    }
    readers_sync(team);
    // A fragments of 16 rows of q and one k-step, in q's own type and order.
    auto q_frag = [&](uint32_t (&a)[4], int mt, int s) {
      const int r = 16 * mt + (lane & 7) + 8 * ((lane >> 3) & 1), chunk = 2 * s + (lane >> 4);
      ldmatrix4(a, s_q32 + r * D * 2 + ((chunk ^ (r & 7)) * 16));
    };
    // The same in f16 and in the order of d in which a thread finds 16 of an
    // e4m3 key's values in one load: for k-step s, k = 2 quad + {0, 1} and
    // 2 quad + 8 + {0, 1} are the 4 values from d on.
    auto q_frag8 = [&](uint32_t (&a)[4], int mt, int s) {
      const int d = (s >> 2) * 64 + quad * 16 + (s & 3) * 4;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 16 * mt + grp + 8 * x;
        const uint2 w = *reinterpret_cast<const uint2*>(s_q + r * D * 2 + (((d >> 3) ^ (r & 7)) * 16) + (d & 7) * 2);
        if constexpr (F16) {
          a[x] = w.x, a[2 + x] = w.y;
        } else {
          const float inv = 1.f / q_unit[r];  // a power of two
          a[x] = attn_sm100::pack_f16(__uint_as_float(w.x << 16) * inv, __uint_as_float(w.x & 0xffff0000u) * inv);
          a[2 + x] = attn_sm100::pack_f16(__uint_as_float(w.y << 16) * inv, __uint_as_float(w.y & 0xffff0000u) * inv);
        }
      }
    };
    uint32_t qa[kHoldQ ? kSteps : 1][4];
    if constexpr (kHoldQ) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if constexpr (FP8) q_frag8(qa[s], 0, s);
        else q_frag(qa[s], 0, s);
      }
    }
    float kd = scale2, vd = 1.f;
    if constexpr (FP8) {
      kd *= p.k_descale * (p.k_descale_heads ? p.k_descale_heads[pc.h] : 1.f);
      vd = p.v_descale * (p.v_descale_heads ? p.v_descale_heads[pc.h] : 1.f);
    }
    float o[MT][kTilesD][4];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -INFINITY, l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
      for (int t = 0; t < kTilesD; ++t) o[mt][t][0] = o[mt][t][1] = o[mt][t][2] = o[mt][t][3] = 0.f;
    }
    bool scaled = !FP8;  // o is in units of the cached values until the new ones come

    for (int k = pc.k0; k < pc.k1; ++k, ++n) {
      const int st = n % C::kStages;
      const uint32_t u = static_cast<uint32_t>(n / C::kStages);
      if (ok)
        ok = __all_sync(0xffffffffu, attn_sm100::mbar_wait_bounded(&full[st], u & 1u, &abort_flag, p.status,
                                                                   kWaitLimitNs));
      const uint32_t ks = s_ring + st * 2 * C::kTile, vs = ks + C::kTile;
      const bool cached = k < pc.cached;
      const int first = cached ? k << split.keys_shift : (k - pc.cached) << split.new_shift;
      const int here = cached ? min(1 << split.keys_shift, pc.r.held - first)
                              : min(1 << split.new_shift, pc.r.count - first);
      const int seg_shift = cached ? min(p.page_shift, split.keys_shift) : split.new_shift;
      // This warp's groups of 16 keys, NG at a time (of a new tile: one).
      const int kb_end = cached ? 16 * C::kGroups * (warp + 1) : 16 * (warp + 1);
      for (int kb = cached ? 16 * C::kGroups * warp : 16 * warp; kb < min(kb_end, here) && ok; kb += 16 * NG) {
        float s[NG][MT][2][4];
        // The group's first row in its page segment.  Groups start on multiples
        // of 16 rows, so the swizzle of a row goes by the lane alone.
        uint32_t kbase[NG], vbase[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int j = kb + 16 * g, seg = j >> seg_shift;
          const uint32_t off = seg * ((cached ? C::kRowBytes : C::kNewRowBytes) << seg_shift) +
                               (j & ((1 << seg_shift) - 1)) * 128;
          kbase[g] = ks + off, vbase[g] = vs + off;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[g][mt][h][0] = s[g][mt][h][1] = s[g][mt][h][2] = s[g][mt][h][3] = 0.f;
        }
        if (FP8 && cached) {
          // Key r (a row of 128 bytes): thread quad loads 16 values at 16 quad
          // and 16 at 64 + 16 quad (see q_frag8).
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint4 w[NG][2];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                w[g][h] = lds128(kbase[g] + h * 1024 + (lane_k ^ (64 * c)));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                uint32_t a[4];
                if constexpr (kHoldQ) a[0] = qa[4 * c + e][0], a[1] = qa[4 * c + e][1], a[2] = qa[4 * c + e][2], a[3] = qa[4 * c + e][3];
                else q_frag8(a, mt, 4 * c + e);
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const uint32_t ww = e == 0 ? w[g][h].x : e == 1 ? w[g][h].y : e == 2 ? w[g][h].z : w[g][h].w;
                    mma16816<true>(s[g][mt][h], a, f16_of_e4m3(ww), f16_of_e4m3(ww >> 16));
                  }
              }
            }
          }
        } else {
#pragma unroll
          for (int x = 0; x < kSteps; ++x) {
#pragma unroll
            for (int g = 0; g < (FP8 ? 1 : NG); ++g) {
              uint32_t b[4];
              ldmatrix4(b, kbase[g] + (x >> 2) * (128 << seg_shift) + (lane_k16 ^ (32 * (x & 3))));
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                uint32_t a[4];
                if constexpr (kHoldQ && !FP8) a[0] = qa[x][0], a[1] = qa[x][1], a[2] = qa[x][2], a[3] = qa[x][3];
                else q_frag(a, mt, x);
                mma16816<F16>(s[g][mt][0], a, b[0], b[1]);
                mma16816<F16>(s[g][mt][1], a, b[2], b[3]);
              }
            }
          }
        }
        // Scale, then the mask (selected after the scale: what a masked key's
        // score was does not matter), then weights: rows grp, grp + 8 of each
        // 16; keys 2 quad + {0, 1} of each 8.  All rows' maxima first, so that
        // their exchanges overlap, and one vote on whether any moved.
        const bool tail = kb + 16 * NG > here;
        float top[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float f = FP8 && cached ? (F16 ? kd : kd * q_unit[16 * mt + grp + 8 * x]) : scale2;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
              for (int h = 0; h < 2; ++h) s[g][mt][h][2 * x] *= f, s[g][mt][h][2 * x + 1] *= f;
          }
        if (!cached) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int r = 16 * mt + grp + 8 * x;
              const bool live = r < rows;
              const int i = (row0 + r) / p.group;  // token of the request
              const uint8_t* const mrow =
                  p.mask + static_cast<int64_t>(pc.r.first + (live ? i : 0)) * p.mask_stride + first;
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int j = kb + 8 * h + 2 * quad + e;
                  bool hide = j >= here || !live;
                  if (!hide) hide = p.mask ? mrow[j] != 0 : first + j > i;
                  if (hide) s[0][mt][h][2 * x + e] = -INFINITY;
#pragma unroll
                  for (int g = 1; g < NG; ++g) s[g][mt][h][2 * x + e] = -INFINITY;
                }
            }
        } else if (tail) {
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (kb + 16 * g + 8 * h + 2 * quad + e >= here) {
#pragma unroll
                  for (int mt = 0; mt < MT; ++mt) s[g][mt][h][e] = s[g][mt][h][2 + e] = -INFINITY;
                }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            top[mt][x] = m[mt][x];
#pragma unroll
            for (int g = 0; g < NG; ++g)
              top[mt][x] = fmaxf(top[mt][x], fmaxf(fmaxf(s[g][mt][0][2 * x], s[g][mt][0][2 * x + 1]),
                                                   fmaxf(s[g][mt][1][2 * x], s[g][mt][1][2 * x + 1])));
          }
#pragma unroll
        for (int d = 1; d <= 2; d *= 2)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              top[mt][x] = fmaxf(top[mt][x], __shfl_xor_sync(0xffffffffu, top[mt][x], d));
        // The running maxima move when one of a warp's rows grows by 2^4 past
        // its own (weights stay below 2^(kShift + 4)): most tiles rescale nothing.
        bool moved = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) moved = moved || top[mt][0] > m[mt][0] + 4.f || top[mt][1] > m[mt][1] + 4.f;
        if (!__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) top[mt][0] = m[mt][0], top[mt][1] = m[mt][1];
        } else {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float a = top[mt][x] == -INFINITY ? 1.f : attn_sm100::ex2(m[mt][x] - top[mt][x]);
              l[mt][x] *= a;
#pragma unroll
              for (int t = 0; t < kTilesD; ++t) o[mt][t][2 * x] *= a, o[mt][t][2 * x + 1] *= a;
              m[mt][x] = top[mt][x];
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float sub = (top[mt][x] == -INFINITY ? 0.f : top[mt][x]) - C::kShift;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& v = s[g][mt][h][2 * x + e];
                  v = attn_sm100::ex2(v - sub);
                  l[mt][x] += v;
                }
          }
        if (!cached && !scaled) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int t = 0; t < kTilesD; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][t][e] *= vd;
          scaled = true;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (FP8 && !cached && g > 0) break;
          uint32_t a[MT][4], rest[MT][4];
          const bool p16 = F16 || (FP8 && cached);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float x0 = s[g][mt][y >> 1][2 * (y & 1)], x1 = s[g][mt][y >> 1][2 * (y & 1) + 1];
              a[mt][y] = p16 ? pack2<true>(x0, x1) : pack2<false>(x0, x1);
              if constexpr (C::kTwoParts)
                rest[mt][y] = pack2<false>(x0 - __uint_as_float(a[mt][y] << 16),
                                           x1 - __uint_as_float(a[mt][y] & 0xffff0000u));
            }
          // The values of keys that are not there are made 0 (their weights
          // are 0, but 0 times what lies in memory there need not be 0).
          const int j0 = kb + 16 * g + 2 * quad;
          if constexpr (FP8) {
            // Thread group grp loads 16 values of each of its four keys (2 quad,
            // + 1, + 8, + 9) at 16 grp; n-tile t is d = 16 n + t, n = 0..7.
            if (cached) {
              uint32_t w[4][4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint4 v = lds128(vbase[g] + (y >> 1) * 1024 + (y & 1 ? lane_v1 : lane_v0));
                w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
              }
              if (tail) {
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  if (j0 + (y & 1) + 8 * (y >> 1) >= here) w[y][0] = w[y][1] = w[y][2] = w[y][3] = 0u;
              }
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  const uint32_t lo = __byte_perm(w[0][c], w[1][c], z ? 0x7362 : 0x5140);
                  const uint32_t hi = __byte_perm(w[2][c], w[3][c], z ? 0x7362 : 0x5140);
                  const uint32_t b0 = f16_of_e4m3(lo), b1 = f16_of_e4m3(hi);
                  const uint32_t b2 = f16_of_e4m3(lo >> 16), b3 = f16_of_e4m3(hi >> 16);
#pragma unroll
                  for (int mt = 0; mt < MT; ++mt) {
                    mma16816<true>(o[mt][4 * c + 2 * z], a[mt], b0, b1);
                    mma16816<true>(o[mt][4 * c + 2 * z + 1], a[mt], b2, b3);
                  }
                }
            } else {
#pragma unroll
              for (int c = 0; c < 2; ++c) {  // 8 of the 16 values at a time
                uint32_t w[4][4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const int r = 2 * quad + (y & 1), chunk = 2 * grp + c;
                  const uint4 v = lds128(vbase[g] + (chunk >> 3) * (128 << seg_shift) + (y >> 1) * 1024 + r * 128 +
                                         (((chunk & 7) ^ r) * 16));
                  w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
                  if (j0 + (y & 1) + 8 * (y >> 1) >= here) w[y][0] = w[y][1] = w[y][2] = w[y][3] = 0u;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
                  const uint32_t b0 = __byte_perm(w[0][e >> 1], w[1][e >> 1], sel);
                  const uint32_t b1 = __byte_perm(w[2][e >> 1], w[3][e >> 1], sel);
#pragma unroll
                  for (int mt = 0; mt < MT; ++mt) mma16816<F16>(o[mt][8 * c + e], a[mt], b0, b1);
                }
              }
            }
          } else {
            const uint32_t live0 = (j0 < here ? 0xffffu : 0u) | (j0 + 1 < here ? 0xffff0000u : 0u);
            const uint32_t live1 = (j0 + 8 < here ? 0xffffu : 0u) | (j0 + 9 < here ? 0xffff0000u : 0u);
#pragma unroll
            for (int t = 0; t < kTilesD / 2; ++t) {
              uint32_t b[4];
              ldmatrix4t(b, vbase[g] + (t >> 2) * (128 << seg_shift) + (lane_v16 ^ (32 * (t & 3))));
              if (tail) b[0] &= live0, b[1] &= live1, b[2] &= live0, b[3] &= live1;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                mma16816<F16>(o[mt][2 * t], a[mt], b[0], b[1]);
                mma16816<F16>(o[mt][2 * t + 1], a[mt], b[2], b[3]);
                if constexpr (C::kTwoParts) {
                  mma16816<F16>(o[mt][2 * t], rest[mt], b[0], b[1]);
                  mma16816<F16>(o[mt][2 * t + 1], rest[mt], b[2], b[3]);
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) attn_sm100::mbar_arrive(&empty[st]);
    }

    // ---------------------------------------------------------- a piece ends
    const bool whole = pc.k0 == 0 && pc.k1 == pc.tiles;
    const int slot = 2 * sid + (share.lo - (pc.k1 - pc.k0) == share_lo ? 0 : 1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[mt][x] += __shfl_xor_sync(0xffffffffu, l[mt][x], 1);
        l[mt][x] += __shfl_xor_sync(0xffffffffu, l[mt][x], 2);
        if (quad == 0) warp_m[warp][16 * mt + grp + 8 * x] = m[mt][x], warp_l[warp][16 * mt + grp + 8 * x] = l[mt][x];
      }
    readers_sync(team);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float factor[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) top = fmaxf(top, warp_m[w][16 * mt + grp + 8 * x]);
        factor[x] = top == -INFINITY ? 0.f : attn_sm100::ex2(m[mt][x] - top);
        if (!scaled) factor[x] *= vd;
      }
      // The row that this thread writes, and its four columns of kJoinCols.
      constexpr int kPer = C::kJoinCols / 4;
      const int wr = 16 * mt + (tid / kPer & 15), wc = (tid % kPer) * 4;
      const bool writes = tid < 16 * kPer && wr < rows;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) top = fmaxf(top, warp_m[w][wr]);
      // A warp that met only scores that are no numbers has the maximum -inf and
      // a sum that is none: it must not be lost.
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) sum += attn_sm100::ex2(warp_m[w][wr] - base_of(top)) * warp_l[w][wr];
      const int at = row0 + wr;
      const int token = pc.r.first + at / p.group, head = pc.h * p.group + at % p.group;
      const float inv =
          whole && writes ? over(p, sum, pc.r.held, pc.r.first, pc.r.count, at / p.group) : 0.f;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += C::kJoinCols) {
        float* const mine = s_join + (warp * 16 + grp) * C::kJoinCols;  // + 8 rows
        // The accumulators of columns c0 .. c0 + kJoinCols - 1 (an e4m3 cache:
        // n-tile t is columns 16 n + t, so they are one thread's of each quad).
        if constexpr (FP8) {
          if (quad == c0 / 32) {
#pragma unroll
            for (int t = 0; t < kTilesD; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (C::kJoinCols == 32)
                  mine[(e >> 1) * 8 * C::kJoinCols + 16 * (e & 1) + t] = o[mt][t][e] * factor[e >> 1];
                else if ((e & 1) == (c0 / 16 & 1))
                  mine[(e >> 1) * 8 * C::kJoinCols + t] = o[mt][t][e] * factor[e >> 1];
              }
          }
        } else {
#pragma unroll
          for (int t = 0; t < C::kJoinCols / 8; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              *reinterpret_cast<float2*>(mine + x * 8 * C::kJoinCols + 8 * t + 2 * quad) =
                  make_float2(o[mt][c0 / 8 + t][2 * x] * factor[x], o[mt][c0 / 8 + t][2 * x + 1] * factor[x]);
        }
        readers_sync(team);
        if (writes) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kMmaWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(s_join + (w * 16 + (wr & 15)) * C::kJoinCols + wc);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          }
          if (whole) {
            *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.o_st + head * p.o_sh + c0 + wc) =
                make_uint2(pack2<F16>(x.x * inv, x.y * inv), pack2<F16>(x.z * inv, x.w * inv));
          } else {
            scratch.o[(static_cast<int64_t>(slot) * C::kRows + wr) * (D / 4) + (c0 + wc) / 4] = x;
          }
        }
        readers_sync(team);
      }
      if (writes && wc == 0) {
        if (whole) {
          if (p.lse)
            p.lse[static_cast<int64_t>(token) * p.Hq + head] =
                sum == 0.f ? -INFINITY : (top - C::kShift + log2f(sum)) * kLn2;
        } else {
          scratch.m[slot * C::kRows + wr] = top;
          scratch.l[slot * C::kRows + wr] = sum;
        }
      }
    }
    if (!whole && pc.k0 == 0 && tid == 0) scratch.record[sid] = make_record(p, split, share, pc, sid, slot);
  }
}

// Joins the pieces of the items that were cut: block (c, y) takes `rows_each`
// query rows of the cut item that begins in share c of the first kernel, if
// any.  What bounds it is latency, a record and then everything else at once:
// a thread has four columns of a row and every G-th piece of the item, brought
// to one maximum as it goes; the G parts meet in shared memory.  The order of
// the sums depends on the lengths alone, so a call gives the same bits every
// time.
constexpr int kJoinThreads = 256;

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads)
    tree_mma_join(const __grid_constant__ Params p, const Scratch scratch, const int rows_each, const float shift) {
  constexpr bool F16 = std::is_same<T, __half>::value;
  constexpr int kCols = D / 4, kParts = kJoinThreads / kCols;  // threads of a row; rows x G at once
  __shared__ float4 part_o[kJoinThreads];
  __shared__ float part_m[kJoinThreads], part_l[kJoinThreads];
  grid_wait();
  grid_release();
  const int c = blockIdx.x, tid = threadIdx.x, col = tid % kCols, part = tid / kCols;
  const Record rec = scratch.record[c];
  const int row_lo = blockIdx.y * rows_each, row_hi = min(rec.rows, row_lo + rows_each);
  if (rec.pieces == 0 || row_lo >= row_hi) return;
  const int n = rec.pieces;
  int G = 1;
  while (G < kParts && 2 * G < n) G *= 2;
  const int step = kParts / G, g = part % G;
  for (int base = row_lo; base < row_hi; base += step) {
    const int row = base + part / G;
    float top = -INFINITY, sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < row_hi) {
      for (int i0 = g; i0 < n; i0 += 4 * G) {
        float m[4], l[4];
        float4 y[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = i0 + x * G;
          m[x] = -INFINITY, l[x] = 0.f, y[x] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < n) {
            const int s = i == 0 ? rec.slot : 2 * (c + i);
            m[x] = scratch.m[s * ROWS + row];
            l[x] = scratch.l[s * ROWS + row];
            y[x] = scratch.o[(static_cast<int64_t>(s) * ROWS + row) * kCols + col];
          }
        }
        const float high = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
        const float base = base_of(high), f = attn_sm100::ex2(top - base);
        top = high;
        sum *= f, a.x *= f, a.y *= f, a.z *= f, a.w *= f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float w = attn_sm100::ex2(m[x] - base);
          sum += w * l[x];
          a.x += w * y[x].x, a.y += w * y[x].y, a.z += w * y[x].z, a.w += w * y[x].w;
        }
      }
    }
    if (G > 1) {
      part_o[tid] = a, part_m[tid] = top, part_l[tid] = sum;
      __syncthreads();
      if (g == 0) {
        for (int i = 1; i < G; ++i) {
          const int o = tid + i * kCols;
          const float m = part_m[o], high = fmaxf(m, top), base = base_of(high);
          const float f = attn_sm100::ex2(top - base), w = attn_sm100::ex2(m - base);
          const float4 y = part_o[o];
          top = high;
          sum = sum * f + w * part_l[o];
          a.x = a.x * f + w * y.x, a.y = a.y * f + w * y.y, a.z = a.z * f + w * y.z, a.w = a.w * f + w * y.w;
        }
      }
      __syncthreads();
    }
    if (g == 0 && row < row_hi) {
      const int at = rec.row + row;
      const float inv = over(p, sum, rec.held, rec.first, rec.count, at / p.group);
      const int token = rec.first + at / p.group, head = rec.h * p.group + at % p.group;
      *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.o_st + head * p.o_sh + 4 * col) =
          make_uint2(pack2<F16>(a.x * inv, a.y * inv), pack2<F16>(a.z * inv, a.w * inv));
      if (col == 0 && p.lse)
        p.lse[static_cast<int64_t>(token) * p.Hq + head] = sum == 0.f ? -INFINITY : (top - shift + log2f(sum)) * kLn2;
    }
  }
}

}  // namespace attn_tree
