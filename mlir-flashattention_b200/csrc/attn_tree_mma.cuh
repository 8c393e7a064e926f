// attn_tree_mma.cuh — attn_tree_fwd for few query rows per kv-head (decode,
// small drafts), and the join of items cut between blocks.
//
// With 16 query rows a cached key of D values costs 4 * 16 * D operations for
// 4 * D bytes: 16 a byte against the 250 a byte that this GPU can do per byte
// it reads, so the kernel is bound by the cache's bytes and everything here
// serves to keep loads in flight: a block is one warp that issues TMA loads of
// page segments into a ring of tiles (64 keys of K and of V each, 128-byte
// swizzle) and four warps that each take 16 of a tile's keys, with their own
// running maximum, sum and accumulators, and meet only when a piece ends.  Two
// blocks share an SM.  Tensor cores by mma.sync m16n8k16: operands go from
// shared memory to registers, so 16 rows cost 16 rows (a 128-row accumulator
// in tensor memory would be 1/8 used and its softmax one warp's work).
//
// An e4m3 cache is met in f16: e4m3 values are f16 values, and a bf16 row of q
// scaled by the power of two that brings its largest value to 2^14..2^15 is
// exact in f16 down to 2^-39 of that value.  New keys and values are 16-bit
// and met in their own type.
//
// Weights are rounded to the operands' type for P V.  In bf16 a rounding by
// 2^-9 would double the error of the result, whose own rounding is the same
// size: P goes in as two bf16 parts, p and p - bf16(p), for twice the small
// product's work.
#pragma once

#include <type_traits>

#include "attn_tree.cuh"
#include "sm100_ptx.cuh"

namespace attn_tree {

constexpr int kMmaRows = 16, kMmaKeys = 64, kMmaWarps = 4;
constexpr int kMmaThreads = 32 * (kMmaWarps + 1);

template <typename T, typename TC, int D>
struct MmaCfg {
  static constexpr bool FP8 = sizeof(TC) == 1;
  static constexpr int kRowBytes = D * static_cast<int>(sizeof(TC));
  static constexpr int kNewRowBytes = D * 2;
  // One operand's part of a stage: 64 cached keys, or as many new ones as fit.
  static constexpr int kTile = kMmaKeys * kRowBytes;
  static constexpr int kStages = 98304 / (2 * kTile);
  static constexpr int kNewKeys = kTile / kNewRowBytes;  // most new keys of a stage
  static constexpr int kJoin = kMmaWarps * kMmaRows * 32 * 4;  // 32 columns of each warp
  // Weights are kept times 2^kShift: in f16 they stay normal down to 2^-22.
  static constexpr float kShift = (FP8 || std::is_same<T, __half>::value) ? 8.f : 0.f;
  static constexpr size_t kSmem = 1024 + kStages * 2 * kTile + kMmaRows * D * 2 + kJoin;
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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
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

// The four reading warps meet.
__device__ __forceinline__ void readers_sync() {
  __syncwarp();
  asm volatile("barrier.sync 1, 128;" ::: "memory");
}

template <typename T, typename TC, int D>
__global__ void __launch_bounds__(kMmaThreads, 2)
    tree_mma_kernel(const __grid_constant__ CUtensorMap map_kc, const __grid_constant__ CUtensorMap map_vc,
                    const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_vn,
                    const __grid_constant__ Params p, const Split split, const Scratch scratch,
                    const int min_units) {
  using C = MmaCfg<T, TC, D>;
  constexpr bool F16 = std::is_same<T, __half>::value;
  constexpr bool FP8 = C::FP8;
  constexpr int kSteps = D / 16;              // k-steps of Q K
  constexpr int kTilesD = D / 8;              // n-tiles of P V
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages];
  __shared__ volatile int abort_flag;
  __shared__ float warp_m[kMmaWarps][kMmaRows], warp_l[kMmaWarps][kMmaRows];
  __shared__ float q_unit[kMmaRows];  // e4m3: the power of two that a row of q was divided by

  uint8_t* smem = raw + ((1024u - (attn_sm100::smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t s_ring = attn_sm100::smem_u32(smem);
  T* const s_q = reinterpret_cast<T*>(smem + C::kStages * 2 * C::kTile);  // [16][D], chunks swizzled
  float* const s_join = reinterpret_cast<float*>(smem + C::kStages * 2 * C::kTile + kMmaRows * D * 2);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      attn_sm100::mbar_init(&full[s], 1);
      attn_sm100::mbar_init(&empty[s], kMmaWarps);
    }
    abort_flag = 0;
    attn_sm100::fence_mbar_init();
    attn_sm100::fence_proxy_async_smem();
  }
  grid_wait();
  grid_release();
  if (tid == 0) scratch.record[blockIdx.x].pieces = 0;
  Share share = find_share(p, split, min_units);  // synchronises the block
  __syncthreads();
  const int64_t share_lo = share.lo;
  Piece pc;

  if (warp == kMmaWarps) {
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      attn_sm100::prefetch_tmap(&map_kc);
      attn_sm100::prefetch_tmap(&map_vc);
      attn_sm100::prefetch_tmap(&map_kn);
      attn_sm100::prefetch_tmap(&map_vn);
    }
    const int seg_shift = min(p.page_shift, split.keys_shift);  // rows of a page segment, log2
    const int seg_bytes = C::kRowBytes << seg_shift;
    int64_t n = 0;  // stages filled
    bool ok = true;
    while (ok && next_piece(p, split, share, pc)) {
      const int32_t* const row = p.table + pc.b * p.table_stride;
      for (int k = pc.k0; k < pc.k1 && ok; ++k, ++n) {
        const int s = static_cast<int>(n % C::kStages);
        const uint32_t u = static_cast<uint32_t>(n / C::kStages);
        const bool cached = k < pc.cached;
        const int first = cached ? k << split.keys_shift : (k - pc.cached) << split.new_shift;
        // Page ids before the wait: the loads overlap it.
        int segs = 1, page = 0, at = 0;
        if (cached) {
          segs = (min(1 << split.keys_shift, pc.r.held - first) + (1 << seg_shift) - 1) >> seg_shift;
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

  // ------------------------------------------------------------- four readers
  const int quad = lane & 3, grp = lane >> 2;
  int64_t n = 0;
  bool ok = true;
  while (next_piece(p, split, share, pc)) {
    const int rows = static_cast<int>(
        min(static_cast<int64_t>(kMmaRows), static_cast<int64_t>(pc.r.count) * p.group - pc.rt * kMmaRows));
    auto row_of = [&](int r, int& token, int& head) {
      const int at = pc.rt * kMmaRows + r;
      token = pc.r.first + at / p.group;
      head = pc.h * p.group + at % p.group;
    };
    // q rows to shared memory (rows behind the last: zeros), 8 threads a row.
    {
      const int r = tid >> 3;
      int token, head;
      row_of(r, token, head);
      uint4 v[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int chunk = (tid & 7) + 8 * c;
        v[c] = make_uint4(0, 0, 0, 0);
        if (r < rows)
          v[c] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + token * p.q_st + head * p.q_sh) + chunk);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(s_q) + r * D * 2 + ((chunk ^ (r & 7)) * 16)) = v[c];
      }
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
    readers_sync();
    // A fragments of q.  For an e4m3 cache the order of d is the one in which
    // a thread finds 16 of a key's values in one load (see below).
    uint32_t qa[kSteps][4];
    const uint32_t s_q32 = attn_sm100::smem_u32(s_q);
    auto q_frag = [&](uint32_t (&a)[4], int s) {  // 16-bit keys: plain order
      const int r = (lane & 7) + 8 * ((lane >> 3) & 1), chunk = 2 * s + (lane >> 4);
      ldmatrix4(a, s_q32 + r * D * 2 + ((chunk ^ (r & 7)) * 16));
    };
    float unit[2] = {1.f, 1.f};
    if constexpr (FP8) {
      float inv[2] = {1.f, 1.f};
      if constexpr (!F16) {
        unit[0] = q_unit[grp], unit[1] = q_unit[grp + 8];
        inv[0] = 1.f / unit[0], inv[1] = 1.f / unit[1];
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = (s >> 2) * 64 + quad * 16 + (s & 3) * 4;  // 4 values from here
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = grp + 8 * x;
          const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(s_q) + r * D * 2 +
                                                          (((d >> 3) ^ (r & 7)) * 16) + (d & 7) * 2);
          if constexpr (F16) {
            qa[s][x] = w.x, qa[s][2 + x] = w.y;
          } else {
            auto half2 = [&](uint32_t b) {
              return attn_sm100::pack_f16(__uint_as_float(b << 16) * inv[x], __uint_as_float(b & 0xffff0000u) * inv[x]);
            };
            qa[s][x] = half2(w.x), qa[s][2 + x] = half2(w.y);
          }
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q_frag(qa[s], s);
    }
    float kd = 1.f, vd = 1.f;
    if constexpr (FP8) {
      kd = p.k_descale * (p.k_descale_heads ? __ldg(p.k_descale_heads + pc.h) : 1.f);
      vd = p.v_descale * (p.v_descale_heads ? __ldg(p.v_descale_heads + pc.h) : 1.f);
    }
    const float scale2 = p.scale * kLog2e;
    float o[kTilesD][4];
#pragma unroll
    for (int t = 0; t < kTilesD; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // Scores (rows grp, grp + 8; keys 2 quad + {0, 1} of two groups of 8) to
    // weights; updates m, l and rescales o where a maximum moved.
    auto softmax = [&](float (&s)[2][4]) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m[x]);
        if (__any_sync(0xffffffffu, top != m[x])) {
          const float a = top == -INFINITY ? 1.f : attn_sm100::ex2(m[x] - top);
          l[x] *= a;
#pragma unroll
          for (int t = 0; t < kTilesD; ++t) o[t][2 * x] *= a, o[t][2 * x + 1] *= a;
          m[x] = top;
        }
        const float sub = (top == -INFINITY ? 0.f : top) - C::kShift;
        float add = 0.f;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[g][2 * x + e] = attn_sm100::ex2(s[g][2 * x + e] - sub);
            add += s[g][2 * x + e];
          }
        l[x] += add;
      }
    };
    bool scaled = !FP8;  // o is in units of the cached values until the new ones come

    for (int k = pc.k0; k < pc.k1; ++k, ++n) {
      const int st = static_cast<int>(n % C::kStages);
      const uint32_t u = static_cast<uint32_t>(n / C::kStages);
      if (ok) ok = __all_sync(0xffffffffu, attn_sm100::mbar_wait_bounded(&full[st], u & 1u, &abort_flag, p.status, kWaitLimitNs));
      const uint32_t ks = s_ring + st * 2 * C::kTile, vs = ks + C::kTile;
      const bool cached = k < pc.cached;
      const int first = cached ? k << split.keys_shift : (k - pc.cached) << split.new_shift;
      const int here = cached ? min(1 << split.keys_shift, pc.r.held - first)
                              : min(1 << split.new_shift, pc.r.count - first);
      const int kb = warp * 16;  // this warp's keys of the tile
      if (kb < here && ok) {
        const int seg_shift = cached ? min(p.page_shift, split.keys_shift) : split.new_shift;
        const int seg = kb >> seg_shift, r0 = kb & ((1 << seg_shift) - 1);
        float s[2][4] = {};
        if (FP8 && cached) {
          // Key r (row of 128 bytes): thread quad loads 16 values at 16 quad and
          // 16 at 64 + 16 quad; k-step s takes 4 of them, for k = 2 quad + {0, 1}
          // and 2 quad + 8 + {0, 1}: q_frag's order.
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int r = r0 + 8 * g + grp;
            const uint32_t base = ks + seg * (C::kRowBytes << seg_shift) + r * 128;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint4 w = lds128(base + (((quad + 4 * c) ^ (r & 7)) * 16));
              const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                mma16816<true>(s[g], qa[4 * c + e], f16_of_e4m3(ww[e]), f16_of_e4m3(ww[e] >> 16));
            }
          }
        } else {
          const uint32_t base = ks + seg * (C::kNewRowBytes << seg_shift);
          const int r = r0 + (lane & 7) + 8 * (lane >> 4);
#pragma unroll
          for (int x = 0; x < kSteps; ++x) {
            const int chunk = 2 * x + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix4(b, base + (chunk >> 3) * (128 << seg_shift) + r * 128 + (((chunk & 7) ^ (r & 7)) * 16));
            if constexpr (FP8) {
              uint32_t a[4];
              q_frag(a, x);
              mma16816<F16>(s[0], a, b[0], b[1]);
              mma16816<F16>(s[1], a, b[2], b[3]);
            } else {
              mma16816<F16>(s[0], qa[x], b[0], b[1]);
              mma16816<F16>(s[1], qa[x], b[2], b[3]);
            }
          }
        }
        // Scale, then the mask (selected after the scale: what a masked key's
        // score was does not matter).
        const float f0 = FP8 && cached ? scale2 * kd * unit[0] : scale2;
        const float f1 = FP8 && cached ? scale2 * kd * unit[1] : scale2;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          s[g][0] *= f0, s[g][1] *= f0, s[g][2] *= f1, s[g][3] *= f1;
        }
        if (cached) {
          if (kb + 16 > here) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (kb + 8 * g + 2 * quad + (e & 1) >= here) s[g][e] = -INFINITY;
          }
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int i = (pc.rt * kMmaRows + grp + 8 * x) / p.group;  // token of the request
            const bool live = grp + 8 * x < rows;
            const uint8_t* mrow = p.mask + static_cast<int64_t>(pc.r.first + (live ? i : 0)) * p.mask_stride;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = kb + 8 * g + 2 * quad + e;
                bool hide = j >= here || !live;
                if (!hide) hide = p.mask ? mrow[first + j] != 0 : first + j > i;
                if (hide) s[g][2 * x + e] = -INFINITY;
              }
          }
        }
        softmax(s);
        // Weights of keys that are not there are 0; their values are made 0 too
        // (0 times what lies in memory there need not be 0).
        const bool tail = kb + 16 > here;
        uint32_t live0 = 0xffffffffu, live1 = 0xffffffffu;
        if (tail) {
          const int j = kb + 2 * quad;
          live0 = (j < here ? 0xffffu : 0u) | (j + 1 < here ? 0xffff0000u : 0u);
          live1 = (j + 8 < here ? 0xffffu : 0u) | (j + 9 < here ? 0xffff0000u : 0u);
        }
        if (!cached && !scaled) {
#pragma unroll
          for (int t = 0; t < kTilesD; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][e] *= vd;
          scaled = true;
        }
        if constexpr (FP8) {
          // Values: thread group grp loads 16 of each of its four keys (2 quad,
          // + 1, + 8, + 9) at 16 grp; n-tile t is d = 16 n + t, n = 0..7.
          if (cached) {
            uint32_t a[4] = {pack2<true>(s[0][0], s[0][1]), pack2<true>(s[0][2], s[0][3]),
                             pack2<true>(s[1][0], s[1][1]), pack2<true>(s[1][2], s[1][3])};
            uint32_t w[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int r = r0 + 2 * quad + (y & 1) + 8 * (y >> 1);
              const uint4 v = lds128(vs + seg * (C::kRowBytes << seg_shift) + r * 128 + ((grp ^ (r & 7)) * 16));
              w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const uint32_t lo = __byte_perm(w[0][c], w[1][c], z ? 0x7362 : 0x5140);
                const uint32_t hi = __byte_perm(w[2][c], w[3][c], z ? 0x7362 : 0x5140);
                mma16816<true>(o[4 * c + 2 * z], a, f16_of_e4m3(lo) & live0, f16_of_e4m3(hi) & live1);
                mma16816<true>(o[4 * c + 2 * z + 1], a, f16_of_e4m3(lo >> 16) & live0, f16_of_e4m3(hi >> 16) & live1);
              }
            }
          } else {
            uint32_t a[4] = {pack2<F16>(s[0][0], s[0][1]), pack2<F16>(s[0][2], s[0][3]),
                             pack2<F16>(s[1][0], s[1][1]), pack2<F16>(s[1][2], s[1][3])};
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // 8 of the 16 values at a time
              uint32_t w[4][4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int r = r0 + 2 * quad + (y & 1) + 8 * (y >> 1), chunk = 2 * grp + c;
                const uint4 v = lds128(vs + (chunk >> 3) * (128 << seg_shift) + r * 128 + (((chunk & 7) ^ (r & 7)) * 16));
                w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
                mma16816<F16>(o[8 * c + e], a, __byte_perm(w[0][e >> 1], w[1][e >> 1], sel) & live0,
                              __byte_perm(w[2][e >> 1], w[3][e >> 1], sel) & live1);
              }
            }
          }
        } else {
          uint32_t a[4], rest[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float x0 = s[y >> 1][2 * (y & 1)], x1 = s[y >> 1][2 * (y & 1) + 1];
            a[y] = pack2<F16>(x0, x1);
            if constexpr (!F16)
              rest[y] = pack2<false>(x0 - __uint_as_float(a[y] << 16), x1 - __uint_as_float(a[y] & 0xffff0000u));
          }
          const uint32_t base = vs + seg * (C::kNewRowBytes << seg_shift);
          const int r = r0 + (lane & 7) + 8 * ((lane >> 3) & 1);
#pragma unroll
          for (int t = 0; t < kTilesD / 2; ++t) {
            const int chunk = 2 * t + (lane >> 4);
            uint32_t b[4];
            ldmatrix4t(b, base + (chunk >> 3) * (128 << seg_shift) + r * 128 + (((chunk & 7) ^ (r & 7)) * 16));
            if (tail) b[0] &= live0, b[1] &= live1, b[2] &= live0, b[3] &= live1;
            mma16816<F16>(o[2 * t], a, b[0], b[1]);
            mma16816<F16>(o[2 * t + 1], a, b[2], b[3]);
            if constexpr (!F16) {
              mma16816<F16>(o[2 * t], rest, b[0], b[1]);
              mma16816<F16>(o[2 * t + 1], rest, b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) attn_sm100::mbar_arrive(&empty[st]);
    }

    // ---------------------------------------------------------- a piece ends
    if (!scaled) {
#pragma unroll
      for (int t = 0; t < kTilesD; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] *= vd;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (quad == 0) warp_m[warp][grp + 8 * x] = m[x], warp_l[warp][grp + 8 * x] = l[x];
    }
    readers_sync();
    float factor[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) top = fmaxf(top, warp_m[w][grp + 8 * x]);
      factor[x] = top == -INFINITY ? 0.f : attn_sm100::ex2(m[x] - top);
    }
    // The row that this thread writes: tid / 8, columns 4 (tid % 8) of 32.
    const int wr = tid >> 3, wc = (tid & 7) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; ++w) top = fmaxf(top, warp_m[w][wr]);
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) sum += attn_sm100::ex2(warp_m[w][wr] - top) * warp_l[w][wr];
    }
    const bool whole = pc.k0 == 0 && pc.k1 == pc.tiles;
    const int slot = 2 * blockIdx.x + (share.lo - (pc.k1 - pc.k0) == share_lo ? 0 : 1);
    int token, head;
    row_of(wr, token, head);
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += 32) {
      // The accumulators of columns c0 .. c0 + 31 (an e4m3 cache: n-tile t is
      // columns 16 n + t, so they are one thread of each quad's).
      if constexpr (FP8) {
        if (quad == c0 / 32) {
#pragma unroll
          for (int t = 0; t < kTilesD; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s_join[(warp * kMmaRows + grp + 8 * (e >> 1)) * 32 + 16 * (e & 1) + t] = o[t][e] * factor[e >> 1];
        }
        __syncwarp();
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            *reinterpret_cast<float2*>(s_join + (warp * kMmaRows + grp + 8 * x) * 32 + 8 * t + 2 * quad) =
                make_float2(o[c0 / 8 + t][2 * x] * factor[x], o[c0 / 8 + t][2 * x + 1] * factor[x]);
      }
      readers_sync();
      if (wr < rows) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_join + (w * kMmaRows + wr) * 32 + wc);
          x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          uint2 w = make_uint2(pack2<F16>(x.x * inv, x.y * inv), pack2<F16>(x.z * inv, x.w * inv));
          *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.o_st + head * p.o_sh + c0 + wc) = w;
        } else {
          scratch.o[(static_cast<int64_t>(slot) * kMmaRows + wr) * (D / 4) + (c0 + wc) / 4] = x;
        }
      }
      readers_sync();
    }
    if ((tid & 7) == 0 && wr < rows) {
      if (whole) {
        if (p.lse)
          p.lse[static_cast<int64_t>(token) * p.Hq + head] =
              sum == 0.f ? -INFINITY : (top - C::kShift + log2f(sum)) * kLn2;
      } else {
        scratch.m[slot * kMmaRows + wr] = top;
        scratch.l[slot * kMmaRows + wr] = sum;
      }
    }
    if (!whole && pc.k0 == 0 && tid == 0) scratch.record[blockIdx.x] = make_record(p, split, share, pc, slot);
  }
}

// Joins the pieces of the items that were cut: block (c, y) takes `rows_each`
// query rows of the cut item that begins in block c of the first kernel, if
// any.  What bounds it is latency, a record and then everything else at once:
// a thread has four columns of a row and every G-th piece of the item, brought
// to one maximum as it goes; the G parts meet in shared memory.  The order of
// the sums depends on the lengths alone, so a call gives the same bits every
// time.
constexpr int kJoinThreads = 256;

template <typename T, int D>
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
            m[x] = scratch.m[s * kMmaRows + row];
            l[x] = scratch.l[s * kMmaRows + row];
            y[x] = scratch.o[(static_cast<int64_t>(s) * kMmaRows + row) * kCols + col];
          }
        }
        const float high = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
        if (high != -INFINITY) {
          const float f = attn_sm100::ex2(top - high);
          top = high;
          sum *= f, a.x *= f, a.y *= f, a.z *= f, a.w *= f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float w = attn_sm100::ex2(m[x] - high);
            sum += w * l[x];
            a.x += w * y[x].x, a.y += w * y[x].y, a.z += w * y[x].z, a.w += w * y[x].w;
          }
        }
      }
    }
    if (G > 1) {
      part_o[tid] = a, part_m[tid] = top, part_l[tid] = sum;
      __syncthreads();
      if (g == 0) {
        for (int i = 1; i < G; ++i) {
          const int o = tid + i * kCols;
          const float m = part_m[o], high = fmaxf(m, top);
          if (high == -INFINITY) continue;
          const float f = attn_sm100::ex2(top - high), w = attn_sm100::ex2(m - high);
          const float4 y = part_o[o];
          top = high;
          sum = sum * f + w * part_l[o];
          a.x = a.x * f + w * y.x, a.y = a.y * f + w * y.y, a.z = a.z * f + w * y.z, a.w = a.w * f + w * y.w;
        }
      }
      __syncthreads();
    }
    if (g == 0 && row < row_hi) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int at = rec.row + row;
      const int token = rec.first + at / p.group, head = rec.h * p.group + at % p.group;
      *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.o_st + head * p.o_sh + 4 * col) =
          make_uint2(pack2<F16>(a.x * inv, a.y * inv), pack2<F16>(a.z * inv, a.w * inv));
      if (col == 0 && p.lse)
        p.lse[static_cast<int64_t>(token) * p.Hq + head] = sum == 0.f ? -INFINITY : (top - shift + log2f(sum)) * kLn2;
    }
  }
}

}  // namespace attn_tree
