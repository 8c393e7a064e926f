// rotary.cuh — rotary positions with several axes (attn_rotary).
//
// Pair i of a head turns by angle_i = pos[axis(i)] * freq_i.  The angle is
// formed in 64 bits and reduced to a fraction of a turn before cos and sin are
// taken in 32: a position of 2^20 times a frequency of order 1 has lost 2^-4
// of a radian in 32 bits.  Every head of a token shares the angles, so a block
// forms them once in shared memory; the rest is one read and one write of Q
// and K, which bounds the kernel: 16384 tokens of 32 + 32 heads of 128 in bf16,
// there and back, 192 us, 5.6 TB/s (memory alone would be 164).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "../../include/attn_rt.h"
#include "sm100_ptx.cuh"

namespace rotary {

constexpr int kThreads = 256;

struct Params {
  int64_t tokens, N;  // B * N, N
  int Hq, H, D, half;  // H = Hq + Hk
  int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn;
  int64_t qo_sb, qo_sh, qo_sn, ko_sb, ko_sh, ko_sn;
  int64_t p_sa, p_sb, p_sn;
  const void* q;
  const void* k;
  void* qo;
  void* ko;
  const void* positions;
  const double* freqs;
  const int32_t* axes;
  int32_t* status;
  int num_axes, positions_64;
  float sign;
  int tile;  // tokens per block
  int lanes_shift, heads_shift;  // threads of a head, heads taken at once, log2
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// V values moved at once, as 32-bit words: 16 bytes, or one value where rows
// are not aligned.
template <typename T, int V>
struct Pack {
  uint4 w;

  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ void open(float (&v)[V]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) {
        v[i] = __uint_as_float(x[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(x[i] << 16), v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void close(const float (&v)[V]) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) x[i] = __float_as_uint(v[i]);
      else if constexpr (std::is_same<T, __half>::value) x[i] = attn_sm100::pack_f16(v[2 * i], v[2 * i + 1]);
      else x[i] = attn_sm100::pack_bf16(v[2 * i], v[2 * i + 1]);
    }
    w = make_uint4(x[0], x[1], x[2], x[3]);
  }
};

template <typename T>
struct Pack<T, 1> {
  T w;

  __device__ __forceinline__ void load(const T* p) { w = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
  __device__ __forceinline__ void open(float (&v)[1]) const { v[0] = to_f(w); }
  __device__ __forceinline__ void close(const float (&v)[1]) { w = from_f<T>(v[0]); }
};

// The V / 2 neighbouring pairs of a pack.
template <typename T, int V>
__device__ __forceinline__ void turn_pairs(Pack<T, V>& a, const float2* w) {
  float v[V];
  a.open(v);
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const float x0 = v[e], x1 = v[e + 1];
    v[e] = x0 * w[e / 2].x - x1 * w[e / 2].y;
    v[e + 1] = x0 * w[e / 2].y + x1 * w[e / 2].x;
  }
  a.close(v);
}

// V pairs, their first values in one pack and their second ones in another.
template <typename T, int V>
__device__ __forceinline__ void turn_packs(Pack<T, V>& a, Pack<T, V>& c, const float2* w) {
  float x[V], y[V];
  a.open(x);
  c.open(y);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float x0 = x[e], x1 = y[e];
    x[e] = x0 * w[e].x - x1 * w[e].y;
    y[e] = x0 * w[e].y + x1 * w[e].x;
  }
  a.close(x);
  c.close(y);
}

// A thread keeps its place in a head (two packs: one of the first halves with
// its partner, or, neighbours, two packs of whole pairs, or two packs of the
// values behind the turned ones; V = 1: a pair, or one value behind them) and
// goes through heads and tokens, so that its cosines and sines stay in
// registers for all heads of a token.
template <typename T, int V, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Params p) {
  extern __shared__ float2 turn[];  // [tile][half]: (cos, sin)
  using P = Pack<T, V>;
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(p.tile);
  const int n_tok = static_cast<int>(min(static_cast<int64_t>(p.tile), p.tokens - t0));
  for (int x = threadIdx.x; x < n_tok * p.half; x += kThreads) {
    const int tok = x / p.half, i = x - tok * p.half;
    const int64_t t = t0 + tok, b = t < p.N ? 0 : t / p.N, n = t - b * p.N;
    int axis = p.axes ? __ldg(p.axes + i) : 0;
    if (axis < 0 || axis >= p.num_axes) {
      atomicCAS(p.status, 0, ATTN_ERR_INVALID);
      axis = 0;
    }
    const int64_t off = axis * p.p_sa + b * p.p_sb + n * p.p_sn;
    const double pos = p.positions_64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[off])
                                      : static_cast<double>(static_cast<const int32_t*>(p.positions)[off]);
    const double turns = pos * __ldg(p.freqs + i) * 0.15915494309189533577;  // 1 / (2 pi)
    const float part = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.f * part, &s, &c);
    turn[x] = make_float2(c, p.sign * s);
  }
  __syncthreads();
  const int turned = 2 * p.half / V, copied = (p.D - 2 * p.half) / V;  // packs
  const int rot = V == 1 ? p.half : (turned + 1) / 2, tail = V == 1 ? copied : (copied + 1) / 2;
  // lanes: threads of a head (a power of two); heads and tokens taken at once.
  const int lanes = 1 << p.lanes_shift, rows = kThreads >> p.lanes_shift;
  const int heads = min(rows, 1 << p.heads_shift), tokens = rows >> min(p.heads_shift, 31 - __clz(rows));
  const int slot = threadIdx.x >> p.lanes_shift;
  const int h0 = slot & (heads - 1), tok0 = slot / heads;
  for (int u = threadIdx.x & (lanes - 1); u < rot + tail; u += lanes) {
    const bool copy = u >= rot;
    int i0, i1;
    bool two = true;
    if (V == 1) {
      i0 = copy ? p.half + u : NEIGHBOURS ? 2 * u : u;
      i1 = NEIGHBOURS ? 2 * u + 1 : u + p.half;
      two = !copy;
    } else if (copy) {
      i0 = 2 * p.half + 2 * (u - rot) * V, i1 = i0 + V;
      two = 2 * (u - rot) + 1 < copied;
    } else {
      i0 = NEIGHBOURS ? 2 * u * V : u * V;
      i1 = NEIGHBOURS ? i0 + V : p.half + i0;
      two = !NEIGHBOURS || 2 * u + 1 < turned;
    }
    for (int tok = tok0; tok < n_tok; tok += tokens) {
      const int64_t t = t0 + tok, b = t < p.N ? 0 : t / p.N, n = t - b * p.N;
      const T* const q = static_cast<const T*>(p.q) + b * p.q_sb + n * p.q_sn;
      const T* const k = static_cast<const T*>(p.k) + b * p.k_sb + n * p.k_sn - p.Hq * p.k_sh;
      T* const qo = static_cast<T*>(p.qo) + b * p.qo_sb + n * p.qo_sn;
      T* const ko = static_cast<T*>(p.ko) + b * p.ko_sb + n * p.ko_sn - p.Hq * p.ko_sh;
      float2 w[V];  // of the pairs of the first pack and its partner, or of both packs
      if (!copy) {
        const float2* const cs = turn + tok * p.half;
#pragma unroll
        for (int e = 0; e < V; ++e)
          w[e] = cs[V == 1 ? u : !NEIGHBOURS ? i0 + e : (e < V / 2 || two) ? i0 / 2 + e : 0];
      }
      // kHeads heads' loads before the first store: an output may be its input,
      // so the compiler keeps later loads behind earlier stores.
      constexpr int kHeads = V == 1 ? 1 : 2;
      for (int g = h0; g < p.H; g += kHeads * heads) {
        P a[kHeads], c[kHeads];
#pragma unroll
        for (int x = 0; x < kHeads; ++x) {
          const int h = g + x * heads;
          if (h < p.H) {
            const T* const src = h >= p.Hq ? k + h * p.k_sh : q + h * p.q_sh;
            a[x].load(src + i0);
            if (two) c[x].load(src + i1);
          }
        }
#pragma unroll
        for (int x = 0; x < kHeads; ++x) {
          const int h = g + x * heads;
          if (h >= p.H) break;
          if (!copy) {
            if constexpr (NEIGHBOURS && V > 1) {
              turn_pairs<T, V>(a[x], w);
              if (two) turn_pairs<T, V>(c[x], w + V / 2);
            } else {
              turn_packs<T, V>(a[x], c[x], w);
            }
          }
          T* const dst = h >= p.Hq ? ko + h * p.ko_sh : qo + h * p.qo_sh;
          a[x].store(dst + i0);
          if (two) c[x].store(dst + i1);
        }
      }
    }
  }
}

}  // namespace rotary
