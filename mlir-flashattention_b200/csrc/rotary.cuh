// rotary.cuh — rotary positions with several axes (attn_rotary).
//
// Pair i of a head turns by angle_i = pos[axis(i)] * freq_i.  The angle is
// formed in 64 bits and reduced to a fraction of a turn before cos and sin are
// taken in 32: a position of 2^20 times a frequency of order 1 has lost 2^-4
// of a radian in 32 bits.  Every head of a token shares the angles, so a block
// forms them once in shared memory; the rest is one read and one write of Q
// and K, which bounds the kernel.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/attn_rt.h"

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
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// V values moved at once: 16 bytes, or one value where rows are not aligned.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Params p) {
  extern __shared__ float2 turn[];  // [tile][half]: (cos, sin)
  using P = Pack<T, V>;
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(p.tile);
  const int n_tok = static_cast<int>(min(static_cast<int64_t>(p.tile), p.tokens - t0));
  for (int x = threadIdx.x; x < n_tok * p.half; x += kThreads) {
    const int tok = x / p.half, i = x - tok * p.half;
    const int64_t t = t0 + tok, b = t / p.N, n = t - b * p.N;
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
  // A unit is one pack of the first halves with its partner (or, neighbours,
  // one pack holding whole pairs), or one pack of the values behind them.
  const int rot = NEIGHBOURS && V > 1 ? 2 * p.half / V : p.half / V;
  const int tail = (p.D - 2 * p.half) / V;
  const int per_head = rot + tail;
  const int units = n_tok * p.H * per_head;
  for (int x = threadIdx.x; x < units; x += kThreads) {
    const int th = x / per_head, u = x - th * per_head;
    const int tok = th / p.H;
    int h = th - tok * p.H;
    const int64_t t = t0 + tok, b = t / p.N, n = t - b * p.N;
    const bool is_k = h >= p.Hq;
    if (is_k) h -= p.Hq;
    const T* src = is_k ? static_cast<const T*>(p.k) + b * p.k_sb + h * p.k_sh + n * p.k_sn
                        : static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh + n * p.q_sn;
    T* dst = is_k ? static_cast<T*>(p.ko) + b * p.ko_sb + h * p.ko_sh + n * p.ko_sn
                  : static_cast<T*>(p.qo) + b * p.qo_sb + h * p.qo_sh + n * p.qo_sn;
    const float2* cs = turn + tok * p.half;
    if (u >= rot) {
      const int at = 2 * p.half + (u - rot) * V;
      *reinterpret_cast<P*>(dst + at) = *reinterpret_cast<const P*>(src + at);
    } else if constexpr (V == 1) {
      const int i0 = NEIGHBOURS ? 2 * u : u, i1 = NEIGHBOURS ? 2 * u + 1 : u + p.half;
      const float2 w = cs[u];
      const float x0 = to_f(src[i0]), x1 = to_f(src[i1]);
      dst[i0] = from_f<T>(x0 * w.x - x1 * w.y);
      dst[i1] = from_f<T>(x0 * w.y + x1 * w.x);
    } else if constexpr (NEIGHBOURS) {
      const int at = u * V;
      P a = *reinterpret_cast<const P*>(src + at);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 w = cs[(at + e) / 2];
        const float x0 = to_f(a.v[e]), x1 = to_f(a.v[e + 1]);
        a.v[e] = from_f<T>(x0 * w.x - x1 * w.y);
        a.v[e + 1] = from_f<T>(x0 * w.y + x1 * w.x);
      }
      *reinterpret_cast<P*>(dst + at) = a;
    } else {
      const int at = u * V;
      P a = *reinterpret_cast<const P*>(src + at);
      P c = *reinterpret_cast<const P*>(src + p.half + at);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 w = cs[at + e];
        const float x0 = to_f(a.v[e]), x1 = to_f(c.v[e]);
        a.v[e] = from_f<T>(x0 * w.x - x1 * w.y);
        c.v[e] = from_f<T>(x0 * w.y + x1 * w.x);
      }
      *reinterpret_cast<P*>(dst + at) = a;
      *reinterpret_cast<P*>(dst + p.half + at) = c;
    }
  }
}

}  // namespace rotary
