// attn_tree.cuh — attention of new tokens over a paged cache (attn_tree_fwd).
//
// For token t of request b and q-head h (kv-head h / g):
//   O = sum_j softmax(scale * q . k_j) v_j
// over the cached keys j < lengths[b] and the request's new keys that the mask
// leaves visible, by the online recurrence with a running maximum m, sum l and
// accumulator in 32 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "../../include/attn_rt.h"

namespace attn_tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

struct Params {
  int B, T, Hq, Hkv, group;
  int W, num_pages, page_shift;
  int max_new;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  int64_t table_stride, mask_stride;
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
// past the table or rows past q would leave the buffers.
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.held = __ldg(p.lengths + b);
  r.first = __ldg(p.starts + b);
  r.count = __ldg(p.starts + b + 1) - r.first;
  const int most = p.W << p.page_shift;
  if (r.held < 0 || r.held > most || r.count < 0 || r.count > p.max_new || r.first < 0 ||
      r.first > p.T - r.count) {
    atomicCAS(p.status, 0, ATTN_ERR_INVALID);
    r.held = r.first = r.count = 0;
  }
  return r;
}

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__nv_fp8_e4m3 x) { return static_cast<float>(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// One block per (row of q, q-head): 4 warps take keys in turn, a key at a time
// per warp, and are joined at the end.
template <typename T, typename TC, int D>
__global__ void __launch_bounds__(128) tree_kernel(const Params p) {
  constexpr int E = D / 32;
  __shared__ float sh_m[4], sh_l[4], sh_o[4][D];
  const int t = blockIdx.x, h = blockIdx.y, hk = h / p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b = -1;
  Request r{};
  for (int i = 0; i < p.B; ++i) {
    r = request(p, i);
    if (t >= r.first && t < r.first + r.count) {
      b = i;
      break;
    }
  }
  if (b < 0) return;
  const int i = t - r.first;
  float q[E], o[E] = {};
  for (int e = 0; e < E; ++e)
    q[e] = to_f(static_cast<const T*>(p.q)[t * p.q_st + h * p.q_sh + lane + 32 * e]);
  const float kd = p.k_descale * (p.k_descale_heads ? p.k_descale_heads[hk] : 1.f);
  const float vd = p.v_descale * (p.v_descale_heads ? p.v_descale_heads[hk] : 1.f);
  float m = -INFINITY, l = 0.f;
  auto step = [&](const float (&k)[E], const float (&v)[E]) {
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale * kLog2e;
    const float top = fmaxf(m, s);
    if (top == -INFINITY) return;
    const float a = exp2f(m - top), w = exp2f(s - top);
    l = l * a + w;
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * v[e];
    m = top;
  };
  float k[E], v[E];
  for (int j = warp; j < r.held; j += 4) {
    const int page = p.table[b * p.table_stride + (j >> p.page_shift)];
    const int at = j & ((1 << p.page_shift) - 1);
    if (page < 0 || page >= p.num_pages) {
      atomicCAS(p.status, 0, ATTN_ERR_INVALID);
      continue;
    }
    const TC* kp = static_cast<const TC*>(p.k_cache) + page * p.kc_sp + hk * p.kc_sh + at * p.kc_st;
    const TC* vp = static_cast<const TC*>(p.v_cache) + page * p.vc_sp + hk * p.vc_sh + at * p.vc_st;
    for (int e = 0; e < E; ++e) {
      k[e] = to_f(kp[lane + 32 * e]) * kd;
      v[e] = to_f(vp[lane + 32 * e]) * vd;
    }
    step(k, v);
  }
  for (int j = warp; j < r.count; j += 4) {
    if (p.mask ? p.mask[t * p.mask_stride + j] != 0 : j > i) continue;
    const T* kp = static_cast<const T*>(p.k_new) + (r.first + j) * p.k_st + hk * p.k_sh;
    const T* vp = static_cast<const T*>(p.v_new) + (r.first + j) * p.v_st + hk * p.v_sh;
    for (int e = 0; e < E; ++e) {
      k[e] = to_f(kp[lane + 32 * e]);
      v[e] = to_f(vp[lane + 32 * e]);
    }
    step(k, v);
  }
  if (lane == 0) {
    sh_m[warp] = m;
    sh_l[warp] = l;
  }
  for (int e = 0; e < E; ++e) sh_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  const float top = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
  float a[4], sum = 0.f;
  for (int w = 0; w < 4; ++w) {
    a[w] = top == -INFINITY ? 0.f : exp2f(sh_m[w] - top);
    sum += a[w] * sh_l[w];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += a[w] * sh_o[w][d];
    static_cast<T*>(p.o)[t * p.o_st + h * p.o_sh + d] = from_f<T>(sum > 0.f ? x / sum : 0.f);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[static_cast<int64_t>(t) * p.Hq + h] = sum > 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

}  // namespace attn_tree
