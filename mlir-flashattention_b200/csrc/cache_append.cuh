// cache_append.cuh — keys and values of new tokens into the pages of the cache
// (attn_cache_append), with the e4m3 quantisation of an 8-bit cache.
//
// A copy: bound by memory (each value read once and written once).  A thread
// moves 16 keys' and 16 values' numbers of one row, four 16-byte loads in flight
// and stores of 16 bytes, e4m3 rows too.  64 tokens 1.9 us; 16384 tokens into an
// e4m3 cache 25 us against 14 for the bytes: the exact division is the rest
// (the product with the reciprocal alone 18 us, but not the formula's bits; a
// product that is corrected by its remainder is untried).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "../../include/attn_rt.h"

namespace cache_append {

constexpr int kThreads = 256;

struct Params {
  int64_t N, T, slots_in_cache;
  int Hkv, chunks;  // 16-value chunks per row
  int page_shift;
  int tile;  // rows per block
  int64_t k_st, k_sh, v_st, v_sh;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  const void* k;
  const void* v;
  void* kc;
  void* vc;
  const int64_t* slots;
  const int32_t* rows;
  const float* k_descale_heads;
  const float* v_descale_heads;
  float k_descale, v_descale;
  int32_t* status;
};

template <bool F16>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if constexpr (F16) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}

// Two values over the descale, saturated to +-448, round to nearest even; the
// division is the exact one, so that a value and its stored form agree with
// the formula to the last bit.
__device__ __forceinline__ uint32_t quantise(float2 x, float descale) {
  return __nv_cvt_float2_to_fp8x2(
      make_float2(__fdiv_rn(x.x, descale), __fdiv_rn(x.y, descale)), __NV_SATFINITE, __NV_E4M3);
}

// 16 values, as the cache holds them, to their place.
template <bool F16, bool FP8>
__device__ __forceinline__ void put(void* cache, int64_t at, int c, uint4 a, uint4 b, float d) {
  if constexpr (FP8) {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      r[k] = quantise(widen<F16>(w[2 * k]), d) | (quantise(widen<F16>(w[2 * k + 1]), d) << 16);
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(cache) + at + 16 * c) = make_uint4(r[0], r[1], r[2], r[3]);
  } else {
    uint4* const dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) + 2 * c;
    dst[0] = a;
    dst[1] = b;
  }
}

template <bool F16, bool FP8>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Params p) {
  const int per_row = p.Hkv * p.chunks;
  const int64_t i0 = blockIdx.x * static_cast<int64_t>(p.tile);
  const int units = static_cast<int>(min(static_cast<int64_t>(p.tile), p.N - i0)) * per_row;
#pragma unroll 2
  for (int u = threadIdx.x; u < units; u += kThreads) {
    const int k = u / per_row, rest = u - k * per_row;
    const int64_t slot = __ldg(p.slots + i0 + k);
    const int64_t row = p.rows ? __ldg(p.rows + i0 + k) : i0 + k;
    if (slot == -1) continue;
    if (slot < 0 || slot >= p.slots_in_cache || row < 0 || row >= p.T) {
      if (rest == 0) atomicCAS(p.status, 0, ATTN_ERR_INVALID);
      continue;
    }
    const int h = rest / p.chunks, c = rest - h * p.chunks;
    const int64_t page = slot >> p.page_shift, at = slot & ((int64_t{1} << p.page_shift) - 1);
    const uint4* const ks =
        reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + row * p.k_st + h * p.k_sh) + 2 * c;
    const uint4* const vs =
        reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + row * p.v_st + h * p.v_sh) + 2 * c;
    const uint4 a = __ldg(ks), b = __ldg(ks + 1), e = __ldg(vs), f = __ldg(vs + 1);
    float kd = p.k_descale, vd = p.v_descale;
    if (FP8 && p.k_descale_heads) kd *= __ldg(p.k_descale_heads + h);
    if (FP8 && p.v_descale_heads) vd *= __ldg(p.v_descale_heads + h);
    put<F16, FP8>(p.kc, page * p.kc_sp + h * p.kc_sh + at * p.kc_st, c, a, b, kd);
    put<F16, FP8>(p.vc, page * p.vc_sp + h * p.vc_sh + at * p.vc_st, c, e, f, vd);
  }
}

}  // namespace cache_append
