// cache_append.cuh — keys and values of new tokens into the pages of the cache
// (attn_cache_append), with the e4m3 quantisation of an 8-bit cache.
//
// A copy: bound by memory (each value read once and written once).  A thread
// moves 16 values, two 16-byte loads and one or two 16-byte stores, so that
// e4m3 rows are stored 16 bytes wide too.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "../../include/attn_rt.h"

namespace cache_append {

struct Params {
  int64_t N, T, slots_in_cache;
  int Hkv, chunks;  // 16-value chunks per row
  int page_shift;
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

template <bool F16, bool FP8>
__global__ void __launch_bounds__(256) append_kernel(const Params p) {
  const int per_row = p.Hkv * p.chunks;
  const int64_t total = p.N * per_row * 2;  // K, then V, of each row
  for (int64_t u = blockIdx.x * int64_t{256} + threadIdx.x; u < total; u += gridDim.x * int64_t{256}) {
    const int64_t i = u / (2 * per_row);
    int rest = static_cast<int>(u - i * 2 * per_row);
    const bool is_v = rest >= per_row;
    if (is_v) rest -= per_row;
    const int h = rest / p.chunks, c = rest - h * p.chunks;
    const int64_t slot = p.slots[i];
    if (slot == -1) continue;
    const int64_t row = p.rows ? p.rows[i] : i;
    if (slot < 0 || slot >= p.slots_in_cache || row < 0 || row >= p.T) {
      if (rest == 0) atomicCAS(p.status, 0, ATTN_ERR_INVALID);
      continue;
    }
    const int64_t page = slot >> p.page_shift, at = slot & ((int64_t{1} << p.page_shift) - 1);
    const int64_t from = is_v ? row * p.v_st + h * p.v_sh : row * p.k_st + h * p.k_sh;
    const int64_t to = is_v ? page * p.vc_sp + h * p.vc_sh + at * p.vc_st
                            : page * p.kc_sp + h * p.kc_sh + at * p.kc_st;
    const uint4* src = reinterpret_cast<const uint4*>(
                           static_cast<const uint16_t*>(is_v ? p.v : p.k) + from) + 2 * c;
    const uint4 a = __ldg(src), b = __ldg(src + 1);
    if constexpr (FP8) {
      const float* heads = is_v ? p.v_descale_heads : p.k_descale_heads;
      const float d = (is_v ? p.v_descale : p.k_descale) * (heads ? __ldg(heads + h) : 1.f);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r[k] = quantise(widen<F16>(w[2 * k]), d) | (quantise(widen<F16>(w[2 * k + 1]), d) << 16);
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(is_v ? p.vc : p.kc) + to + 16 * c) =
          make_uint4(r[0], r[1], r[2], r[3]);
    } else {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v ? p.vc : p.kc) + to) + 2 * c;
      dst[0] = a;
      dst[1] = b;
    }
  }
}

}  // namespace cache_append
