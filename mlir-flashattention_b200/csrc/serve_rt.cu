// serve_rt.cu — host side of the serving calls in include/attn_rt.h: checks of
// the descriptors, choice of kernel and launch.  No call waits for the device.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <utility>

#include "attn_tree_mma.cuh"
#include "attn_tree_tc.cuh"
#include "cache_append.cuh"
#include "cache_plan.cuh"
#include "rotary.cuh"
#include "rt_host.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return rt_host::fail_with(code, buf);
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(ATTN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  rt_host::count_launches(1);
  return ATTN_OK;
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int page_shift(int page_size) {
  for (int s = 4; s <= 10; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

int check_flags(int32_t flags) {
  if (flags & ~ATTN_FLAG_DEVICE_POINTERS) return fail(ATTN_ERR_INVALID, "unknown flags 0x%x", flags);
  return ATTN_OK;
}

// Kernels read these with TMA and plain loads: host memory would fault.
template <size_t N>
int check_pointers(int32_t flags, const void* const (&list)[N]) {
  if (flags & ATTN_FLAG_DEVICE_POINTERS) return ATTN_OK;
  for (const void* p : list)
    if (p && !rt_host::on_device(p)) return fail(ATTN_ERR_INVALID, "serving calls take device pointers");
  return ATTN_OK;
}

// A stride matters only along an extent of two or more.
bool stride_ok(int64_t stride, int64_t extent, int64_t multiple) {
  return extent <= 1 || stride % multiple == 0;
}

// Of what a call writes: rows of `row` elements along a stride are apart.
bool apart(int64_t stride, int64_t extent, int64_t row) {
  return extent <= 1 || stride >= row || stride <= -row;
}

int pow2_shift(int64_t n, int lo, int hi) {
  int s = lo;
  while (s < hi && (int64_t{1} << s) < n) ++s;
  return s;
}

constexpr int64_t kInt32 = (int64_t{1} << 31) - 1;

// ------------------------------------------------------------------- plan
int check(const AttnCachePlan& d) {
  int rc = check_flags(d.flags);
  if (rc != ATTN_OK) return rc;
  if (d.B < 0 || d.W < 0 || d.num_pages < 0 || d.tokens < 0)
    return fail(ATTN_ERR_SHAPE, "extents must not be negative");
  const int shift = page_shift(d.page_size);
  if (shift < 0)
    return fail(ATTN_ERR_UNSUPPORTED, "page_size must be a power of two from 16 to 1024 (got %d)",
                d.page_size);
  if (d.B > cache_plan::kMaxRequests)
    return fail(ATTN_ERR_UNSUPPORTED, "at most %d requests a call (got %lld)",
                cache_plan::kMaxRequests, (long long)d.B);
  if (d.num_pages > kInt32 || d.tokens > kInt32 || d.W > kInt32 || (d.W << shift) > kInt32 ||
      d.B * d.W > kInt32)
    return fail(ATTN_ERR_SHAPE, "extent too large");
  if (d.B > 1 && d.table_stride < d.W) return fail(ATTN_ERR_STRIDE, "block_table rows overlap");
  if (!d.free_count || !d.free_count_out || !d.starts ||
      (d.B > 0 && (!d.lengths || !d.targets || !d.lengths_out)) ||
      (d.B > 0 && d.W > 0 && !d.block_table) || (d.num_pages > 0 && !d.free_pages) ||
      (d.tokens > 0 && !d.slots))
    return fail(ATTN_ERR_INVALID, "null pointer");
  return ATTN_OK;
}

int run(const AttnCachePlan& d, cudaStream_t s) {
  rt_host::Device dev;
  int rc = rt_host::device_ready(&dev);
  if (rc != ATTN_OK) return rc;
  rc = check_pointers(d.flags, {d.lengths, d.targets, d.block_table, d.free_pages, d.free_count,
                                d.lengths_out, d.free_count_out, d.starts, d.positions, d.slots,
                                d.status});
  if (rc != ATTN_OK) return rc;
  cache_plan::Params p{};
  p.B = static_cast<int>(d.B);
  p.W = static_cast<int>(d.W);
  p.page_shift = page_shift(d.page_size);
  p.num_pages = static_cast<int>(d.num_pages);
  p.tokens = static_cast<int>(d.tokens);
  p.table_stride = d.table_stride;
  p.lengths = d.lengths;
  p.targets = d.targets;
  p.table = d.block_table;
  p.free_pages = d.free_pages;
  p.free_count = d.free_count;
  p.lengths_out = d.lengths_out;
  p.free_count_out = d.free_count_out;
  p.starts = d.starts;
  p.positions = d.positions;
  p.slots = d.slots;
  p.status = d.status ? d.status : dev.status;
  const size_t smem = (5 * static_cast<size_t>(d.B) + 3) * sizeof(int);
  static std::once_flag once[64];
  static cudaError_t attr[64];
  std::call_once(once[dev.index], [&] {
    attr[dev.index] = cudaFuncSetAttribute(cache_plan::plan_kernel,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (5 * cache_plan::kMaxRequests + 3) * int{sizeof(int)});
  });
  if (attr[dev.index] != cudaSuccess) return cuda_fail(attr[dev.index], "cudaFuncSetAttribute");
  const int64_t work = std::max(d.B, d.tokens);
  const int blocks = static_cast<int>(std::min<int64_t>(8, (work + 4095) / 4096));
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(std::max(1, blocks));
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(at.val.clusterDim.x);
  cfg.blockDim = dim3(work <= 256 ? 256 : 1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, cache_plan::plan_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "cache_plan launch");
  rt_host::count_launches(1);
  return ATTN_OK;
}

// ----------------------------------------------------------------- append
int check(const AttnCacheAppend& d) {
  int rc = check_flags(d.flags);
  if (rc != ATTN_OK) return rc;
  if (d.N < 0 || d.T < 0 || d.Hkv < 0 || d.D < 0 || d.num_pages < 0)
    return fail(ATTN_ERR_SHAPE, "extents must not be negative");
  if (d.dtype != ATTN_BF16 && d.dtype != ATTN_F16)
    return fail(ATTN_ERR_DTYPE, "keys and values must be bf16 or f16");
  if (d.cache_dtype != d.dtype && d.cache_dtype != ATTN_E4M3)
    return fail(ATTN_ERR_DTYPE, "the cache must have the keys' type or e4m3");
  if (page_shift(d.page_size) < 0)
    return fail(ATTN_ERR_UNSUPPORTED, "page_size must be a power of two from 16 to 1024 (got %d)",
                d.page_size);
  if (d.D % 16 != 0)
    return fail(ATTN_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 (got %lld)", (long long)d.D);
  if (d.N > kInt32 || d.T > kInt32 || d.num_pages > kInt32 || d.Hkv * d.D > kInt32)
    return fail(ATTN_ERR_SHAPE, "extent too large");
  if (!d.rows && d.N > d.T)
    return fail(ATTN_ERR_SHAPE, "more slots (%lld) than rows (%lld)", (long long)d.N, (long long)d.T);
  if (d.N == 0 || d.Hkv == 0 || d.D == 0) return ATTN_OK;
  if (!d.slots || (d.T > 0 && (!d.k || !d.v)) || (d.num_pages > 0 && (!d.k_cache || !d.v_cache)))
    return fail(ATTN_ERR_INVALID, "null pointer");
  const bool fp8 = d.cache_dtype == ATTN_E4M3;
  if (fp8 && !(d.k_descale > 0.f && d.v_descale > 0.f && std::isfinite(d.k_descale) &&
               std::isfinite(d.v_descale)))
    return fail(ATTN_ERR_INVALID, "e4m3 descales must be positive and finite");
  if (!fp8 && (d.k_descale_heads || d.v_descale_heads || d.k_descale != 1.f || d.v_descale != 1.f))
    return fail(ATTN_ERR_DTYPE, "descales apply to e4m3 caches only");
  const int64_t ca = fp8 ? 16 : 8;
  for (const void* ptr : {d.k, d.v, static_cast<const void*>(d.k_cache), static_cast<const void*>(d.v_cache)})
    if (!aligned(ptr, 16)) return fail(ATTN_ERR_ALIGN, "keys, values and caches must be 16-byte aligned");
  for (const int64_t* st : {d.k_stride, d.v_stride})
    if (!stride_ok(st[0], d.T, 8) || !stride_ok(st[1], d.Hkv, 8))
      return fail(ATTN_ERR_ALIGN, "strides of keys and values must be multiples of 16 bytes");
  for (const int64_t* st : {d.k_cache_stride, d.v_cache_stride})
    if (!stride_ok(st[0], d.num_pages, ca) || !stride_ok(st[1], d.Hkv, ca) || st[2] % ca != 0)
      return fail(ATTN_ERR_ALIGN, "cache strides must be multiples of 16 bytes");
  for (const int64_t* st : {d.k_cache_stride, d.v_cache_stride})
    if (!apart(st[0], d.num_pages, d.D) || !apart(st[1], d.Hkv, d.D) || !apart(st[2], d.page_size, d.D))
      return fail(ATTN_ERR_STRIDE, "rows of the cache overlap");
  return ATTN_OK;
}

int run(const AttnCacheAppend& d, cudaStream_t s) {
  if (d.N == 0 || d.Hkv == 0 || d.D == 0) return ATTN_OK;
  rt_host::Device dev;
  int rc = rt_host::device_ready(&dev);
  if (rc != ATTN_OK) return rc;
  rc = check_pointers(d.flags, {d.k, d.v, d.k_cache, d.v_cache, d.slots, d.rows, d.k_descale_heads,
                                d.v_descale_heads, d.status});
  if (rc != ATTN_OK) return rc;
  cache_append::Params p{};
  p.N = d.N;
  p.T = d.T;
  p.page_shift = page_shift(d.page_size);
  p.slots_in_cache = d.num_pages << p.page_shift;
  p.Hkv = static_cast<int>(d.Hkv);
  p.chunks = static_cast<int>(d.D / 16);
  p.k_st = d.k_stride[0], p.k_sh = d.k_stride[1];
  p.v_st = d.v_stride[0], p.v_sh = d.v_stride[1];
  p.kc_sp = d.k_cache_stride[0], p.kc_sh = d.k_cache_stride[1], p.kc_st = d.k_cache_stride[2];
  p.vc_sp = d.v_cache_stride[0], p.vc_sh = d.v_cache_stride[1], p.vc_st = d.v_cache_stride[2];
  p.k = d.k, p.v = d.v, p.kc = d.k_cache, p.vc = d.v_cache;
  p.slots = d.slots;
  p.rows = d.rows;
  p.k_descale_heads = d.k_descale_heads, p.v_descale_heads = d.v_descale_heads;
  p.k_descale = d.k_descale, p.v_descale = d.v_descale;
  p.status = d.status ? d.status : dev.status;
  // Rows per block: two chunks a thread where there are rows enough to fill
  // the GPU, else one row a block.
  const int per_row = p.Hkv * p.chunks;
  p.tile = d.N <= 4 * dev.sms ? 1 : std::max(1, 2 * cache_append::kThreads / per_row);
  const unsigned blocks = static_cast<unsigned>((d.N + p.tile - 1) / p.tile);
  const bool fp8 = d.cache_dtype == ATTN_E4M3;
  auto kern = d.dtype == ATTN_F16
                  ? (fp8 ? cache_append::append_kernel<true, true> : cache_append::append_kernel<true, false>)
                  : (fp8 ? cache_append::append_kernel<false, true>
                         : cache_append::append_kernel<false, false>);
  kern<<<blocks, cache_append::kThreads, 0, s>>>(p);
  return launched("cache_append launch");
}

// ----------------------------------------------------------------- rotary
int check(const AttnRotary& d) {
  int rc = check_flags(d.flags);
  if (rc != ATTN_OK) return rc;
  if (d.B < 0 || d.N < 0 || d.Hq < 0 || d.Hk < 0 || d.D < 0 || d.R < 0)
    return fail(ATTN_ERR_SHAPE, "extents must not be negative");
  if (d.dtype != ATTN_F32 && d.dtype != ATTN_BF16 && d.dtype != ATTN_F16)
    return fail(ATTN_ERR_DTYPE, "rotary takes f32, bf16 or f16");
  if (d.R % 2 != 0 || d.R > d.D)
    return fail(ATTN_ERR_SHAPE, "the turned values must be an even number up to head_dim (%lld of %lld)",
                (long long)d.R, (long long)d.D);
  if (d.D > 1024) return fail(ATTN_ERR_UNSUPPORTED, "rotary supports head_dim <= 1024");
  if (d.num_axes < 1) return fail(ATTN_ERR_SHAPE, "positions need an axis");
  if (d.N > kInt32 || d.B > kInt32 || d.B * d.N > kInt32 || (d.Hq + d.Hk) * d.D > kInt32)
    return fail(ATTN_ERR_SHAPE, "extent too large");
  if (d.B * d.N == 0 || (d.Hq + d.Hk) * d.D == 0) return ATTN_OK;
  if ((d.Hq > 0 && (!d.q || !d.qo)) || (d.Hk > 0 && (!d.k || !d.ko)) ||
      (d.R > 0 && (!d.positions || !d.freqs)))
    return fail(ATTN_ERR_INVALID, "null pointer");
  const unsigned eb = d.dtype == ATTN_F32 ? 4 : 2;
  for (const void* ptr : {d.q, d.k, static_cast<const void*>(d.qo), static_cast<const void*>(d.ko)})
    if (!aligned(ptr, eb)) return fail(ATTN_ERR_ALIGN, "Q and K must be aligned to their elements");
  struct { const int64_t* st; int64_t heads; } outs[] = {{d.qo_stride, d.Hq}, {d.ko_stride, d.Hk}};
  for (const auto& o : outs)
    if (o.heads > 0 && (!apart(o.st[0], d.B, d.D) || !apart(o.st[1], o.heads, d.D) || !apart(o.st[2], d.N, d.D)))
      return fail(ATTN_ERR_STRIDE, "rows of the results overlap");
  return ATTN_OK;
}

template <typename T, int V>
int launch_rotary(const AttnRotary& d, const rotary::Params& p, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((p.tokens + p.tile - 1) / p.tile);
  const size_t smem = sizeof(float2) * p.tile * p.half;
  if (d.neighbours)
    rotary::rotary_kernel<T, V, true><<<blocks, rotary::kThreads, smem, s>>>(p);
  else
    rotary::rotary_kernel<T, V, false><<<blocks, rotary::kThreads, smem, s>>>(p);
  return launched("rotary launch");
}

int run(const AttnRotary& d, cudaStream_t s) {
  if (d.B * d.N == 0 || (d.Hq + d.Hk) * d.D == 0) return ATTN_OK;
  rt_host::Device dev;
  int rc = rt_host::device_ready(&dev);
  if (rc != ATTN_OK) return rc;
  rc = check_pointers(d.flags, {d.Hq ? d.q : nullptr, d.Hk ? d.k : nullptr, d.Hq ? d.qo : nullptr,
                                d.Hk ? d.ko : nullptr, d.positions, d.freqs, d.axes, d.status});
  if (rc != ATTN_OK) return rc;
  rotary::Params p{};
  p.tokens = d.B * d.N;
  p.N = d.N;
  p.Hq = static_cast<int>(d.Hq);
  p.H = static_cast<int>(d.Hq + d.Hk);
  p.D = static_cast<int>(d.D);
  p.half = static_cast<int>(d.R / 2);
  p.q_sb = d.q_stride[0], p.q_sh = d.q_stride[1], p.q_sn = d.q_stride[2];
  p.k_sb = d.k_stride[0], p.k_sh = d.k_stride[1], p.k_sn = d.k_stride[2];
  p.qo_sb = d.qo_stride[0], p.qo_sh = d.qo_stride[1], p.qo_sn = d.qo_stride[2];
  p.ko_sb = d.ko_stride[0], p.ko_sh = d.ko_stride[1], p.ko_sn = d.ko_stride[2];
  p.p_sa = d.pos_stride[0], p.p_sb = d.pos_stride[1], p.p_sn = d.pos_stride[2];
  p.q = d.q, p.k = d.k, p.qo = d.qo, p.ko = d.ko;
  p.positions = d.positions;
  p.freqs = d.freqs;
  p.axes = d.axes;
  p.status = d.status ? d.status : dev.status;
  p.num_axes = d.num_axes;
  p.positions_64 = d.positions_64;
  p.sign = d.inverse ? -1.f : 1.f;
  // 16-byte packs where every row, its second half and its tail allow them.
  const int eb = d.dtype == ATTN_F32 ? 4 : 2, vec = 16 / eb;
  bool wide = p.D % vec == 0 && p.half % vec == 0;
  struct { const void* ptr; const int64_t* st; int64_t heads; } ops[] = {
      {d.q, d.q_stride, d.Hq}, {d.qo, d.qo_stride, d.Hq}, {d.k, d.k_stride, d.Hk}, {d.ko, d.ko_stride, d.Hk}};
  for (const auto& o : ops)
    if (o.heads > 0)
      wide = wide && aligned(o.ptr, 16) && stride_ok(o.st[0], d.B, vec) && stride_ok(o.st[1], o.heads, vec) &&
             stride_ok(o.st[2], d.N, vec);
  // Units of a head: two packs each (one by one where rows are not aligned).
  const int per_head = !wide ? p.D - p.half
                             : ((2 * p.half / vec) + 1) / 2 + ((p.D - 2 * p.half) / vec + 1) / 2;
  p.lanes_shift = pow2_shift(per_head, 0, 8);
  p.heads_shift = p.H > 1 ? pow2_shift(p.H, 0, 8) - (p.H & (p.H - 1) ? 1 : 0) : 0;  // rounded down
  // Tokens per block: eight units a thread where there are tokens enough to
  // fill the GPU so, else one; and angles within 32 KB.
  const int per_token = std::max(1, p.H << p.lanes_shift);
  const int64_t units = p.tokens * per_token;
  const int each = units >= int64_t{8} * rotary::kThreads * 8 * dev.sms ? 8 : 1;
  p.tile = std::max(1, each * rotary::kThreads / per_token);
  if (p.half > 0) p.tile = std::max(1, std::min(p.tile, 4096 / p.half));
  switch (d.dtype) {
    case ATTN_F32: return wide ? launch_rotary<float, 4>(d, p, s) : launch_rotary<float, 1>(d, p, s);
    case ATTN_F16: return wide ? launch_rotary<__half, 8>(d, p, s) : launch_rotary<__half, 1>(d, p, s);
    default:
      return wide ? launch_rotary<__nv_bfloat16, 8>(d, p, s) : launch_rotary<__nv_bfloat16, 1>(d, p, s);
  }
}

// ------------------------------------------------------------------- tree
int check(const AttnTree& d) {
  int rc = check_flags(d.flags);
  if (rc != ATTN_OK) return rc;
  if (d.B < 0 || d.T < 0 || d.Hq < 0 || d.Hkv < 0 || d.W < 0 || d.num_pages < 0 || d.max_new < 0)
    return fail(ATTN_ERR_SHAPE, "extents must not be negative");
  if (d.dtype != ATTN_BF16 && d.dtype != ATTN_F16)
    return fail(ATTN_ERR_DTYPE, "queries must be bf16 or f16");
  if (d.cache_dtype != d.dtype && d.cache_dtype != ATTN_E4M3)
    return fail(ATTN_ERR_DTYPE, "the cache must have the queries' type or e4m3");
  const int shift = page_shift(d.page_size);
  if (shift < 0)
    return fail(ATTN_ERR_UNSUPPORTED, "page_size must be a power of two from 16 to 1024 (got %d)",
                d.page_size);
  if (d.cache_dtype == ATTN_E4M3 ? d.D != 128 : (d.D != 64 && d.D != 128))
    return fail(ATTN_ERR_UNSUPPORTED, "head_dim must be 64 or 128, with an e4m3 cache 128 (got %lld)",
                (long long)d.D);
  if (d.Hq > 0 && (d.Hkv <= 0 || d.Hq % d.Hkv != 0))
    return fail(ATTN_ERR_SHAPE, "query heads (%lld) must be a multiple of key/value heads (%lld)",
                (long long)d.Hq, (long long)d.Hkv);
  if (d.Hq > 0 && d.Hq / d.Hkv > 64)
    return fail(ATTN_ERR_UNSUPPORTED, "at most 64 query heads share a key head (got %lld)",
                (long long)(d.Hq / d.Hkv));
  if (d.B > 65535 || d.T > kInt32 || d.Hq > 65535 || d.max_new > kInt32 || d.num_pages > kInt32 ||
      d.W > kInt32 || (d.W << shift) > kInt32 || d.T * d.Hq > kInt32)
    return fail(ATTN_ERR_SHAPE, "extent too large");
  if (d.B == 0 || d.T == 0 || d.Hq == 0 || d.max_new == 0) return ATTN_OK;
  if (!d.q || !d.k_new || !d.v_new || !d.o || !d.lengths || !d.starts ||
      (d.W > 0 && !d.block_table) || (d.num_pages > 0 && (!d.k_cache || !d.v_cache)))
    return fail(ATTN_ERR_INVALID, "null pointer");
  if (d.B > 1 && d.table_stride < d.W) return fail(ATTN_ERR_STRIDE, "block_table rows overlap");
  if (d.mask && d.T > 1 && d.mask_stride < d.max_new)
    return fail(ATTN_ERR_STRIDE, "mask rows must hold max_new columns");
  if (!std::isfinite(d.scale)) return fail(ATTN_ERR_INVALID, "scale must be finite");
  const bool fp8 = d.cache_dtype == ATTN_E4M3;
  if (fp8 && !(d.k_descale > 0.f && d.v_descale > 0.f && std::isfinite(d.k_descale) &&
               std::isfinite(d.v_descale)))
    return fail(ATTN_ERR_INVALID, "e4m3 descales must be positive and finite");
  if (!fp8 && (d.k_descale_heads || d.v_descale_heads || d.k_descale != 1.f || d.v_descale != 1.f))
    return fail(ATTN_ERR_DTYPE, "descales apply to e4m3 caches only");
  for (const void* ptr : {d.q, d.k_new, d.v_new, d.k_cache, d.v_cache, static_cast<const void*>(d.o)})
    if (!aligned(ptr, 16)) return fail(ATTN_ERR_ALIGN, "queries, keys, values and output must be 16-byte aligned");
  struct { const int64_t* st; int64_t heads; } rows[] = {
      {d.q_stride, d.Hq}, {d.k_stride, d.Hkv}, {d.v_stride, d.Hkv}, {d.o_stride, d.Hq}};
  for (const auto& r : rows)
    if (!stride_ok(r.st[0], d.T, 8) || !stride_ok(r.st[1], r.heads, 8))
      return fail(ATTN_ERR_ALIGN, "strides must be multiples of 16 bytes");
  const int64_t ca = fp8 ? 16 : 8;
  for (const int64_t* st : {d.k_cache_stride, d.v_cache_stride})
    if (!stride_ok(st[0], d.num_pages, ca) || !stride_ok(st[1], d.Hkv, ca) || st[2] % ca != 0)
      return fail(ATTN_ERR_ALIGN, "cache strides must be multiples of 16 bytes");
  if (!apart(d.o_stride[0], d.T, d.D) || !apart(d.o_stride[1], d.Hq, d.D))
    return fail(ATTN_ERR_STRIDE, "rows of the result overlap");
  return ATTN_OK;
}

// Tensor maps of 5 dimensions, innermost first, with 128-byte swizzle.
// Strides in bytes, of dimensions 1 to 4.
int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, const int64_t (&dims)[5],
             int64_t (&strides)[4], const int (&box)[5]) {
  const rt_host::EncodeTiled encode = rt_host::tensor_map_encoder();
  if (!encode) return fail(ATTN_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], step[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < 5; ++i) d[i] = static_cast<cuuint64_t>(dims[i]), b[i] = static_cast<cuuint32_t>(box[i]);
  for (int i = 0; i < 4; ++i) {
    if (dims[i + 1] == 1) strides[i] = 128;  // never stepped along
    if (strides[i] < 0 || strides[i] % 16 != 0 || strides[i] >= (int64_t{1} << 40))
      return fail(ATTN_ERR_STRIDE, "a stride is negative or past 2^40 bytes");
    s[i] = static_cast<cuuint64_t>(strides[i]);
  }
  const CUresult r = encode(map, type, 5, const_cast<void*>(base), d, s, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ATTN_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return ATTN_OK;
}

// The four key and value operands as [pages][heads][halves][tokens][128 bytes]
// (new tokens: one page): boxes of `box` cached or `new_box` new tokens of one
// head, all halves of its row at once or one.
struct KeyMaps {
  CUtensorMap kc, vc, kn, vn;
};

int make_key_maps(KeyMaps* m, const AttnTree& d, int box, int new_box, bool all_halves) {
  const CUtensorMapDataType t16 =
      d.dtype == ATTN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto one = [&](CUtensorMap* map, const void* base, CUtensorMapDataType type, int eb, int64_t tokens, int64_t pages,
                 int64_t s_token, int64_t s_head, int64_t s_page, int rows) {
    const int64_t inner = 128 / eb, halves = d.D * eb / 128;
    const int64_t dims[5] = {inner, tokens, halves, d.Hkv, pages};
    int64_t strides[4] = {s_token * eb, 128, s_head * eb, s_page * eb};
    const int b[5] = {static_cast<int>(inner), rows, all_halves ? static_cast<int>(halves) : 1, 1, 1};
    return make_map(map, base, type, dims, strides, b);
  };
  const bool fp8 = d.cache_dtype == ATTN_E4M3;
  const CUtensorMapDataType tc = fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : t16;
  const int eb = fp8 ? 1 : 2;
  const int64_t *ks = d.k_cache_stride, *vs = d.v_cache_stride;
  // A cache without pages is never read: its map stands on q.
  const void* kc = d.num_pages ? d.k_cache : d.q;
  const void* vc = d.num_pages ? d.v_cache : d.q;
  const int64_t pages = std::max<int64_t>(d.num_pages, 1);
  int rc;
  if ((rc = one(&m->kc, kc, tc, eb, d.page_size, pages, ks[2], ks[1], ks[0], box)) != ATTN_OK ||
      (rc = one(&m->vc, vc, tc, eb, d.page_size, pages, vs[2], vs[1], vs[0], box)) != ATTN_OK ||
      (rc = one(&m->kn, d.k_new, t16, 2, d.T, 1, d.k_stride[0], d.k_stride[1], 0, new_box)) != ATTN_OK ||
      (rc = one(&m->vn, d.v_new, t16, 2, d.T, 1, d.v_stride[0], d.v_stride[1], 0, new_box)) != ATTN_OK)
    return rc;
  return ATTN_OK;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Scratch for the cut items of a launch whose work is cut into `shares`.
int tree_scratch(attn_tree::Scratch* out, void** base, int shares, int rows, int D, cudaStream_t s) {
  const size_t slots = 2 * static_cast<size_t>(shares);
  const size_t rec = round256(shares * sizeof(attn_tree::Record)), ml = round256(slots * rows * sizeof(float));
  const cudaError_t e = rt_host::scratch(base, rec + 2 * ml + slots * rows * D * sizeof(float), s);
  if (e != cudaSuccess) return cuda_fail(e, "stream-ordered scratch (cut items)");
  char* at = static_cast<char*>(*base);
  out->record = reinterpret_cast<attn_tree::Record*>(at);
  out->m = reinterpret_cast<float*>(at + rec);
  out->l = reinterpret_cast<float*>(at + rec + ml);
  out->o = reinterpret_cast<float4*>(at + rec + 2 * ml);
  return ATTN_OK;
}

// Programmatic launch: the kernel is set up while the one before it in the
// stream still runs, and waits on the device for that one's end.
template <typename... K, typename... A>
cudaError_t launch_early(void (*kern)(K...), dim3 grid, int threads, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}

// Both kernels keep the SM's memory split as the first one needs it: a change
// of it between them would drain the SM.
// `pool`: what the kernel's warpgroups divide among themselves has to fit in
// the registers that a block is launched with, or the raise would wait forever.
template <typename K, typename J>
cudaError_t prepare_kernels(K kern, J join, size_t smem, int threads, int pool) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(join, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  cudaFuncAttributes fa{};
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kern);
  if (e == cudaSuccess && fa.numRegs * threads < pool) e = cudaErrorLaunchOutOfResources;
  return e;
}

template <typename T, typename TC, int D, int MT>
int launch_tree_mma(const AttnTree& d, const attn_tree::Params& p, const rt_host::Device& dev, cudaStream_t s) {
  using C = attn_tree::MmaCfg<T, TC, D, MT>;
  auto kern = attn_tree::tree_mma_kernel<T, TC, D, MT>;
  auto join = attn_tree::tree_mma_join<T, D, C::kRows>;
  static std::once_flag once[64];
  static cudaError_t attr[64];
  std::call_once(once[dev.index], [&] {
    attr[dev.index] = prepare_kernels(kern, join, C::kSmem, attn_tree::kMmaThreads, attn_tree::kMmaRegPool);
  });
  if (attr[dev.index] != cudaSuccess) return cuda_fail(attr[dev.index], "set-up of a kernel");
  attn_tree::Split split;
  split.rows = C::kRows;
  split.keys_shift = C::kKeysShift;
  split.new_shift = pow2_shift(p.max_new, 3, C::kNewShift);
  KeyMaps m;
  int rc = make_key_maps(&m, d, std::min(1 << p.page_shift, 1 << C::kKeysShift), 1 << split.new_shift, true);
  if (rc != ATTN_OK) return rc;
  const int shares = attn_tree::kMmaTeams * dev.sms;
  const int rows = static_cast<int>(std::min<int64_t>(C::kRows, static_cast<int64_t>(p.max_new) * p.group));
  attn_tree::Scratch sc{};
  void* base = nullptr;
  if ((rc = tree_scratch(&sc, &base, shares, C::kRows, D, s)) != ATTN_OK) return rc;
  cudaError_t e = launch_early(kern, dim3(dev.sms), attn_tree::kMmaThreads, C::kSmem, s, m.kc, m.vc, m.kn, m.vn, p,
                               split, sc, 1);
  if (e == cudaSuccess) {
    // Rows of a join block: about twice the blocks that fit at once; more
    // would come too late to hide their start.
    const int at_once = dev.sms * (2048 / attn_tree::kJoinThreads);
    const int each = std::max(1, shares * rows / (2 * at_once));
    e = launch_early(join, dim3(shares, (rows + each - 1) / each), attn_tree::kJoinThreads, 0, s, p, sc, each,
                     C::kShift);
  }
  cudaFreeAsync(base, s);
  if (e != cudaSuccess) return cuda_fail(e, "attn_tree launch");
  rt_host::count_launches(2);
  return ATTN_OK;
}

// The kernel for few rows, with one 16-row tile, two or (D = 64, more than 40
// rows, work for every SM) three, which read each key once where two tiles are
// two items.  Measured, us, 48 rows by three and by two: 256 items of up to 4096
// keys 100 and 115, 800 of 8000 keys 281 and 351, of 100 keys 52 and 49; 32 items
// 42 and 38.  40 rows: 400 items of 8000 keys 157 and 152, of 1500 81 and 69.
template <typename T, typename TC, int D>
int launch_tree_few(const AttnTree& d, const attn_tree::Params& p, int64_t rows, const rt_host::Device& dev,
                    cudaStream_t s) {
  if (rows <= 16) return launch_tree_mma<T, TC, D, 1>(d, p, dev, s);
  if constexpr (D == 64) {
    if (rows > 40 && d.B * d.Hkv >= dev.sms) return launch_tree_mma<T, TC, D, 3>(d, p, dev, s);
  }
  return launch_tree_mma<T, TC, D, 2>(d, p, dev, s);
}

template <typename T, int D, bool MASK, bool ALONE>
int launch_tree_tc(const AttnTree& d, const attn_tree::Params& p, const rt_host::Device& dev, cudaStream_t s) {
  using C = attn_tree::tc::Cfg<T, D, MASK, ALONE>;
  auto kern = attn_tree::tc::tree_tc_kernel<T, D, MASK, ALONE>;
  static std::once_flag once[64];
  static cudaError_t attr[64];
  std::call_once(once[dev.index], [&] {
    attr[dev.index] = prepare_kernels(kern, attn_tree::tc::tree_tc_join<T, D>, C::kSmem, attn_tree::tc::kThreads,
                                      attn_tree::tc::kRegPool);
  });
  if (attr[dev.index] != cudaSuccess) return cuda_fail(attr[dev.index], "set-up of a kernel");
  attn_tree::tc::Tiles tiles;
  tiles.box = std::max(1, std::min(attn_tree::tc::kTileRows / p.group, p.max_new));
  tiles.rows = tiles.box * p.group;
  attn_tree::Split split;
  split.rows = 2 * tiles.rows;
  split.keys_shift = 7;
  split.new_shift = pow2_shift(p.max_new, 3, 7);
  KeyMaps m;
  int rc = make_key_maps(&m, d, std::min(1 << p.page_shift, attn_tree::tc::kTileKeys), 1 << split.new_shift, false);
  if (rc != ATTN_OK) return rc;
  // Q as [kv heads][halves][tokens][heads of a group][128 bytes].
  CUtensorMap mq;
  const int64_t dims[5] = {64, p.group, d.T, D / 64, d.Hkv};
  int64_t strides[4] = {d.q_stride[1] * 2, d.q_stride[0] * 2, 128, d.q_stride[1] * 2 * p.group};
  const int box[5] = {64, p.group, tiles.box, 1, 1};
  const CUtensorMapDataType t16 = C::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if ((rc = make_map(&mq, d.q, t16, dims, strides, box)) != ATTN_OK) return rc;
  const int blocks = dev.sms;
  const int rows = static_cast<int>(std::min<int64_t>(split.rows, static_cast<int64_t>(p.max_new) * p.group));
  attn_tree::Scratch sc{};
  void* base = nullptr;
  if ((rc = tree_scratch(&sc, &base, blocks, 256, D, s)) != ATTN_OK) return rc;
  cudaError_t e = launch_early(kern, dim3(blocks), attn_tree::tc::kThreads, C::kSmem, s, mq, m.kc, m.vc, m.kn, m.vn,
                               p, split, tiles, sc, 1);
  if (e == cudaSuccess)
    e = launch_early(attn_tree::tc::tree_tc_join<T, D>,
                     dim3(blocks, (rows + attn_tree::tc::kJoinRows - 1) / attn_tree::tc::kJoinRows),
                     attn_tree::tc::kJoinThreads, 0, s, p, sc);
  cudaFreeAsync(base, s);
  if (e != cudaSuccess) return cuda_fail(e, "attn_tree launch");
  rt_host::count_launches(2);
  return ATTN_OK;
}

// The kernel for many rows; a request of one row tile is alone with its keys.
template <typename T, int D>
int launch_tree_many(const AttnTree& d, const attn_tree::Params& p, int64_t rows, const rt_host::Device& dev,
                     cudaStream_t s) {
  if (rows <= attn_tree::tc::kTileRows / p.group * p.group)
    return d.mask ? launch_tree_tc<T, D, true, true>(d, p, dev, s) : launch_tree_tc<T, D, false, true>(d, p, dev, s);
  return d.mask ? launch_tree_tc<T, D, true, false>(d, p, dev, s) : launch_tree_tc<T, D, false, false>(d, p, dev, s);
}

// The choice of kernel.
int launch_tree(const AttnTree& d, const attn_tree::Params& p, const rt_host::Device& dev, cudaStream_t s) {
  using H = __half;
  using N = __nv_bfloat16;
  using E = __nv_fp8_e4m3;
  const bool fp8 = d.cache_dtype == ATTN_E4M3;
  const int64_t rows = static_cast<int64_t>(p.max_new) * p.group;
  // Measured, us, by the mma kernel (two row tiles) and by tcgen05.  D = 64,
  // 100 requests with a mask, 1500 keys: 40 rows 69 and 86, 48 rows 135 and
  // 164, 64 rows 93 and 87, 96 rows 227 and 165.  D = 128: 40 rows 100 and 102,
  // without a mask 98 and 86, 64 rows 132 and 87.
  if (!fp8 && rows > (d.D == 64 ? 48 : 32)) {
    if (d.dtype == ATTN_F16)
      return d.D == 64 ? launch_tree_many<H, 64>(d, p, rows, dev, s) : launch_tree_many<H, 128>(d, p, rows, dev, s);
    return d.D == 64 ? launch_tree_many<N, 64>(d, p, rows, dev, s) : launch_tree_many<N, 128>(d, p, rows, dev, s);
  }
  auto launch = d.dtype == ATTN_F16 ? (fp8 ? launch_tree_few<H, E, 128>
                                           : d.D == 64 ? launch_tree_few<H, H, 64> : launch_tree_few<H, H, 128>)
                                    : (fp8 ? launch_tree_few<N, E, 128>
                                           : d.D == 64 ? launch_tree_few<N, N, 64> : launch_tree_few<N, N, 128>);
  return launch(d, p, rows, dev, s);
}

// With rows that may be hidden from a new key: values that are no numbers stay
// where they are seen (see clean_values).
template <typename T, int D>
int launch_tree_hidden(const AttnTree& d, const attn_tree::Params& p, const rt_host::Device& dev, cudaStream_t s) {
  constexpr int kThreads = attn_tree::kValueThreads;
  auto clean = attn_tree::clean_values<T, D>;
  auto whole = attn_tree::whole_values<T, D>;
  static std::once_flag once[64];
  static cudaError_t attr[64];
  std::call_once(once[dev.index], [&] {
    cudaError_t& e = attr[dev.index];
    e = cudaFuncSetAttribute(clean, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(whole, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
  if (attr[dev.index] != cudaSuccess) return cuda_fail(attr[dev.index], "set-up of a kernel");
  const int64_t packs = d.T * d.Hkv * (D / 8);
  const int blocks = static_cast<int>(std::min<int64_t>((packs + kThreads - 1) / kThreads, 4ll * dev.sms));
  const size_t flags = round256(blocks * sizeof(int));
  void* base = nullptr;
  cudaError_t e = rt_host::scratch(&base, flags + packs * 16, s);
  if (e != cudaSuccess) return cuda_fail(e, "stream-ordered scratch (new values)");
  int* const odd = static_cast<int*>(base);
  AttnTree c = d;
  c.v_new = static_cast<char*>(base) + flags;
  c.v_stride[0] = d.Hkv * D, c.v_stride[1] = D;
  e = launch_early(clean, dim3(blocks), kThreads, 0, s, p, reinterpret_cast<uint4*>(static_cast<char*>(base) + flags),
                   odd);
  const int rc = e == cudaSuccess ? launch_tree(c, p, dev, s) : ATTN_OK;
  if (e == cudaSuccess && rc == ATTN_OK) {
    // At most 16 blocks go over a request's values of one head.
    const int rows_each = std::max(128, (p.max_new + 15) / 16), splits = (p.max_new + rows_each - 1) / rows_each;
    const int64_t items = d.B * d.Hkv * splits;
    e = launch_early(whole, dim3(static_cast<unsigned>(std::min<int64_t>(items, dev.sms))), kThreads, 0, s, p, odd, blocks,
                     rows_each, splits);
  }
  cudaFreeAsync(base, s);
  if (rc != ATTN_OK) return rc;
  if (e != cudaSuccess) return cuda_fail(e, "attn_tree launch");
  rt_host::count_launches(2);
  return ATTN_OK;
}

int run(const AttnTree& d, cudaStream_t s) {
  if (d.B == 0 || d.T == 0 || d.Hq == 0 || d.max_new == 0) return ATTN_OK;
  rt_host::Device dev;
  int rc = rt_host::device_ready(&dev);
  if (rc != ATTN_OK) return rc;
  rc = check_pointers(d.flags, {d.q, d.k_new, d.v_new, d.k_cache, d.v_cache, d.o, d.lse, d.block_table,
                                d.lengths, d.starts, d.mask, d.k_descale_heads, d.v_descale_heads,
                                d.status});
  if (rc != ATTN_OK) return rc;
  attn_tree::Params p{};
  p.B = static_cast<int>(d.B);
  p.T = static_cast<int>(d.T);
  p.Hq = static_cast<int>(d.Hq);
  p.Hkv = static_cast<int>(d.Hkv);
  p.group = static_cast<int>(d.Hq / d.Hkv);
  p.W = static_cast<int>(d.W);
  p.num_pages = static_cast<int>(d.num_pages);
  p.page_shift = page_shift(d.page_size);
  p.max_new = static_cast<int>(std::min(d.max_new, d.T));
  p.q_st = d.q_stride[0], p.q_sh = d.q_stride[1];
  p.k_st = d.k_stride[0], p.k_sh = d.k_stride[1];
  p.v_st = d.v_stride[0], p.v_sh = d.v_stride[1];
  p.o_st = d.o_stride[0], p.o_sh = d.o_stride[1];
  p.kc_sp = d.k_cache_stride[0], p.kc_sh = d.k_cache_stride[1], p.kc_st = d.k_cache_stride[2];
  p.vc_sp = d.v_cache_stride[0], p.vc_sh = d.v_cache_stride[1], p.vc_st = d.v_cache_stride[2];
  p.table_stride = d.table_stride;
  p.mask_stride = d.mask_stride;
  p.mask_align = d.T > 1 ? static_cast<int>((reinterpret_cast<uintptr_t>(d.mask) | d.mask_stride) & 15u)
                         : static_cast<int>(reinterpret_cast<uintptr_t>(d.mask) & 15u);
  p.mask_align = p.mask_align == 0 ? 16 : p.mask_align & -p.mask_align;
  p.q = d.q, p.k_new = d.k_new, p.v_new = d.v_new;
  p.k_cache = d.k_cache, p.v_cache = d.v_cache;
  p.o = d.o, p.lse = d.lse;
  p.table = d.block_table, p.lengths = d.lengths, p.starts = d.starts, p.mask = d.mask;
  p.k_descale_heads = d.k_descale_heads, p.v_descale_heads = d.v_descale_heads;
  p.scale = d.scale, p.k_descale = d.k_descale, p.v_descale = d.v_descale;
  p.status = d.status ? d.status : dev.status;
  if (p.max_new == 1 && !d.mask) return launch_tree(d, p, dev, s);
  if (d.dtype == ATTN_F16)
    return d.D == 64 ? launch_tree_hidden<__half, 64>(d, p, dev, s) : launch_tree_hidden<__half, 128>(d, p, dev, s);
  return d.D == 64 ? launch_tree_hidden<__nv_bfloat16, 64>(d, p, dev, s)
                   : launch_tree_hidden<__nv_bfloat16, 128>(d, p, dev, s);
}

template <typename Desc>
int call(const Desc* desc, void* stream) {
  if (!desc) return fail(ATTN_ERR_INVALID, "null descriptor");
  const int rc = check(*desc);
  return rc != ATTN_OK ? rc : run(*desc, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

int attn_cache_plan(const AttnCachePlan* desc, void* stream) { return call(desc, stream); }
int attn_cache_append(const AttnCacheAppend* desc, void* stream) { return call(desc, stream); }
int attn_rotary(const AttnRotary* desc, void* stream) { return call(desc, stream); }
int attn_tree_fwd(const AttnTree* desc, void* stream) { return call(desc, stream); }

}  // extern "C"
