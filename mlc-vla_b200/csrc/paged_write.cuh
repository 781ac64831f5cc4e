// New keys and values into the 8-bit page cache.
//
// The scale of a (page, kv head) is the smallest power of two s ≥ 2^-64 with max|x| ≤ 448·s over
// the page's tokens (e4m3 reaches 448), and a code is e4m3(x / s): dividing by a power of two is
// exact, so the only rounding is e4m3's, to nearest even. Tokens that join a page which holds some
// already keep or raise its scale; when it rises, the codes there are rounded once more, to the
// new step (exact for every code that stays above e4m3's subnormals). An infinity or a NaN has no
// finite code: it is stored as NaN and does not count for the scale.
//
// Bound by HBM: 2 bytes read and 1 written per element, plus the scales.
#pragma once

#include "paged_common.cuh"

namespace pi0 {
namespace paged {

constexpr int kWriteThreads = 128;

struct WriteArgs {
  const void* x[2];          // keys, values: [tokens, kv heads, head_dim], last dimension contiguous
  int64_t tok_stride[2], head_stride[2];
  const int* cu;
  const int* kv_lens;        // tokens cached before the new ones
  const int* slots;
  int* err;
  Cache cache;
  int tokens;
};

// smallest power of two s ≥ 2^-64 with amax ≤ 448·s: amax = f·2^e with f in [1, 2), 448 = 1.75·2^8
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127;
  const int x = (b & 0x7fffff) <= 0x600000 ? e - 8 : e - 7;
  return __uint_as_float((uint32_t)(max(x, -64) + 127) << 23);
}

__device__ __forceinline__ uint16_t to_e4m3x2(float a, float b) {
  if (isinf(a)) a = NAN;
  if (isinf(b)) b = NAN;
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// One block per (page that the request's new tokens touch, kv head, key or value).
template <typename T>
__global__ void __launch_bounds__(kWriteThreads) write_kv_kernel(WriteArgs a) {
  const int r = blockIdx.z, h = blockIdx.y >> 1, kind = blockIdx.y & 1;
  const Cache& c = a.cache;
  const int ps = c.page_size, hd = c.head_dim, vec = hd / 8;
  const int tid = threadIdx.x;
  __shared__ float s_max[kWriteThreads / 32];
  const int start = max(a.kv_lens[r], 0);
  const int t0 = min(max(a.cu[r], 0), a.tokens), t1 = min(max(a.cu[r + 1], t0), a.tokens);
  if (t1 == t0) return;
  const int64_t end = (int64_t)start + (t1 - t0);
  const int p0 = start / ps, pages = (int)((end - 1) / ps) - p0 + 1;
  const T* x = reinterpret_cast<const T*>(a.x[kind]) + h * a.head_stride[kind];
  for (int j = blockIdx.x; j < pages; j += gridDim.x) {
    const int64_t lo = max((int64_t)start, (int64_t)(p0 + j) * ps);
    const int64_t hi = min(end, (int64_t)(p0 + j + 1) * ps);
    const int tok = t0 + (int)(lo - start), row = (int)(lo % ps), n = (int)(hi - lo);
    const int slot = a.slots[tok];
    if (slot < 0) continue;  // not admitted to the pool
    const int page = slot / ps;
    if (page >= c.num_pages || slot % ps != row) {
      if (tid == 0) set_err(a.err, PI0_PAGED_ERR_PAGE);
      continue;
    }
    float am = 0.f;
    for (int i = tid; i < n * vec; i += kWriteThreads) {
      float v[8];
      load8(x + (int64_t)(tok + i / vec) * a.tok_stride[kind] + (i % vec) * 8, v);
#pragma unroll
      for (int u = 0; u < 8; ++u) am = fmaxf(am, isfinite(v[u]) ? fabsf(v[u]) : 0.f);
    }
    am = warp_max(am);
    __syncthreads();  // s_max of the page before has been read
    if ((tid & 31) == 0) s_max[tid >> 5] = am;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWriteThreads / 32; ++w) am = fmaxf(am, s_max[w]);
    const int64_t ph = (int64_t)page * c.kv_heads + h;
    float* sp = (kind ? c.vs : c.ks) + ph;
    uint8_t* codes = (kind ? c.v : c.k) + ph * ps * hd;
    float s = pow2_scale(am);
    if (row > 0) {
      const float old = *sp;
      if (old >= s) {
        s = old;
      } else {
        const float ratio = old / s;
        for (int i = tid; i < row * vec; i += kWriteThreads) {
          float v[8];
          load8(codes + (int64_t)i * 8, ratio, v);
          uint16_t o[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) o[u] = to_e4m3x2(v[2 * u], v[2 * u + 1]);
          *reinterpret_cast<uint2*>(codes + (int64_t)i * 8) = *reinterpret_cast<uint2*>(o);
        }
      }
    }
    const float inv = 1.f / s;
    for (int i = tid; i < n * vec; i += kWriteThreads) {
      float v[8];
      load8(x + (int64_t)(tok + i / vec) * a.tok_stride[kind] + (i % vec) * 8, v);
      __align__(8) uint16_t o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = to_e4m3x2(v[2 * u] * inv, v[2 * u + 1] * inv);
      *reinterpret_cast<uint2*>(codes + (int64_t)row * hd + (int64_t)i * 8) =
          *reinterpret_cast<uint2*>(o);
    }
    __syncthreads();  // every thread has read the old scale
    if (tid == 0) *sp = s;
  }
}

}  // namespace paged
}  // namespace pi0
