// New keys and values into the 8-bit page cache.
//
// The scale of a (page, kv head) is the smallest power of two s ≥ 2^-64 with max|x| ≤ 448·s over
// the page's tokens (e4m3 reaches 448), and a code is e4m3(x / s): dividing by a power of two is
// exact, so the only rounding is e4m3's, to nearest even. Tokens that join a page which holds some
// already keep or raise its scale; when it rises, the codes there are rounded once more, to the
// new step (exact for every code that stays above e4m3's subnormals). An infinity or a NaN has no
// finite code: it is stored as NaN and does not count for the scale. Neither does a token that is
// left out: one without a slot, or whose slot is not its row of the page that the first token with
// a slot of its own row names.
//
// Bound by HBM: 2 bytes read and 1 written per element, plus the scales. A (page, kv head) is held in
// the registers of the few warps that take it, up to 16 vectors of 16 bytes a lane: one pass over the
// data, whose loads are all in flight before the first is used, and no wait but one between those
// warps. Larger pages are read twice. Measured: 32771 tokens of 8 heads of 128 in pages of 32, 39.0 us
// (5166 GB/s, 79 % of the measured copy rate); 16 vectors a lane in two blocks per SM, against 53 us
// with 8 in three and 62 us with 4 in four: what counts is the bytes in flight. 256 single tokens
// 4.7 us, bound by latency. The launch has blocks for every request's longest: one prompt of 8192
// beside 256 single tokens takes 595 us for 8 us of bytes, so such batches are better written apart.
#pragma once

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace pi0 {
namespace paged {

constexpr int kWriteWarps = 8;

struct WriteArgs {
  const void* x[2];          // keys, values: [tokens, kv heads, head_dim], last dimension contiguous
  int64_t tok_stride[2], head_stride[2];
  const int* cu;
  const int* kv_lens;        // tokens cached before the new ones
  const int* slots;
  int* err;
  Cache cache;
  int tokens;
  int warps;                 // per (page, kv head, key or value): 1, 2, 4 or 8
};

// smallest power of two s ≥ 2^-64 with amax ≤ 448·s: amax = f·2^e with f in [1, 2), 448 = 1.75·2^8
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127;
  const int x = (b & 0x7fffff) <= 0x600000 ? e - 8 : e - 7;
  return __uint_as_float((uint32_t)(max(x, -64) + 127) << 23);
}

// codes of eight values times `inv`
__device__ __forceinline__ uint2 to_e4m3x8(const float (&v)[8], float inv) {
  const uint64_t inv2 = pack2(inv, inv);
  __align__(8) uint16_t o[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    o[u] = __nv_cvt_float2_to_fp8x2(unpack2(mul2(pack2(v[2 * u], v[2 * u + 1]), inv2)),
                                    __NV_SATFINITE, __NV_E4M3);
  return *reinterpret_cast<uint2*>(o);
}

template <typename T>
__device__ __forceinline__ void unpack8(uint4 u, float (&x)[8]) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Tr<T>::f(e[i]);
}

// Largest magnitudes of two 16-bit floats at a time; a NaN stays. Without a sign they order like their
// bits, so lanes compare them as whole numbers: from the type's infinity up they are no numbers.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (Tr<T>::kBf16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, uint4 v) {
  const uint32_t a = max2<T>(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
  const uint32_t b = max2<T>(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
  return max2<T>(m, max2<T>(a, b));
}
// the same, of the numbers only
template <typename T>
__device__ __forceinline__ uint32_t max_bits_finite(uint32_t m, uint4 v, uint32_t inf) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    m = max2<T>(m, (lo < inf ? lo : 0u) | (hi < inf ? hi << 16 : 0u));
  }
  return m;
}

// VECS: vectors a lane holds
template <typename T, int VECS>
__global__ void __launch_bounds__(32 * kWriteWarps, VECS > 4 ? 2 : 4) write_kv_kernel(WriteArgs a) {
  constexpr uint32_t kInf = Tr<T>::kBf16 ? 0x7f80u : 0x7c00u;
  const Cache& c = a.cache;
  const int ps = c.page_size, hd = c.head_dim, vec = hd / 8, kinds = 2 * c.kv_heads;
  const int lanes = 32 * a.warps, units = kWriteWarps / a.warps;  // of a unit, of a block
  const int unit = threadIdx.x / lanes, g = threadIdx.x % lanes;
  __shared__ uint32_t s_max[3][kWriteWarps];
  const int r = blockIdx.z;
  const int start = max(a.kv_lens[r], 0);
  const int t0 = min(max(a.cu[r], 0), a.tokens), t1 = min(max(a.cu[r + 1], t0), a.tokens);
  if (t1 == t0) return;
  const int64_t end = (int64_t)start + (t1 - t0);
  const int p0 = start / ps, pages = (int)((end - 1) / ps) - p0 + 1;
  // the warps of a unit meet at a barrier of their own
  auto meet = [&]() {
    if (a.warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + unit), "r"(lanes) : "memory");
  };
  auto most = [&](uint32_t m, int slot) -> uint32_t {
    m = __reduce_max_sync(~0u, m);
    if (a.warps > 1) {
      if ((threadIdx.x & 31) == 0) s_max[slot][threadIdx.x >> 5] = m;
      meet();
      for (int w = 0; w < a.warps; ++w) m = max(m, s_max[slot][unit * a.warps + w]);
    }
    return m;
  };

  // unit x of the request: page x / kinds, and head and kind x % kinds. Neighbours share tokens.
  for (int64_t x = (int64_t)blockIdx.x * units + unit; x < (int64_t)pages * kinds;
       x += (int64_t)gridDim.x * units) {
    const int j = (int)(x / kinds), h = (int)(x % kinds) >> 1, kind = (int)(x % kinds) & 1;
    const int64_t lo = max((int64_t)start, (int64_t)(p0 + j) * ps);
    const int64_t hi = min(end, (int64_t)(p0 + j + 1) * ps);
    const int tok = t0 + (int)(lo - start), row = (int)(lo % ps), n = (int)(hi - lo);
    const T* src = reinterpret_cast<const T*>(a.x[kind]) + tok * a.tok_stride[kind] +
                   h * a.head_stride[kind];
    // vector i of this lane is vector v = g + i·lanes of the unit, at (token, column) = (t, d)
    const int nv = n * vec, dt = lanes / vec, dd = lanes % vec;
    const int64_t tok_stride = a.tok_stride[kind];
    auto at = [&](int v) { return src + (v / vec) * tok_stride + (v % vec) * 8; };
    const int* slots = a.slots + tok;
    int slot0 = slots[0];  // of the run's first token
    const int mine = g < n ? slots[g] : slot0 + g;
    uint4 held[VECS];
    {
      int d = g % vec;
      const T* p = at(g);
      const int64_t step = dt * tok_stride + dd * 8, wrap = tok_stride - vec * 8;
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        held[i] = g + i * lanes < nv ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
        p += step;
        d += dd;
        if (d >= vec) {
          d -= vec;
          p += wrap;
        }
      }
    }
    // Every token at its row of one page, which is the first's: looked at while the vectors are on
    // their way. If not, the unit takes the path of infinities, which looks at each token.
    const int pool = c.num_pages * ps;
    bool odd = (unsigned)slot0 >= (unsigned)pool || slot0 % ps != row || mine != slot0 + g;
    float* scales = kind ? c.vs : c.ks;
    auto scale_at = [&]() { return scales + (int64_t)(slot0 / ps) * c.kv_heads + h; };
    float old = row > 0 && !odd ? *scale_at() : 0.f;
    for (int i = g + lanes; i < n; i += lanes) odd |= slots[i] != slot0 + i;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VECS; ++i) m = max_bits<T>(m, held[i]);
#pragma unroll 1
    for (int v = g + VECS * lanes; v < nv; v += lanes)
      m = max_bits<T>(m, *reinterpret_cast<const uint4*>(at(v)));
    m = most(max(m & 0xffffu, m >> 16) | (odd ? 0x10000u : 0u), 0);
    odd = m >= kInf;
    if (odd) {
      uint32_t left = 0;  // n − i for the first token i whose slot is its row of a page
#pragma unroll 1
      for (int i = g; i < n; i += lanes)
        if ((unsigned)slots[i] < (unsigned)pool && slots[i] % ps == row + i)
          left = max(left, (uint32_t)(n - i));
      left = most(left, 1);
      slot0 = left ? slots[n - left] - (int)(n - left) : -1;
#pragma unroll 1
      for (int i = g; i < n; i += lanes)
        if (slots[i] >= 0 && (!left || slots[i] != slot0 + i)) set_err(a.err, PI0_PAGED_ERR_PAGE);
      m = 0;
#pragma unroll 1
      for (int v = g; v < nv; v += lanes)
        if (left && slots[v / vec] == slot0 + v / vec)
          m = max_bits_finite<T>(m, *reinterpret_cast<const uint4*>(at(v)), kInf);
      m = most(max(m & 0xffffu, m >> 16), 2);
      if (!left) {  // the same for all lanes of the unit
        meet();     // they have read s_max
        continue;
      }
      if (row > 0) old = *scale_at();
    }
    float* sp = scale_at();
    uint8_t* codes = (kind ? c.v : c.k) + (sp - scales) * ps * hd;
    const uint16_t bits = (uint16_t)m;
    float s = pow2_scale(Tr<T>::f(*reinterpret_cast<const T*>(&bits)));
    if (row > 0) {
      if (old >= s) {
        s = old;
      } else {
        const float ratio = old / s;
        for (int i = g; i < row * vec; i += lanes) {
          float v[8];
          load8(codes + (int64_t)i * 8, 1.f, v);
          *reinterpret_cast<uint2*>(codes + (int64_t)i * 8) = to_e4m3x8(v, ratio);
        }
      }
    }
    const float inv = 1.f / s;
    uint8_t* dst = codes + (int64_t)row * hd;
    const int rest = odd ? 0 : VECS;  // first vector of a lane that is read (again)
    if (!odd) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int v = g + i * lanes;
        if (v < nv) {
          float f[8];
          unpack8<T>(held[i], f);
          *reinterpret_cast<uint2*>(dst + v * 8) = to_e4m3x8(f, inv);
        }
      }
    }
#pragma unroll 1
    for (int v = g + rest * lanes; v < nv; v += lanes) {
      if (odd && slots[v / vec] != slot0 + v / vec) continue;
      float f[8];
      load8(at(v), f);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (isinf(f[u])) f[u] = NAN;  // it has no code
      *reinterpret_cast<uint2*>(dst + v * 8) = to_e4m3x8(f, inv);
    }
    meet();  // every lane has read the old scale, and s_max
    if (g == 0) *sp = s;
  }
}

}  // namespace paged
}  // namespace pi0
