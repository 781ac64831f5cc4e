// Shared parts of the text-generation operators: the error codes their kernels record, the layout
// of the 8-bit page cache, and attention of one query row by one warp.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "pi0b200.h"

namespace pi0 {
namespace paged {

// the first code wins, as with the bounded waits
__device__ __forceinline__ void set_err(int* err, int code) {
  if (err) atomicCAS(err, 0, code);
}

// Key/value pages of one attention layer: e4m3 codes [pages, kv heads, page, head_dim], one fp32
// scale per (page, kv head). Rows are counted over the whole pool, (page·KV + head)·page_size + row,
// in 64 bits: a pool may hold more than 2^32 bytes.
struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int num_pages, page_size, kv_heads, head_dim;
};

// 8 consecutive 16-bit values as floats
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Tr<T>::f(e[i]);
}

__device__ __forceinline__ float e4m3_f(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// 8 consecutive e4m3 codes as floats, times the scale of their page
__device__ __forceinline__ void load8(const uint8_t* p, float scale, float (&x)[8]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const uint8_t* e = reinterpret_cast<const uint8_t*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = e4m3_f(e[i]) * scale;
}

// o = Σ_j softmax_j(c·q·k_j) v_j over the keys j < n of one row, by one warp: lane l holds the
// elements [8l, 8l + 8) of q and of the sum, the running maximum and sum are fp32, exponentials in
// base 2 (c includes log2 e). No key that the row does not see is read, so whatever lies there
// (NaN, infinities, unwritten pages) cannot reach the result. n = 0 gives zeros. A row whose
// logits are all −inf, or that meets a NaN, gives NaN, as the formula does.
template <typename T, class Load>
__device__ __forceinline__ void attend_row(const T* q, int hd, int n, float c, const Load& kv,
                                           T* out) {
  const int lane = threadIdx.x & 31;
  const bool on = lane * 8 < hd;
  float qv[8] = {}, acc[8] = {};
  if (on) load8(q + lane * 8, qv);
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < n; ++j) {
    float x[8] = {}, s = 0.f;
    if (on) kv.k8(j, lane * 8, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(qv[i], x[i], s);
    s = warp_sum(s) * c;
    const float mn = fmaxf(m, s);
    const float ref = mn == -INFINITY ? 0.f : mn;  // while every logit is −inf, their weight is 0
    const float a = exp2f(m - ref), p = exp2f(s - ref);
    m = mn;
    l = l * a + p;
    if (on) kv.v8(j, lane * 8, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(p, x[i], acc[i] * a);
  }
  if (on) {
    const float inv = n > 0 ? 1.f / l : 0.f;
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Tr<T>::pack(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    *reinterpret_cast<uint4*>(out + lane * 8) = o;
  }
}

}  // namespace paged
}  // namespace pi0
