// Attention over packed prompts: grouped heads, causal with a bidirectional prefix per request.
//
// Query i of a request with Lq new tokens and Lk keys sees the keys j < n(i),
// n(i) = min(Lk, max(i + Lk − Lq + 1, prefix)): always a leading part of the request's keys.
#pragma once

#include "paged_common.cuh"

namespace pi0 {
namespace paged {

struct PromptArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides, elements
  const int* cu_q;
  const int* cu_k;
  const int* prefix;   // or null: causal
  int* err;
  float c;             // logit scale · log2 e
  int batch, total_q, total_k, heads, kv_heads, head_dim;
};

// first token and length of request r, inside [0, total)
__device__ __forceinline__ void seq_span(const int* cu, int r, int total, int& t0, int& n) {
  t0 = min(max(cu[r], 0), total);
  n = min(max(cu[r + 1], t0), total) - t0;
}

// keys that query i of a request sees
__device__ __forceinline__ int visible(int i, int lq, int lk, int prefix) {
  return max(0, min(lk, max(i + lk - lq + 1, prefix)));
}

template <typename T>
struct PromptKV {
  const T* k;
  const T* v;
  int64_t k_tok, v_tok;
  __device__ __forceinline__ void k8(int j, int d, float (&x)[8]) const {
    load8(k + (int64_t)j * k_tok + d, x);
  }
  __device__ __forceinline__ void v8(int j, int d, float (&x)[8]) const {
    load8(v + (int64_t)j * v_tok + d, x);
  }
};

constexpr int kRowWarps = 4;

// One warp per (token, head), for the head sizes without a tensor-core form.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) prompt_rows_kernel(PromptArgs a) {
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int t = (int)(row / a.heads), h = (int)(row % a.heads);
  if (t >= a.total_q) return;
  T* out = reinterpret_cast<T*>(a.out) + t * a.o_tok + h * a.o_head;
  // the last request that starts at or before t
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  int q0, lq, k0, lk;
  seq_span(a.cu_q, lo, a.total_q, q0, lq);
  seq_span(a.cu_k, lo, a.total_k, k0, lk);
  const int i = t - q0;
  // a token outside of every request (padding of the packed batch) gives zeros
  const int n = i >= 0 && i < lq ? visible(i, lq, lk, a.prefix ? a.prefix[lo] : 0) : 0;
  const int g = h / (a.heads / a.kv_heads);
  const PromptKV<T> kv{reinterpret_cast<const T*>(a.k) + k0 * a.k_tok + g * a.k_head,
                       reinterpret_cast<const T*>(a.v) + k0 * a.v_tok + g * a.v_head, a.k_tok,
                       a.v_tok};
  attend_row(reinterpret_cast<const T*>(a.q) + t * a.q_tok + h * a.q_head, a.head_dim, n, a.c, kv,
             out);
}

}  // namespace paged
}  // namespace pi0
