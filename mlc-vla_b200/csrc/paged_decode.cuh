// Attention of one query token per request over the 8-bit page cache.
#pragma once

#include "paged_common.cuh"

namespace pi0 {
namespace paged {

struct DecodeArgs {
  const void* q;       // [batch, heads, head_dim]
  void* out;
  int64_t q_tok, q_head, o_tok, o_head;
  Cache cache;
  const int* table;    // [batch, max_pages]
  int64_t table_stride;
  const int* kv_lens;
  int* err;
  float c;             // logit scale · log2 e
  int batch, heads, max_pages;
};

template <typename T>
struct PagedKV {
  const Cache* c;
  const int* table;
  int head;
  __device__ __forceinline__ int64_t ph(int j) const {
    return (int64_t)table[j / c->page_size] * c->kv_heads + head;
  }
  __device__ __forceinline__ void k8(int j, int d, float (&x)[8]) const {
    const int64_t p = ph(j);
    load8(c->k + (p * c->page_size + j % c->page_size) * c->head_dim + d, c->ks[p], x);
  }
  __device__ __forceinline__ void v8(int j, int d, float (&x)[8]) const {
    const int64_t p = ph(j);
    load8(c->v + (p * c->page_size + j % c->page_size) * c->head_dim + d, c->vs[p], x);
  }
};

// Cached tokens of request b that can be read: its length, held to its table row and to the pages
// before the first number that names no page of the pool. Uniform over the warp.
__device__ __forceinline__ int readable_len(const DecodeArgs& a, int b) {
  const int lane = threadIdx.x & 31, ps = a.cache.page_size;
  int n = a.kv_lens[b];
  if (n < 0 || n > (int64_t)a.max_pages * ps) {
    if (lane == 0) set_err(a.err, PI0_PAGED_ERR_TABLE);
    n = n < 0 ? 0 : a.max_pages * ps;
  }
  const int* row = a.table + b * a.table_stride;
  const int pages = (n + ps - 1) / ps;
  for (int p = 0; p < pages; p += 32) {
    const bool bad = p + lane < pages && (unsigned)row[p + lane] >= (unsigned)a.cache.num_pages;
    const unsigned any = __ballot_sync(~0u, bad);
    if (any) {
      if (lane == 0) set_err(a.err, PI0_PAGED_ERR_PAGE);
      return (p + __ffs(any) - 1) * ps;
    }
  }
  return n;
}

// One warp per (request, head), for the head sizes without a tensor-core form.
template <typename T>
__global__ void __launch_bounds__(32) paged_rows_kernel(DecodeArgs a) {
  const int b = blockIdx.y, h = blockIdx.x;
  const int n = readable_len(a, b);
  const PagedKV<T> kv{&a.cache, a.table + b * a.table_stride, h / (a.heads / a.cache.kv_heads)};
  attend_row(reinterpret_cast<const T*>(a.q) + b * a.q_tok + h * a.q_head, a.cache.head_dim, n, a.c,
             kv, reinterpret_cast<T*>(a.out) + b * a.o_tok + h * a.o_head);
}

}  // namespace paged
}  // namespace pi0
