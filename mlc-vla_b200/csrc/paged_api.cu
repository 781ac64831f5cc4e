// The text-generation operators of include/pi0b200.h: block tables and slot maps, the 8-bit page
// cache, attention over packed prompts and attention of single tokens over the cache. Context-free,
// like pi0_embed_language: every buffer is the caller's, every call is asynchronous on the stream.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "pi0b200.h"
#include "paged_slots.cuh"
#include "paged_write.cuh"
#include "paged_prompt.cuh"
#include "paged_decode.cuh"

using namespace pi0;
using namespace pi0::paged;

namespace {

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
bool dtype_ok(int dtype) { return dtype == PI0_F16 || dtype == PI0_BF16; }
int launched() { return cudaGetLastError() == cudaSuccess ? PI0_OK : PI0_ERR_CUDA; }

// n int32 numbers from p on
struct Ints {
  const int32_t* p;
  int64_t n;
  bool meets(const Ints& o) const { return n > 0 && o.n > 0 && p < o.p + o.n && o.p < p + n; }
};

// one 16-bit operand [tokens, heads, head_dim]: 16-byte vectors along the last dimension
bool rows_ok(const void* p, int64_t tok, int64_t head) {
  return p && !off16(p) && tok > 0 && head > 0 && tok % 8 == 0 && head % 8 == 0;
}

// whether two operands [tokens, heads, head_dim] surely share elements: they begin at the same one, or
// both are contiguous and their ranges meet (others may lie between one another's rows)
struct Operand {
  const void* p;
  int64_t tokens, heads, head_dim, tok, head;
  bool dense() const { return tok == heads * head_dim && head == head_dim; }
  bool meets(const Operand& o) const {
    if (tokens == 0 || o.tokens == 0) return false;
    if (p == o.p) return true;
    const auto *x = static_cast<const uint16_t*>(p), *y = static_cast<const uint16_t*>(o.p);
    return dense() && o.dense() && x < y + o.tokens * o.tok && y < x + tokens * tok;
  }
};

bool cache_ok(const pi0_kv8* c) {
  return c && c->k && c->v && c->k_scale && c->v_scale && !off16(c->k) && !off16(c->v) &&
         c->num_pages >= 1 && c->page_size >= 1 && c->kv_heads >= 1 && c->head_dim >= 8 &&
         c->head_dim % 8 == 0 && c->head_dim <= 256 &&
         (int64_t)c->num_pages * c->page_size <= INT_MAX;
}

Cache cache_of(const pi0_kv8* c) {
  return Cache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale,
               c->num_pages, c->page_size, c->kv_heads, c->head_dim};
}

constexpr int kMaxDevices = 64;

// SMs of the current device (0: the runtime failed)
int sm_count(int* device) {
  static std::atomic<int> known[kMaxDevices];
  if (cudaGetDevice(device) != cudaSuccess || *device < 0 || *device >= kMaxDevices) return 0;
  int n = known[*device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device) != cudaSuccess) return 0;
    known[*device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// lets kernel F use `bytes` of dynamic shared memory, once per device
template <auto F>
bool allow_smem(int device, int bytes) {
  static std::atomic<bool> done[kMaxDevices];
  if (done[device].load(std::memory_order_relaxed)) return true;
  if (cudaFuncSetAttribute(F, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return false;
  done[device].store(true, std::memory_order_relaxed);
  return true;
}

// ---- TMA tensor maps (driver entry point fetched through the runtime, no libcuda link) ------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn f = known.load(std::memory_order_acquire);
  if (f) return f;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess)
    return nullptr;
  f = reinterpret_cast<EncodeTiledFn>(fn);
  known.store(f, std::memory_order_release);
  return f;
}

// Map of `rank` dimensions, innermost first; strides in bytes of the dimensions behind it. Out of
// bounds reads as zero. Swizzled over `span` bytes, the width of a box.
template <int RANK>
int make_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, const cuuint64_t (&dims)[RANK],
             const cuuint64_t (&strides)[RANK - 1], const cuuint32_t (&box)[RANK], int span) {
  const EncodeTiledFn f = encode_fn();
  if (!f) return PI0_ERR_CUDA;
  cuuint32_t ones[RANK];
  for (auto& o : ones) o = 1;
  const CUresult r = f(m, type, RANK, const_cast<void*>(base), dims, strides, box, ones,
                       CU_TENSOR_MAP_INTERLEAVE_NONE,
                       span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PI0_OK : PI0_ERR_CUDA;
}

// ---- attention over prompts -----------------------------------------------------------------

template <typename T, int HD>
int run_prompt(const PromptArgs& a, int device, int sms, cudaStream_t st) {
  using C = PromptCfg<HD>;
  constexpr CUtensorMapDataType type =
      Tr<T>::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // a tile's 128 rows are the group's heads of as many tokens as fit
  const int group = a.heads / a.kv_heads, tok = 128 / group;
  auto map = [&](CUtensorMap* m, const void* p, int heads, int total, int64_t head_stride,
                 int64_t token_stride, int box_heads, int box_tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)heads, (cuuint64_t)total};
    const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    return make_map<3>(m, type, p, dims, strides, box, 128);
  };
  CUtensorMap tq, tk, tv;
  int rc = map(&tq, a.q, a.heads, a.total_q, a.q_head, a.q_tok, group, tok);
  if (!rc) rc = map(&tk, a.k, a.kv_heads, a.total_k, a.k_head, a.k_tok, 1, kKeys);
  if (!rc) rc = map(&tv, a.v, a.kv_heads, a.total_k, a.v_head, a.v_tok, 1, C::VKEYS);
  if (rc) return rc;
  if (!allow_smem<prompt_tc_kernel<T, HD>>(device, C::SMEM)) return PI0_ERR_CUDA;
  // Steps at most: every request has at most one tile of queries that is not full, and no tile has
  // more tiles of keys than there are.
  const int64_t tiles = (int64_t)a.total_q / (C::NQ * tok) + a.batch;
  const int64_t most = tiles * a.kv_heads * ((a.total_k + kKeys - 1) / kKeys);
  const int ctas = (int)std::min<int64_t>(sms, most);
  prompt_tc_kernel<T, HD><<<ctas, C::THREADS, C::SMEM, st>>>(tq, tk, tv, a, tok);
  if (cudaGetLastError() != cudaSuccess) return PI0_ERR_CUDA;
  if (a.total_k <= kKeys) return PI0_OK;  // a tile has one step: none is split
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, C::NQ * (HD / 32));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prompt_join_kernel<T, HD>, a, tok, ctas) == cudaSuccess
             ? PI0_OK : PI0_ERR_CUDA;
}

template <int HD>
int64_t prompt_ws(int sms) {
  return (int64_t)sms * (16 + 2 * PromptCfg<HD>::PARTIAL * (int64_t)sizeof(float));
}

bool prompt_tc(int heads, int kv_heads, int head_dim) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && heads / kv_heads <= 128;
}

template <typename T>
int run_prompt_any(const PromptArgs& a, int device, int sms, cudaStream_t st) {
  switch (a.head_dim) {
    case 64: return run_prompt<T, 64>(a, device, sms, st);
    case 128: return run_prompt<T, 128>(a, device, sms, st);
    default: return run_prompt<T, 256>(a, device, sms, st);
  }
}

// ---- attention over the cache ---------------------------------------------------------------

// Whether the tensor-core form takes these sizes: a head fills whole swizzle rows, a page divides a
// tile of 128 keys into boxes of whole 8-row groups or is made of whole tiles.
bool paged_tc(int head_dim, int page_size, int64_t planes) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
         (page_size % 128 == 0 || (page_size % 8 == 0 && 128 % page_size == 0)) && planes <= INT_MAX;
}

// Heads of a unit's columns: the softmax does its work for all of them, so groups of up to 4 and up
// to 8 have their own; wider groups go 16 at a time.
int paged_heads(int heads, int kv_heads) {
  const int group = heads / kv_heads;
  return group <= 4 ? 4 : group <= 8 ? 8 : 16;
}

template <int HD, int NH>
int64_t paged_ws(int sms) {
  using C = DecCfg<HD, NH>;
  return (int64_t)sms * C::OCC * (16 + 2 * C::PARTIAL * (int64_t)sizeof(float));
}

template <typename T, int HD, int NH>
int run_paged(const DecodeArgs& a, int device, int sms, cudaStream_t st) {
  using C = DecCfg<HD, NH>;
  const Cache& c = a.cache;
  CUtensorMap tk, tv;
  const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)c.page_size,
                              (cuuint64_t)c.num_pages * c.kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)HD, (cuuint64_t)HD * c.page_size};
  const cuuint32_t box[3] = {(cuuint32_t)C::ROW, (cuuint32_t)std::min(c.page_size, kDecTile), 1};
  int rc = make_map<3>(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.k, dims, strides, box, C::ROW);
  if (!rc) rc = make_map<3>(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.v, dims, strides, box, C::ROW);
  if (rc) return rc;
  if (!allow_smem<paged_decode_kernel<T, HD, NH>>(device, C::SMEM)) return PI0_ERR_CUDA;
  const int group = a.heads / c.kv_heads;
  const int64_t most = (int64_t)a.batch * c.kv_heads * ((group + NH - 1) / NH) *
                       (((int64_t)a.max_pages * c.page_size + kDecTile - 1) / kDecTile);
  if (most > INT_MAX) return PI0_ERR_UNSUPPORTED;
  const int ctas = (int)std::min<int64_t>((int64_t)sms * C::OCC, most);
  paged_decode_kernel<T, HD, NH><<<ctas, kDecThreads, C::SMEM, st>>>(tk, tv, a);
  if (cudaGetLastError() != cudaSuccess) return PI0_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, std::min(NH, group));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, HD, NH>, a, ctas) == cudaSuccess
             ? PI0_OK : PI0_ERR_CUDA;
}

template <typename T>
int run_paged_any(const DecodeArgs& a, int device, int sms, cudaStream_t st) {
  const int nh = paged_heads(a.heads, a.cache.kv_heads);
  auto run = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    return nh == 4   ? run_paged<T, HD, 4>(a, device, sms, st)
           : nh == 8 ? run_paged<T, HD, 8>(a, device, sms, st)
                     : run_paged<T, HD, 16>(a, device, sms, st);
  };
  switch (a.cache.head_dim) {
    case 64: return run(std::integral_constant<int, 64>());
    case 128: return run(std::integral_constant<int, 128>());
    default: return run(std::integral_constant<int, 256>());
  }
}

}  // namespace

extern "C" {

int pi0_build_slots(int batch, const int32_t* kv_lens, const int32_t* new_lens,
                    int32_t* block_table, int64_t table_stride, int max_pages,
                    const int32_t* free_pages, int n_free, const int32_t* free_pos, int num_pages,
                    int page_size, int num_tokens, int32_t* cu_seqlens, int32_t* positions,
                    int32_t* slot_mapping, int32_t* kv_lens_out, int32_t* free_pos_out, int* err,
                    pi0_stream_t stream) {
  if (batch < 0 || max_pages < 1 || table_stride < max_pages || n_free < 0 || num_pages < 1 ||
      page_size < 1 || num_tokens < 0 || (int64_t)num_pages * page_size > INT_MAX)
    return PI0_ERR_INVALID;
  if (!free_pos || !cu_seqlens || !free_pos_out || (n_free && !free_pages) ||
      (batch && (!kv_lens || !new_lens || !block_table || !kv_lens_out)) ||
      (num_tokens && (!positions || !slot_mapping)))
    return PI0_ERR_INVALID;
  if (batch > kSlotMaxBatch) return PI0_ERR_UNSUPPORTED;
  // Blocks read the inputs at any time while others write the outputs.
  const Ints in[] = {{kv_lens, batch}, {new_lens, batch}, {free_pages, n_free}, {free_pos, 1}};
  const Ints out[] = {{cu_seqlens, (int64_t)batch + 1}, {positions, num_tokens},
                      {slot_mapping, num_tokens}, {kv_lens_out, batch}, {free_pos_out, 1}};
  for (const Ints& o : out) {
    for (const Ints& i : in)
      if (o.meets(i)) return PI0_ERR_INVALID;
    for (const Ints& x : out)
      if (&x != &o && o.meets(x)) return PI0_ERR_INVALID;
  }
  int device;
  const int sms = sm_count(&device);
  if (!sms) return PI0_ERR_CUDA;
  const auto smem = [](int n) { return (int)(2 * sizeof(int)) * (n + 1); };
  // the limit of the largest batch, once: a limit per call could be lowered between another host
  // thread's limit and launch
  if (!allow_smem<build_slots_kernel>(device, smem(kSlotMaxBatch))) return PI0_ERR_CUDA;
  SlotArgs a{kv_lens, new_lens, block_table, table_stride, free_pages, free_pos, cu_seqlens,
             positions, slot_mapping, kv_lens_out, free_pos_out, err, batch, max_pages, n_free,
             num_pages, page_size, num_tokens};
  // two tokens a thread until one block per SM is reached
  const int grid = std::max(1, std::min(sms, (int)((num_tokens + 2 * kSlotThreads - INT64_C(1)) /
                                                   (2 * kSlotThreads))));
  build_slots_kernel<<<grid, kSlotThreads, smem(batch), stream>>>(a);
  return launched();
}

int pi0_write_kv(int dtype, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                 const void* v, int64_t v_token_stride, int64_t v_head_stride, int num_tokens,
                 int batch, const int32_t* cu_seqlens, const int32_t* kv_lens,
                 const int32_t* slot_mapping, int max_new, const pi0_kv8* cache, int* err,
                 pi0_stream_t stream) {
  if (!dtype_ok(dtype) || num_tokens < 0 || batch < 0 || max_new < 0 || !cache_ok(cache))
    return PI0_ERR_INVALID;
  if (num_tokens == 0 || batch == 0) return PI0_OK;
  max_new = std::max(1, std::min(max_new, num_tokens));  // a size of the launch, whatever it says
  if (!rows_ok(k, k_token_stride, k_head_stride) || !rows_ok(v, v_token_stride, v_head_stride) ||
      !cu_seqlens || !kv_lens || !slot_mapping)
    return PI0_ERR_INVALID;
  if (batch > 65535 || cache->kv_heads > 32767) return PI0_ERR_UNSUPPORTED;
  // as many vectors a lane, then as many warps, as hold a (page, kv head) in registers
  const int64_t vecs = (int64_t)std::min(cache->page_size, max_new) *
                       (cache->head_dim / 8);
  const int held = vecs <= 32 ? 1 : vecs <= 128 ? 4 : 16;
  int warps = 1;
  while (warps < kWriteWarps && vecs > (int64_t)warps * 32 * held) warps *= 2;
  WriteArgs a{{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride},
              cu_seqlens, kv_lens, slot_mapping, err, cache_of(cache), num_tokens, warps};
  // n tokens touch at most ⌈(n − 1)/page⌉ + 1 pages; a request with more than max_new loops
  const int64_t pages = (max_new + (int64_t)cache->page_size - 2) / cache->page_size + 1;
  const int units = kWriteWarps / warps;
  const int64_t blocks = (pages * 2 * cache->kv_heads + units - 1) / units;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, INT_MAX), 1, batch);
  const int threads = 32 * kWriteWarps;
  auto go = [&](auto kernel) { kernel<<<grid, threads, 0, stream>>>(a); };
  const bool half = dtype == PI0_F16;
  if (held == 1) go(half ? write_kv_kernel<__half, 1> : write_kv_kernel<__nv_bfloat16, 1>);
  else if (held == 4) go(half ? write_kv_kernel<__half, 4> : write_kv_kernel<__nv_bfloat16, 4>);
  else go(half ? write_kv_kernel<__half, 16> : write_kv_kernel<__nv_bfloat16, 16>);
  return launched();
}

int64_t pi0_attention_prompt_workspace(int heads, int kv_heads, int head_dim) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads) return -1;
  if (!prompt_tc(heads, kv_heads, head_dim)) return 0;
  int device;
  const int sms = sm_count(&device);
  if (!sms) return -1;
  return head_dim == 64 ? prompt_ws<64>(sms) : head_dim == 128 ? prompt_ws<128>(sms)
                                                               : prompt_ws<256>(sms);
}

int pi0_attention_prompt(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                         const void* k, int64_t k_token_stride, int64_t k_head_stride,
                         const void* v, int64_t v_token_stride, int64_t v_head_stride,
                         int total_q, int total_k, int heads, int kv_heads, int head_dim,
                         int batch, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                         const int32_t* prefix_lens, float scale, void* out,
                         int64_t o_token_stride, int64_t o_head_stride, void* workspace,
                         int64_t workspace_bytes, int* err, pi0_stream_t stream) {
  if (!dtype_ok(dtype) || total_q < 0 || total_k < 0 || heads < 1 || kv_heads < 1 ||
      heads % kv_heads || head_dim < 8 || head_dim % 8 || head_dim > 256 || batch < 0)
    return PI0_ERR_INVALID;
  if (total_q == 0) return PI0_OK;
  if (batch == 0 || !cu_seqlens_q || !cu_seqlens_k || !rows_ok(q, q_token_stride, q_head_stride) ||
      !rows_ok(out, o_token_stride, o_head_stride) ||
      (total_k && (!rows_ok(k, k_token_stride, k_head_stride) ||
                   !rows_ok(v, v_token_stride, v_head_stride))))
    return PI0_ERR_INVALID;
  const int64_t rows = (int64_t)total_q * heads;
  if (rows > INT_MAX) return PI0_ERR_UNSUPPORTED;
  // queries, keys and values are read again after rows have been written
  const Operand o{out, total_q, heads, head_dim, o_token_stride, o_head_stride};
  if (o.meets({q, total_q, heads, head_dim, q_token_stride, q_head_stride}) ||
      o.meets({k, total_k, kv_heads, head_dim, k_token_stride, k_head_stride}) ||
      o.meets({v, total_k, kv_heads, head_dim, v_token_stride, v_head_stride}))
    return PI0_ERR_INVALID;
  PromptArgs a{q, k, v, out, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
               v_token_stride, v_head_stride, o_token_stride, o_head_stride, cu_seqlens_q,
               cu_seqlens_k, prefix_lens, err, static_cast<float*>(workspace),
               scale * 1.4426950408889634f, batch, total_q, total_k,
               heads, kv_heads, head_dim};
  // The tensor-core form takes the largest product for the largest logit; a scale that turns the order
  // round, or levels it, is not worth a step's time (3 % when the sign was looked at there).
  if (prompt_tc(heads, kv_heads, head_dim) && total_k > 0 && a.c > 0.f) {
    int device;
    const int sms = sm_count(&device);
    if (!sms) return PI0_ERR_CUDA;
    if (!workspace || off16(workspace) || !err ||
        workspace_bytes < pi0_attention_prompt_workspace(heads, kv_heads, head_dim))
      return PI0_ERR_INVALID;
    return dtype == PI0_F16 ? run_prompt_any<__half>(a, device, sms, stream)
                            : run_prompt_any<__nv_bfloat16>(a, device, sms, stream);
  }
  const unsigned grid = (unsigned)((rows + kRowWarps - 1) / kRowWarps);
  if (dtype == PI0_F16) prompt_rows_kernel<__half><<<grid, 32 * kRowWarps, 0, stream>>>(a);
  else prompt_rows_kernel<__nv_bfloat16><<<grid, 32 * kRowWarps, 0, stream>>>(a);
  return launched();
}

int64_t pi0_attention_paged_workspace(int heads, int kv_heads, int head_dim, int page_size) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || page_size < 1) return -1;
  if (!paged_tc(head_dim, page_size, 1)) return 0;
  int device;
  const int sms = sm_count(&device);
  if (!sms) return -1;
  const int nh = paged_heads(heads, kv_heads);
  auto bytes = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    return nh == 4 ? paged_ws<HD, 4>(sms) : nh == 8 ? paged_ws<HD, 8>(sms) : paged_ws<HD, 16>(sms);
  };
  switch (head_dim) {
    case 64: return bytes(std::integral_constant<int, 64>());
    case 128: return bytes(std::integral_constant<int, 128>());
    default: return bytes(std::integral_constant<int, 256>());
  }
}

int pi0_attention_paged(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                        int batch, int heads, const pi0_kv8* cache, const int32_t* block_table,
                        int64_t table_stride, int max_pages, const int32_t* kv_lens, float scale,
                        void* out, int64_t o_token_stride, int64_t o_head_stride, void* workspace,
                        int64_t workspace_bytes, int* err, pi0_stream_t stream) {
  if (!dtype_ok(dtype) || batch < 0 || heads < 1 || !cache_ok(cache) || heads % cache->kv_heads ||
      max_pages < 1 || table_stride < max_pages)
    return PI0_ERR_INVALID;
  if (batch == 0) return PI0_OK;
  if (!rows_ok(q, q_token_stride, q_head_stride) || !rows_ok(out, o_token_stride, o_head_stride) ||
      !block_table || !kv_lens)
    return PI0_ERR_INVALID;
  if (batch > 65535) return PI0_ERR_UNSUPPORTED;
  DecodeArgs a{q, out, q_token_stride, q_head_stride, o_token_stride, o_head_stride,
               cache_of(cache), block_table, table_stride, kv_lens, err,
               static_cast<float*>(workspace), scale * 1.4426950408889634f, batch, heads, max_pages};
  if (paged_tc(cache->head_dim, cache->page_size, (int64_t)cache->num_pages * cache->kv_heads)) {
    const int64_t need = pi0_attention_paged_workspace(heads, cache->kv_heads, cache->head_dim,
                                                       cache->page_size);
    if (need < 0) return PI0_ERR_CUDA;
    if (!workspace || off16(workspace) || workspace_bytes < need || !err) return PI0_ERR_INVALID;
    int device;
    const int sms = sm_count(&device);
    return dtype == PI0_F16 ? run_paged_any<__half>(a, device, sms, stream)
                            : run_paged_any<__nv_bfloat16>(a, device, sms, stream);
  }
  const dim3 grid(heads, batch);
  if (dtype == PI0_F16) paged_rows_kernel<__half><<<grid, 32, 0, stream>>>(a);
  else paged_rows_kernel<__nv_bfloat16><<<grid, 32, 0, stream>>>(a);
  return launched();
}

}  // extern "C"
