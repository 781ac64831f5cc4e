// Python binding of the text-generation operators: the checks of their arguments, the outputs,
// workspaces and error flags, and the calls of the C entry points of include/pi0b200.h. A decode
// step makes these calls once per layer and token; from Python the checks alone took 11 us a call,
// longer than the kernels.
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <vector>

#include "pi0b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// the library's entry points (this module is not linked against it: the package opens it by path)
struct Entries {
  decltype(&pi0_build_slots) build_slots = nullptr;
  decltype(&pi0_write_kv) write_kv = nullptr;
  decltype(&pi0_attention_prompt) attention_prompt = nullptr;
  decltype(&pi0_attention_paged) attention_paged = nullptr;
  decltype(&pi0_attention_prompt_workspace) attention_prompt_workspace = nullptr;
  decltype(&pi0_attention_paged_workspace) attention_paged_workspace = nullptr;
} g_lib;

void bind(uint64_t build_slots, uint64_t write_kv, uint64_t attention_prompt,
          uint64_t attention_paged, uint64_t attention_prompt_workspace,
          uint64_t attention_paged_workspace) {
  g_lib.build_slots = reinterpret_cast<decltype(g_lib.build_slots)>(build_slots);
  g_lib.write_kv = reinterpret_cast<decltype(g_lib.write_kv)>(write_kv);
  g_lib.attention_prompt = reinterpret_cast<decltype(g_lib.attention_prompt)>(attention_prompt);
  g_lib.attention_paged = reinterpret_cast<decltype(g_lib.attention_paged)>(attention_paged);
  g_lib.attention_prompt_workspace =
      reinterpret_cast<decltype(g_lib.attention_prompt_workspace)>(attention_prompt_workspace);
  g_lib.attention_paged_workspace =
      reinterpret_cast<decltype(g_lib.attention_paged_workspace)>(attention_paged_workspace);
}

// a nonzero status, for the Python side to raise
struct Status : std::exception {
  int code;
  const char* name;
  Status(int c, const char* n) : code(c), name(n) {}
};

void check_status(int rc, const char* name) {
  if (rc) throw Status(rc, name);
}

// Never freed: a static destructor would run after CUDA is gone.
std::mutex g_mutex;
auto& g_flags = *new std::map<int, Tensor>;

bool capturing(cudaStream_t stream) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &s));
  return s != cudaStreamCaptureStatusNone;
}

// the error flag of a device, for calls without one of their own
const Tensor& flag_of(int device) {
  std::lock_guard<std::mutex> lock(g_mutex);
  auto it = g_flags.find(device);
  if (it == g_flags.end()) {
    TORCH_CHECK(!capturing(c10::cuda::getCurrentCUDAStream(device).stream()),
                "the device's error flag does not exist yet: make one call before the capture, or "
                "give `err`");
    Tensor t = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
    C10_CUDA_CHECK(cudaDeviceSynchronize());  // zero before any stream's kernel may write it
    it = g_flags.emplace(device, std::move(t)).first;
  }
  return it->second;
}

OptTensor flag(int device) {
  std::lock_guard<std::mutex> lock(g_mutex);
  auto it = g_flags.find(device);
  return it == g_flags.end() ? OptTensor() : OptTensor(it->second);
}

// Room for the partial sums of one call, from the stream's pool and back to it.
Tensor workspace(int device, int64_t bytes) {
  return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
}

int dtype_code(const Tensor& t, const char* name) {
  const auto type = t.scalar_type();
  TORCH_CHECK_VALUE(t.is_cuda() && (type == at::kHalf || type == at::kBFloat16), name,
                    " must be a float16 or bfloat16 CUDA tensor");
  return type == at::kHalf ? PI0_F16 : PI0_BF16;
}

void check_head_dim(int64_t d) {
  TORCH_CHECK_VALUE(d >= 8 && d % 8 == 0 && d <= 256, "head_dim must be a multiple of 8 up to 256, "
                    "not ", d);
}

bool on(const Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

// int32 array of n numbers (n < 0: any), or of n rows
int32_t* ints(const Tensor& t, const char* name, int device, int dim, int64_t n = -1) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && on(t, device) && t.dim() == dim, name,
                    " must be a ", dim, "-dimensional int32 tensor on cuda:", device);
  TORCH_CHECK_VALUE(n < 0 || t.size(0) == n, name, " must hold ", n, " numbers, not ", t.size(0));
  TORCH_CHECK_VALUE((t.size(dim - 1) < 2 || t.stride(dim - 1) == 1) &&
                        (dim < 2 || t.size(0) < 2 || t.stride(0) >= t.size(1)),
                    name, " must be contiguous along its last dimension and not expanded");
  return static_cast<int32_t*>(t.data_ptr());
}

// [tokens, heads, head_dim] in 16 bits, read in 16-byte vectors along the last dimension
struct Rows {
  void* p;
  int64_t tok, head;
};

Rows rows(const Tensor& t, const char* name, int device, at::ScalarType type) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && on(t, device), name, " must be a ", type,
                    " tensor on cuda:", device);
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be [tokens, heads, head_dim]");
  // a stride that no second token or head uses is free: take a valid one
  Rows r{t.data_ptr(), t.size(0) < 2 ? t.size(1) * t.size(2) : t.stride(0),
         t.size(1) < 2 ? t.size(2) : t.stride(1)};
  TORCH_CHECK_VALUE(t.numel() == 0 || (t.stride(2) == 1 && r.tok > 0 && r.head > 0 &&
                                       r.tok % 8 == 0 && r.head % 8 == 0 &&
                                       reinterpret_cast<uintptr_t>(r.p) % 16 == 0),
                    name, " must be contiguous along its last dimension, with token and head "
                    "strides that are multiples of 8 elements (not expanded) and a 16-byte aligned "
                    "start");
  return r;
}

void check_shape(const Tensor& t, const char* name, at::IntArrayRef want) {
  TORCH_CHECK_VALUE(t.sizes() == want, name, " must have the shape ", want, ", not ", t.sizes());
}

pi0_kv8 cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int device) {
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes(),
                    "cache codes must be [pages, kv heads, page, head_dim], alike for k and v");
  check_head_dim(k.size(3));
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat8_e4m3fn && on(*t, device) &&
                          t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                      "cache codes must be contiguous, 16-byte aligned float8_e4m3fn tensors on "
                      "cuda:", device);
  for (const Tensor* t : {&ks, &vs})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && on(*t, device) && t->is_contiguous() &&
                          t->sizes() == k.sizes().slice(0, 2),
                      "cache scales must be contiguous float32 [pages, kv heads] tensors on cuda:",
                      device);
  TORCH_CHECK_VALUE(k.size(0) > 0 && k.size(0) * k.size(2) < (int64_t(1) << 31),
                    "a cache holds at least one page and fewer than 2^31 tokens");
  return pi0_kv8{k.data_ptr(), v.data_ptr(), static_cast<float*>(ks.data_ptr()),
                 static_cast<float*>(vs.data_ptr()), (int32_t)k.size(0), (int32_t)k.size(2),
                 (int32_t)k.size(1), (int32_t)k.size(3)};
}

int fits32(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n >= 0 && n < (int64_t(1) << 31), name, " must be in [0, 2^31), not ", n);
  return (int)n;
}

int* err_of(const OptTensor& err, int device) {
  if (err) return ints(*err, "err", device, 1, 1);
  return static_cast<int*>(flag_of(device).data_ptr());
}

// The attentions have no backward pass. A result of inputs that ask for gradients says so when one is
// asked of it, rather than being a constant without a word.
bool wants_grad(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->requires_grad()) return true;
  return false;
}

void no_grad_out(const OptTensor& out, bool wanted) {
  TORCH_CHECK(!(out && (wanted || wants_grad({&*out}))),
              "out= does not support gradients: call under torch.no_grad()");
}

void no_backward(Tensor& o, const char* name, std::initializer_list<const Tensor*> inputs) {
  torch::autograd::edge_list edges;
  for (const Tensor* t : inputs)
    if (t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
  auto node = std::shared_ptr<torch::autograd::NotImplemented>(
      new torch::autograd::NotImplemented(name, std::move(edges)), torch::autograd::deleteNode);
  torch::autograd::set_history(o, node);
}

// n elements of a one-dimensional tensor from `first` on, without the dispatcher's way around
Tensor part_of(const Tensor& t, int64_t first, int64_t n) {
  Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(),
                                                      t.dtype());
  v.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  v.unsafeGetTensorImpl()->set_storage_offset(first);
  return v;
}

std::vector<Tensor> build_slots(const Tensor& kv_lens, const Tensor& new_lens,
                                const Tensor& block_table, const Tensor& free_pages,
                                const Tensor& free_pos, int64_t page_size, int64_t num_tokens,
                                std::optional<int64_t> num_pages, const OptTensor& err) {
  TORCH_CHECK_VALUE(block_table.is_cuda(), "block_table must be a CUDA tensor");
  const int dev = block_table.get_device();
  int32_t* table = ints(block_table, "block_table", dev, 2);
  const int64_t batch = block_table.size(0), columns = block_table.size(1);
  const int32_t* kv = ints(kv_lens, "kv_lens", dev, 1, batch);
  const int32_t* nw = ints(new_lens, "new_lens", dev, 1, batch);
  const int32_t* pos = ints(free_pos, "free_pos", dev, 1, 1);
  const int32_t* pages = ints(free_pages, "free_pages", dev, 1);
  TORCH_CHECK_VALUE(page_size > 0 && num_tokens >= 0 && columns > 0,
                    "page_size and the block table's columns must be positive, num_tokens not "
                    "negative");
  const int64_t pool = num_pages ? *num_pages : (int64_t(0x7fffffff)) / page_size;
  TORCH_CHECK_VALUE(pool > 0 && pool < (int64_t(1) << 31) / page_size + 1 &&
                        pool * page_size < (int64_t(1) << 31),
                    "num_pages * page_size must be below 2^31");
  TORCH_CHECK_VALUE(batch <= 16384, "at most 16384 requests");
  fits32(num_tokens, "num_tokens");
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev) guard.set_index(dev);
  at::AutoDispatchBelowAutograd below;
  // one allocation for the five results
  const Tensor buf = at::empty({2 * batch + 2 + 2 * num_tokens}, block_table.options());
  std::vector<Tensor> out{part_of(buf, 0, batch + 1), part_of(buf, batch + 1, num_tokens),
                          part_of(buf, batch + 1 + num_tokens, num_tokens),
                          part_of(buf, batch + 1 + 2 * num_tokens, batch),
                          part_of(buf, 2 * batch + 1 + 2 * num_tokens, 1)};
  int32_t* p = static_cast<int32_t*>(buf.data_ptr());
  check_status(g_lib.build_slots((int)batch, kv, nw, table,
                                 batch < 2 ? columns : block_table.stride(0), (int)columns, pages,
                                 fits32(free_pages.size(0), "free_pages"), pos, (int)pool,
                                 (int)page_size, (int)num_tokens, p, p + batch + 1,
                                 p + batch + 1 + num_tokens, p + batch + 1 + 2 * num_tokens,
                                 p + 2 * batch + 1 + 2 * num_tokens, err_of(err, dev),
                                 c10::cuda::getCurrentCUDAStream(dev).stream()),
               "pi0_build_slots");
  return out;
}

void write_kv(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs,
              const Tensor& k, const Tensor& v, const Tensor& cu_seqlens, const Tensor& kv_lens,
              const Tensor& slot_mapping, std::optional<int64_t> max_new, const OptTensor& err) {
  const int code = dtype_code(k, "k");
  const int dev = k.get_device();
  const pi0_kv8 c = cache_of(ck, cv, cks, cvs, dev);
  const Rows kr = rows(k, "k", dev, k.scalar_type()), vr = rows(v, "v", dev, k.scalar_type());
  const int tokens = fits32(k.size(0), "tokens");
  check_shape(k, "k", {tokens, c.kv_heads, c.head_dim});
  check_shape(v, "v", {tokens, c.kv_heads, c.head_dim});
  const int32_t* lens = ints(kv_lens, "kv_lens", dev, 1);
  const int64_t batch = kv_lens.size(0);
  const int32_t* cu = ints(cu_seqlens, "cu_seqlens", dev, 1, batch + 1);
  const int32_t* slots = ints(slot_mapping, "slot_mapping", dev, 1, tokens);
  const int most = max_new ? fits32(*max_new, "max_new") : tokens;
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev) guard.set_index(dev);
  check_status(g_lib.write_kv(code, kr.p, kr.tok, kr.head, vr.p, vr.tok, vr.head, tokens,
                              fits32(batch, "kv_lens"), cu, lens, slots, most, &c, err_of(err, dev),
                              c10::cuda::getCurrentCUDAStream(dev).stream()),
               "pi0_write_kv");
}

Tensor attention_prompt(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q,
                        const OptTensor& cu_k, const OptTensor& prefix, std::optional<double> scale,
                        const OptTensor& out, const OptTensor& err) {
  const int code = dtype_code(q, "q");
  const int dev = q.get_device();
  const auto type = q.scalar_type();
  const Rows qr = rows(q, "q", dev, type), kr = rows(k, "k", dev, type), vr = rows(v, "v", dev, type);
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = k.size(1);
  check_head_dim(dim);
  TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && k.size(2) == dim, heads,
                    " query heads of ", dim, " cannot share ", kv_heads, " kv heads of ", k.size(2));
  check_shape(v, "v", k.sizes());
  const int32_t* cq = ints(cu_q, "cu_seqlens_q", dev, 1);
  const int64_t batch = cu_q.size(0) - 1;
  TORCH_CHECK_VALUE(batch > 0 || (batch == 0 && tokens == 0),
                    "cu_seqlens_q must hold one number more than there are requests");
  const int32_t* ck = cu_k ? ints(*cu_k, "cu_seqlens_k", dev, 1, batch + 1) : cq;
  const int32_t* pre = prefix ? ints(*prefix, "prefix_lens", dev, 1, batch) : nullptr;
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev) guard.set_index(dev);
  at::AutoDispatchBelowAutograd below;
  const bool grad = wants_grad({&q, &k, &v});
  no_grad_out(out, grad);
  Tensor o = out ? *out : at::empty(q.sizes(), q.options());
  const Rows orr = rows(o, "out", dev, type);
  check_shape(o, "out", q.sizes());
  if (out && tokens > 0)
    for (const Tensor* t : {&q, &k, &v}) {
      const auto s = at::get_overlap_status(o, *t);
      TORCH_CHECK_VALUE((t->numel() == 0 || o.data_ptr() != t->data_ptr()) &&
                            s != at::MemOverlapStatus::Full && s != at::MemOverlapStatus::Partial,
                        "out may not overlap q, k or v");
    }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const int64_t bytes = g_lib.attention_prompt_workspace(fits32(heads, "heads"), (int)kv_heads, (int)dim);
  if (bytes < 0) throw Status(PI0_ERR_CUDA, "pi0_attention_prompt_workspace");
  const Tensor ws = workspace(dev, bytes);
  check_status(g_lib.attention_prompt(code, qr.p, qr.tok, qr.head, kr.p, kr.tok, kr.head, vr.p,
                                      vr.tok, vr.head, fits32(tokens, "tokens"),
                                      fits32(k.size(0), "keys"), fits32(heads, "heads"),
                                      (int)kv_heads, (int)dim, fits32(batch, "requests"), cq, ck, pre,
                                      scale ? (float)*scale : 1.f / std::sqrt((float)dim), orr.p,
                                      orr.tok, orr.head, ws.data_ptr(), ws.numel(),
                                      err_of(err, dev), stream),
               "pi0_attention_prompt");
  if (grad) no_backward(o, "attention_prompt", {&q, &k, &v});
  return o;
}

Tensor attention_paged(const Tensor& q, const Tensor& ck, const Tensor& cv, const Tensor& cks,
                       const Tensor& cvs, const Tensor& block_table, const Tensor& kv_lens,
                       std::optional<double> scale, const OptTensor& out, const OptTensor& err) {
  const int code = dtype_code(q, "q");
  const int dev = q.get_device();
  const pi0_kv8 c = cache_of(ck, cv, cks, cvs, dev);
  const Rows qr = rows(q, "q", dev, q.scalar_type());
  const int64_t batch = q.size(0), heads = q.size(1);
  TORCH_CHECK_VALUE(q.size(2) == c.head_dim && heads > 0 && c.kv_heads > 0 && heads % c.kv_heads == 0,
                    "q ", q.sizes(), " does not fit a cache of ", c.kv_heads, " kv heads of ",
                    c.head_dim);
  const int32_t* table = ints(block_table, "block_table", dev, 2, batch);
  const int32_t* lens = ints(kv_lens, "kv_lens", dev, 1, batch);
  const int64_t columns = block_table.size(1);
  TORCH_CHECK_VALUE(columns > 0, "block_table must have a column");
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev) guard.set_index(dev);
  at::AutoDispatchBelowAutograd below;
  const bool grad = wants_grad({&q, &cks, &cvs});
  no_grad_out(out, grad);
  Tensor o = out ? *out : at::empty(q.sizes(), q.options());
  const Rows orr = rows(o, "out", dev, q.scalar_type());
  check_shape(o, "out", q.sizes());
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const int64_t bytes = g_lib.attention_paged_workspace(fits32(heads, "heads"), c.kv_heads,
                                                        c.head_dim, c.page_size);
  if (bytes < 0) throw Status(PI0_ERR_CUDA, "pi0_attention_paged_workspace");
  const Tensor ws = workspace(dev, bytes);
  check_status(g_lib.attention_paged(code, qr.p, qr.tok, qr.head, fits32(batch, "requests"),
                                     (int)heads, &c, table,
                                     batch < 2 ? columns : block_table.stride(0),
                                     fits32(columns, "columns"), lens,
                                     scale ? (float)*scale : 1.f / std::sqrt((float)c.head_dim),
                                     orr.p, orr.tok, orr.head, ws.data_ptr(), ws.numel(),
                                     err_of(err, dev), stream),
               "pi0_attention_paged");
  if (grad) no_backward(o, "attention_paged", {&q, &cks, &cvs});
  return o;
}

}  // namespace

PYBIND11_MODULE(_paged_native, m) {
  static PyObject* status = nullptr;
  m.def("bind", &bind);
  m.def("flag", &flag);
  // the exception class of a nonzero status, called with (code, entry point)
  m.def("raise_status_with", [](py::object cls) { status = cls.release().ptr(); });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Status& s) {
      py::object e = py::reinterpret_borrow<py::object>(status)(s.code, s.name);
      PyErr_SetObject(status, e.ptr());
    }
  });
  m.def("build_slots", &build_slots);
  m.def("write_kv", &write_kv);
  m.def("attention_prompt", &attention_prompt);
  m.def("attention_paged", &attention_paged);
}
