"""Text generation in packed batches over a key/value cache of 8-bit pages.

Four operators, for a prefix expert that answers in text (prompts of different lengths, then one
token per request and step):

* ``build_slots``: block tables, positions and slots of the new tokens, on the GPU, from lengths;
* ``write_kv``: new keys and values into the pages, e4m3 codes with a power-of-two scale for each
  page and kv head;
* ``attention_prompt``: attention of packed prompts, grouped heads, causal with an optional
  bidirectional prefix per request;
* ``attention_paged``: attention of one token per request over the pages.

Every call is asynchronous on the current stream of its tensors' device. What only the device can
see (a negative length, an exhausted pool, a page number outside the pool) is recorded in `err`, a
device int32 tensor of one element, or, where none is given, in a flag of the device that
``check()`` reads, clears and raises.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Dict, NamedTuple, Optional

import torch

from mlc_vla import _lib

_DTYPE = {torch.float16: _lib.PI0_F16, torch.bfloat16: _lib.PI0_BF16}

PAGED_ERRORS = {
    1: "a bounded wait in a kernel gave up", 2: "a bounded wait in a kernel gave up",
    3: "a bounded wait in a kernel gave up",
    16: "a length below zero, or more new tokens than num_tokens",
    17: "a request longer than its row of the block table",
    18: "no free page left for a request",
    19: "a page number outside the pool, or a slot that is not its token's",
}


class KVCache8(NamedTuple):
    """Pages of one attention layer: e4m3 codes [pages, kv heads, page, head_dim] and fp32 scales
    [pages, kv heads], for keys and values."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def empty(num_pages: int, page_size: int, kv_heads: int, head_dim: int,
              device="cuda") -> "KVCache8":
        shape = (num_pages, kv_heads, page_size, head_dim)
        codes = [torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        scales = [torch.empty(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return KVCache8(*codes, *scales)


class Slots(NamedTuple):
    """What ``build_slots`` makes for a packed batch of new tokens."""

    cu_seqlens: torch.Tensor    # [batch + 1] int32
    positions: torch.Tensor     # [num_tokens] int32
    slot_mapping: torch.Tensor  # [num_tokens] int32, -1 where a token has no place
    kv_lens: torch.Tensor       # [batch] int32, the new tokens included
    free_pos: torch.Tensor      # [1] int32


_flags: Dict[int, torch.Tensor] = {}


def _flag(device: torch.device) -> torch.Tensor:
    f = _flags.get(device.index)
    if f is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the device's error flag does not exist yet: make one call before "
                               "the capture, or give `err`")
        f = _flags[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.synchronize(device)  # zero before any stream's kernel may write it
    return f


def check(device="cuda") -> None:
    """Wait for the device, and raise what the calls without an `err` of their own recorded."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    f = _flags.get(index)
    if f is None:
        return
    torch.cuda.synchronize(index)
    code = int(f.item())
    if code:
        f.zero_()
        raise _lib.Pi0Error(code, PAGED_ERRORS.get(code, "a kernel reported an error"))


def _err_ptr(err: Optional[torch.Tensor], device: torch.device) -> int:
    if err is None:
        return _flag(device).data_ptr()
    _ints(err, "err", device, 1, 1)
    return err.data_ptr()


# The checks below run on every call of a decode step, so they ask a tensor for each of its
# properties once.

def _ints(t: torch.Tensor, name: str, device: torch.device, dim: int,
          n: Optional[int] = None) -> None:
    shape = t.shape
    if t.dtype is not torch.int32 or t.device != device or len(shape) != dim:
        raise ValueError(f"{name} must be a {dim}-dimensional int32 tensor on {device}")
    if n is not None and shape[0] != n:
        raise ValueError(f"{name} must hold {n} numbers, not {shape[0]}")
    if not t.is_contiguous():
        stride = t.stride()
        if (shape[-1] > 1 and stride[-1] != 1) or (
                dim == 2 and shape[0] > 1 and stride[0] < shape[1]):
            raise ValueError(f"{name} must be contiguous along its last dimension and not expanded")


def _rows(t: torch.Tensor, name: str, device: torch.device, dtype, shape=None):
    """[tokens, heads, head_dim] in 16 bits, read in 16-byte vectors along the last dimension:
    its start, token stride and head stride."""
    if t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    have = t.shape
    if len(have) != 3 or (shape is not None and have != shape):
        raise ValueError(f"{name} must be [tokens, heads, head_dim]"
                         + (f" = {tuple(shape)}, not {tuple(have)}" if shape is not None else ""))
    tokens, heads, dim = have
    tok, head, last = t.stride()
    # a stride that no second token or head uses is free: take a valid one
    if tokens < 2:
        tok = heads * dim
    if heads < 2:
        head = dim
    ptr = t.data_ptr()
    if (last != 1 or ptr & 15 or tok & 7 or head & 7 or not tok or not head) and t.numel():
        raise ValueError(f"{name} must be contiguous along its last dimension, with token and "
                         f"head strides that are multiples of 8 elements (not expanded) and a "
                         f"16-byte aligned start")
    return ptr, tok, head


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPE.get(t.dtype)
    if code is None or not t.is_cuda:
        raise ValueError(f"{name} must be a float16 or bfloat16 CUDA tensor")
    return code


def _head_dim(d: int) -> None:
    if d < 8 or d % 8 or d > 256:
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, not {d}")


def _cache(c: KVCache8, device: torch.device) -> _lib.Pi0Kv8C:
    k, v, k_scale, v_scale = c
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("cache codes must be [pages, kv heads, page, head_dim], alike for k and v")
    pages, heads, page, dim = shape
    _head_dim(dim)
    kp, vp = k.data_ptr(), v.data_ptr()
    if not (k.dtype is v.dtype is torch.float8_e4m3fn and k.device == device and v.device == device
            and k.is_contiguous() and v.is_contiguous()) or (kp | vp) & 15:
        raise ValueError(f"cache codes must be contiguous, 16-byte aligned float8_e4m3fn tensors "
                         f"on {device}")
    planes = shape[:2]
    if not (k_scale.dtype is v_scale.dtype is torch.float32 and k_scale.device == device
            and v_scale.device == device and k_scale.shape == planes and v_scale.shape == planes
            and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError(f"cache scales must be contiguous float32 [pages, kv heads] tensors on "
                         f"{device}")
    return _lib.Pi0Kv8C(kp, vp, k_scale.data_ptr(), v_scale.data_ptr(), pages, page, heads, dim)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # absent without CUDA


def _call(name: str, device: torch.device, *args) -> None:
    f = getattr(_lib._lib or _lib.load(), name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, None, name)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(device: torch.device, heads: int, kv_heads: int, dim: int, page: int) -> int:
    with torch.cuda.device(device):
        n = _lib.load().pi0_attention_paged_workspace(heads, kv_heads, dim, page)
    if n < 0:
        raise _lib.Pi0Error(_lib.PI0_ERR_CUDA, "pi0_attention_paged_workspace")
    return n


_workspaces: Dict[tuple, torch.Tensor] = {}


def _workspace(device: torch.device, heads: int, kv_heads: int, dim: int, page: int) -> torch.Tensor:
    """Room for the partial sums of one call. Calls on one stream follow each other, so a stream's
    calls share a buffer; a captured graph may be replayed on any stream and has its own."""
    n = _workspace_bytes(device, heads, kv_heads, dim, page)
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(n, dtype=torch.uint8, device=device)
    key = (device.index, _raw_stream(device.index))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < n:
        ws = _workspaces[key] = torch.empty(n, dtype=torch.uint8, device=device)
    return ws


def build_slots(kv_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                free_pages: torch.Tensor, free_pos: torch.Tensor, page_size: int, num_tokens: int,
                num_pages: Optional[int] = None, err: Optional[torch.Tensor] = None) -> Slots:
    """Places for ``new_lens[r]`` tokens behind the ``kv_lens[r]`` cached ones of each request.

    New pages are taken from ``free_pages[free_pos:]`` in the order of the requests and written
    into ``block_table`` [batch, max_pages] in place, behind the pages a request holds already.
    ``num_tokens``: rows of the packed batch (rows behind the last request's get slot -1).
    ``num_pages``: pages of the pool (default: no bound but that of the slots' 31 bits). A request
    that its table row or the pool cannot hold is not admitted (slots -1, length unchanged) and an
    error is recorded."""
    dev = block_table.device
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor")
    _ints(block_table, "block_table", dev, 2)
    batch, max_pages = block_table.shape
    _ints(kv_lens, "kv_lens", dev, 1, batch)
    _ints(new_lens, "new_lens", dev, 1, batch)
    _ints(free_pos, "free_pos", dev, 1, 1)
    _ints(free_pages, "free_pages", dev, 1)
    if page_size < 1 or num_tokens < 0 or max_pages < 1:
        raise ValueError("page_size and the block table's columns must be positive, num_tokens "
                         "not negative")
    if num_pages is None:
        num_pages = (2 ** 31 - 1) // page_size
    if num_pages < 1 or num_pages * page_size >= 2 ** 31:
        raise ValueError("num_pages * page_size must be below 2^31")
    if batch > 16384:
        raise ValueError("at most 16384 requests")
    # one allocation for the five results
    sizes = (batch + 1, num_tokens, num_tokens, batch, 1)
    buf = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
    out = Slots(*buf.split_with_sizes(sizes))
    cu = buf.data_ptr()
    pos = cu + 4 * (batch + 1)
    slots = pos + 4 * num_tokens
    lens = slots + 4 * num_tokens
    _call("pi0_build_slots", dev, batch, kv_lens.data_ptr(), new_lens.data_ptr(),
          block_table.data_ptr(), max(block_table.stride(0), max_pages), max_pages,
          free_pages.data_ptr(), free_pages.shape[0], free_pos.data_ptr(), num_pages, page_size,
          num_tokens, cu, pos, slots, lens, lens + 4 * batch, _err_ptr(err, dev))
    return out


def write_kv(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
             kv_lens: torch.Tensor, slot_mapping: torch.Tensor, max_new: Optional[int] = None,
             err: Optional[torch.Tensor] = None) -> None:
    """Keys and values [tokens, kv heads, head_dim] into the pages of ``cache`` at
    ``slot_mapping``. ``cu_seqlens`` [batch + 1]: the requests' tokens; ``kv_lens`` [batch]: their
    tokens cached before these. ``max_new``: the most new tokens of one request, which sizes the
    launch (default: all of them)."""
    code = _dtype(k, "k")
    dev = k.device
    c = _cache(cache, dev)
    tokens, batch = k.shape[0], kv_lens.shape[0]
    shape = torch.Size((tokens, c.kv_heads, c.head_dim))
    _ints(kv_lens, "kv_lens", dev, 1)
    _ints(cu_seqlens, "cu_seqlens", dev, 1, batch + 1)
    _ints(slot_mapping, "slot_mapping", dev, 1, tokens)
    if max_new is not None and max_new < 0:
        raise ValueError("max_new must not be negative")
    _call("pi0_write_kv", dev, code, *_rows(k, "k", dev, k.dtype, shape),
          *_rows(v, "v", dev, k.dtype, shape), tokens, batch, cu_seqlens.data_ptr(),
          kv_lens.data_ptr(), slot_mapping.data_ptr(), tokens if max_new is None else max_new,
          ctypes.byref(c), _err_ptr(err, dev))


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     cu_seqlens_q: torch.Tensor, cu_seqlens_k: Optional[torch.Tensor] = None,
                     prefix_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None,
                     err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed prompts: q [tokens, heads, head_dim], k and v [keys, kv heads,
    head_dim]. Request r has the queries ``cu_seqlens_q[r]:cu_seqlens_q[r + 1]`` and the keys
    ``cu_seqlens_k[r]:cu_seqlens_k[r + 1]`` (default: the same), the last query at the last key.
    Query i of Lq sees key j of Lk if ``j <= i + Lk - Lq`` or ``j < prefix_lens[r]`` (default 0:
    causal; Lk: every key). ``scale``: of the logits, 1/sqrt(head_dim) by default. A query that
    sees no key gives zeros."""
    code = _dtype(q, "q")
    dev = q.device
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [tokens, heads, head_dim]")
    dtype, (tokens, heads, dim), (keys, kv_heads, k_dim) = q.dtype, q.shape, k.shape
    _head_dim(dim)
    if kv_heads < 1 or heads % kv_heads or k_dim != dim:
        raise ValueError(f"{heads} query heads of {dim} cannot share {kv_heads} kv heads of {k_dim}")
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    batch = cu_seqlens_q.shape[0] - 1
    if batch < 0 or (batch == 0 and tokens):
        raise ValueError("cu_seqlens_q must hold one number more than there are requests")
    _ints(cu_seqlens_q, "cu_seqlens_q", dev, 1)
    _ints(cu_seqlens_k, "cu_seqlens_k", dev, 1, batch + 1)
    if prefix_lens is not None:
        _ints(prefix_lens, "prefix_lens", dev, 1, batch)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _call("pi0_attention_prompt", dev, code, *_rows(q, "q", dev, dtype), *_rows(k, "k", dev, dtype),
          *_rows(v, "v", dev, dtype, k.shape), tokens, keys, heads, kv_heads, dim, batch,
          cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
          None if prefix_lens is None else prefix_lens.data_ptr(),
          dim ** -0.5 if scale is None else scale, *_rows(out, "out", dev, dtype, q.shape),
          _err_ptr(err, dev))
    return out


def attention_paged(q: torch.Tensor, cache: KVCache8, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None,
                    err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per request, q [batch, heads, head_dim], over its ``kv_lens[r]``
    tokens in the pages ``block_table[r]`` of ``cache`` (its own among them: ``write_kv`` goes
    before). A request without any gives zeros."""
    code = _dtype(q, "q")
    dev = q.device
    c = _cache(cache, dev)
    dtype = q.dtype
    q_rows = _rows(q, "q", dev, dtype)
    batch, heads, dim = q.shape
    if dim != c.head_dim or heads < 1 or heads % c.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {c.kv_heads} kv heads of "
                         f"{c.head_dim}")
    _ints(block_table, "block_table", dev, 2, batch)
    _ints(kv_lens, "kv_lens", dev, 1, batch)
    max_pages = block_table.shape[1]
    if max_pages < 1:
        raise ValueError("block_table must have a column")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ws = _workspace(dev, heads, c.kv_heads, dim, c.page_size)
    _call("pi0_attention_paged", dev, code, *q_rows, batch, heads, ctypes.byref(c),
          block_table.data_ptr(), max(block_table.stride(0), max_pages), max_pages,
          kv_lens.data_ptr(), dim ** -0.5 if scale is None else scale,
          *_rows(out, "out", dev, dtype, q.shape), ws.data_ptr(), ws.numel(), _err_ptr(err, dev))
    return out


__all__ = ["KVCache8", "Slots", "build_slots", "write_kv", "attention_prompt", "attention_paged",
           "check", "PAGED_ERRORS"]
