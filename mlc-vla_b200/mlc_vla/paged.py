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
import math
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
    _ints(err, "err", device, 1)
    return err.data_ptr()


def _ints(t: torch.Tensor, name: str, device: torch.device, dim: int) -> None:
    if t.dtype != torch.int32 or t.device != device or t.dim() != dim or (
            t.shape[-1] > 1 and t.stride(-1) != 1) or (
            dim == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must be a {dim}-dimensional int32 tensor on {device}, "
                         f"contiguous along its last dimension and not expanded")


def _rows(t: torch.Tensor, name: str, device: torch.device, dtype, shape=None) -> None:
    """[tokens, heads, head_dim] in 16 bits, read in 16-byte vectors along the last dimension."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] {dtype} tensor on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.numel() and (t.stride(2) != 1 or t.data_ptr() % 16
                      or any(x % 8 or x == 0 for x in _strides(t))):
        raise ValueError(f"{name} must be contiguous along its last dimension, with token and "
                         f"head strides that are multiples of 8 elements (not expanded) and a "
                         f"16-byte aligned start")


def _strides(t: torch.Tensor):
    """Token and head stride; one that no second token or head uses is free, so a valid one."""
    dim = t.shape[2]
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * dim,
            t.stride(1) if t.shape[1] > 1 else dim)


def _dtype(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda or t.dtype not in _DTYPE:
        raise ValueError(f"{name} must be a float16 or bfloat16 CUDA tensor")
    return _DTYPE[t.dtype]


def _head_dim(d: int) -> None:
    if d < 8 or d % 8 or d > 256:
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, not {d}")


def _cache(c: KVCache8, device: torch.device) -> _lib.Pi0Kv8C:
    if c.k.dim() != 4 or c.k.shape != c.v.shape:
        raise ValueError("cache codes must be [pages, kv heads, page, head_dim], alike for k and v")
    pages, heads, page, dim = c.k.shape
    _head_dim(dim)
    for t in (c.k, c.v):
        if t.dtype != torch.float8_e4m3fn or t.device != device or not t.is_contiguous() or (
                t.data_ptr() % 16):
            raise ValueError(f"cache codes must be contiguous, 16-byte aligned float8_e4m3fn "
                             f"tensors on {device}")
    for t in (c.k_scale, c.v_scale):
        if t.dtype != torch.float32 or t.device != device or not t.is_contiguous() or (
                t.shape != c.k.shape[:2]):
            raise ValueError(f"cache scales must be contiguous float32 [pages, kv heads] tensors "
                             f"on {device}")
    return _lib.Pi0Kv8C(c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(),
                        pages, page, heads, dim)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _call(name: str, device: torch.device, *args) -> None:
    lib = _lib.load()
    if torch.cuda.current_device() == device.index:
        rc = getattr(lib, name)(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, _stream(device))
    if rc:
        _lib.check(rc, None, name)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(device: torch.device, heads: int, kv_heads: int, dim: int, page: int) -> int:
    with torch.cuda.device(device):
        n = _lib.load().pi0_attention_paged_workspace(heads, kv_heads, dim, page)
    if n < 0:
        raise _lib.Pi0Error(_lib.PI0_ERR_CUDA, "pi0_attention_paged_workspace")
    return n


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
    for t, name, n in ((kv_lens, "kv_lens", batch), (new_lens, "new_lens", batch),
                       (free_pos, "free_pos", 1), (free_pages, "free_pages", None)):
        _ints(t, name, dev, 1)
        if n is not None and t.shape[0] != n:
            raise ValueError(f"{name} must hold {n} numbers")
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
    buf = torch.empty(2 * batch + 2 + 2 * num_tokens, dtype=torch.int32, device=dev)
    out = Slots(buf[:batch + 1], buf[2 * batch + 2:2 * batch + 2 + num_tokens],
                buf[2 * batch + 2 + num_tokens:], buf[batch + 1:2 * batch + 1],
                buf[2 * batch + 1:2 * batch + 2])
    base = buf.data_ptr()
    _call("pi0_build_slots", dev, batch, kv_lens.data_ptr(), new_lens.data_ptr(),
          block_table.data_ptr(), max(block_table.stride(0), max_pages), max_pages,
          free_pages.data_ptr(), free_pages.shape[0], free_pos.data_ptr(), num_pages, page_size,
          num_tokens, base, base + 4 * (2 * batch + 2), base + 4 * (2 * batch + 2 + num_tokens),
          base + 4 * (batch + 1), base + 4 * (2 * batch + 1), _err_ptr(err, dev))
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
    tokens = k.shape[0]
    _rows(k, "k", dev, k.dtype, (tokens, c.kv_heads, c.head_dim))
    _rows(v, "v", dev, k.dtype, (tokens, c.kv_heads, c.head_dim))
    for t, name, n in ((cu_seqlens, "cu_seqlens", kv_lens.shape[0] + 1),
                       (kv_lens, "kv_lens", kv_lens.shape[0]),
                       (slot_mapping, "slot_mapping", tokens)):
        _ints(t, name, dev, 1)
        if t.shape[0] != n:
            raise ValueError(f"{name} must hold {n} numbers")
    if max_new is not None and max_new < 0:
        raise ValueError("max_new must not be negative")
    _call("pi0_write_kv", dev, code, k.data_ptr(), *_strides(k), v.data_ptr(),
          *_strides(v), tokens, kv_lens.shape[0], cu_seqlens.data_ptr(),
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
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    _head_dim(dim)
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} kv heads")
    _rows(q, "q", dev, q.dtype)
    _rows(k, "k", dev, q.dtype, (k.shape[0], kv_heads, dim))
    _rows(v, "v", dev, q.dtype, k.shape)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    batch = cu_seqlens_q.shape[0] - 1
    if batch < 0 or (batch == 0 and tokens):
        raise ValueError("cu_seqlens_q must hold one number more than there are requests")
    for t, name, n in ((cu_seqlens_q, "cu_seqlens_q", batch + 1),
                       (cu_seqlens_k, "cu_seqlens_k", batch + 1),
                       (prefix_lens, "prefix_lens", batch)):
        if t is None:
            continue
        _ints(t, name, dev, 1)
        if t.shape[0] != n:
            raise ValueError(f"{name} must hold {n} numbers")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=dev)
    else:
        _rows(out, "out", dev, q.dtype, q.shape)
    _call("pi0_attention_prompt", dev, code, q.data_ptr(), *_strides(q), k.data_ptr(),
          *_strides(k), v.data_ptr(), *_strides(v), tokens, k.shape[0],
          heads, kv_heads, dim, batch, cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
          None if prefix_lens is None else prefix_lens.data_ptr(),
          1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(), *_strides(out),
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
    _rows(q, "q", dev, q.dtype)
    batch, heads, dim = q.shape
    if dim != c.head_dim or heads % c.kv_heads or heads < 1:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {c.kv_heads} kv heads of "
                         f"{c.head_dim}")
    _ints(block_table, "block_table", dev, 2)
    _ints(kv_lens, "kv_lens", dev, 1)
    if block_table.shape[0] != batch or kv_lens.shape[0] != batch or block_table.shape[1] < 1:
        raise ValueError(f"block_table and kv_lens must hold {batch} requests")
    if out is None:
        out = torch.empty((batch, heads, dim), dtype=q.dtype, device=dev)
    else:
        _rows(out, "out", dev, q.dtype, q.shape)
    max_pages = block_table.shape[1]
    ws = torch.empty(_workspace_bytes(dev, heads, c.kv_heads, dim, c.page_size), dtype=torch.uint8,
                     device=dev)
    _call("pi0_attention_paged", dev, code, q.data_ptr(), *_strides(q), batch, heads,
          ctypes.byref(c), block_table.data_ptr(), max(block_table.stride(0), max_pages),
          max_pages, kv_lens.data_ptr(), 1.0 / math.sqrt(dim) if scale is None else scale,
          out.data_ptr(), *_strides(out), ws.data_ptr(), ws.numel(), _err_ptr(err, dev))
    return out


__all__ = ["KVCache8", "Slots", "build_slots", "write_kv", "attention_prompt", "attention_paged",
           "check", "PAGED_ERRORS"]
