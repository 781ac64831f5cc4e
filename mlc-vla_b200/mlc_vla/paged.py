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

There is no backward pass: an attention of tensors that ask for gradients gives a result whose
backward raises, and what ``write_kv`` stores has no history.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from mlc_vla import _lib

PAGED_ERRORS = {
    1: "a bounded wait in a kernel gave up", 2: "a bounded wait in a kernel gave up",
    3: "a bounded wait in a kernel gave up",
    16: "a length below zero, or more new tokens than num_tokens",
    17: "a request longer than its row of the block table",
    18: "no free page left for a request",
    19: "a page number outside the pool, or a slot that is not its token's",
}


def _native():
    return _lib._native or _lib.load_paged()


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


def check(device="cuda") -> None:
    """Wait for the device, and raise what the calls without an `err` of their own recorded."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    f = _native().flag(index)
    if f is None:
        return
    torch.cuda.synchronize(index)
    code = int(f.item())
    if code:
        f.zero_()
        raise _lib.Pi0Error(code, PAGED_ERRORS.get(code, "a kernel reported an error"))


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
    return Slots(*_native().build_slots(kv_lens, new_lens, block_table, free_pages, free_pos,
                                        page_size, num_tokens, num_pages, err))


def write_kv(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
             kv_lens: torch.Tensor, slot_mapping: torch.Tensor, max_new: Optional[int] = None,
             err: Optional[torch.Tensor] = None) -> None:
    """Keys and values [tokens, kv heads, head_dim] into the pages of ``cache`` at
    ``slot_mapping``. ``cu_seqlens`` [batch + 1]: the requests' tokens; ``kv_lens`` [batch]: their
    tokens cached before these. ``max_new``: the most new tokens of one request, which sizes the
    launch (default: all of them)."""
    _native().write_kv(*cache, k, v, cu_seqlens, kv_lens, slot_mapping, max_new, err)


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
    sees no key gives zeros. ``out``: for the result, apart from q, k and v."""
    return _native().attention_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, prefix_lens, scale, out,
                                      err)


def attention_paged(q: torch.Tensor, cache: KVCache8, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None,
                    err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per request, q [batch, heads, head_dim], over its ``kv_lens[r]``
    tokens in the pages ``block_table[r]`` of ``cache`` (its own among them: ``write_kv`` goes
    before). A request without any gives zeros. ``out``: for the result; it may be q."""
    return _native().attention_paged(q, *cache, block_table, kv_lens, scale, out, err)


__all__ = ["KVCache8", "Slots", "build_slots", "write_kv", "attention_prompt", "attention_paged",
           "check", "PAGED_ERRORS"]
