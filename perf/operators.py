"""The operators of text generation behind the prefix expert, as cases to be measured: block tables
and slot maps built from request lengths, the paged key/value cache in 8 bits, attention over
packed prompts, and attention of single tokens over the cache.

The definitions, for every operator here:

* A page holds `page` tokens of one request. The table of a request lists its pages in order; token
  `pos` of the request lies in page `table[pos // page]` at row `pos % page`, and its slot is
  `table[pos // page] * page + pos % page`. New pages are taken from the free list in the order of
  the requests.
* The cache keeps e4m3 codes [pages, kv heads, page, head_dim] and one fp32 scale for each page and
  kv head, for keys and values apart. A scale is the smallest power of two (not below 2^-64) with
  which the largest magnitude of the page's tokens fits into +-448. Tokens that join a page keep or
  raise its scale; when it rises, the codes already there are rounded to the new scale.
* Attention over prompts: key j of a request is seen by its query i (both counted within the
  request, the last query at the last key) if j <= i + keys - queries, or if j is below the
  request's bidirectional prefix.
* Attention over the cache: one query token per request sees all its cached tokens; a request
  without any gives zeros.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

FP8_MAX = 448.0
MIN_SCALE = 2.0 ** -64


# ---- cases ----------------------------------------------------------------------------------------

def _slots(batch, held, new, page, lens_seed):
    return {"op": "slots", "batch": batch, "held_min": held[0], "held_max": held[1],
            "new_min": new[0], "new_max": new[1], "page": page, "lens_seed": lens_seed}


def _write(batch, held, new, page, kv_heads, head_dim, dtype, lens_seed):
    return {**_slots(batch, held, new, page, lens_seed), "op": "write", "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype}


def _prompt(batch, held, new, prefix, heads, kv_heads, head_dim, dtype, lens_seed):
    return {"op": "prompt", "batch": batch, "held_min": held[0], "held_max": held[1],
            "new_min": new[0], "new_max": new[1], "prefix": prefix, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "lens_seed": lens_seed}


def _paged(batch, held, page, heads, kv_heads, head_dim, dtype, lens_seed):
    return {"op": "paged", "batch": batch, "held_min": held[0], "held_max": held[1], "page": page,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "lens_seed": lens_seed}


def listed():
    return [
        # one token for each of 32 observations that are answering in text: the smallest call
        {"name": "slots_decode", **_slots(32, (700, 1100), (1, 1), 64, 1)},
        # admission of many requests at once, fresh ones and ones that go on, odd lengths
        {"name": "slots_prompts", **_slots(1024, (0, 2000), (1, 401), 16, 2)},
        # the prefixes of 32 observations (700 to 968 valid tokens each) into the cache, one kv head
        {"name": "write_prefix", **_write(32, (0, 0), (700, 968), 64, 1, 256, "float16", 3)},
        # one new token for each of 256 requests, into pages that mostly hold tokens already
        {"name": "write_decode", **_write(256, (0, 1023), (1, 1), 16, 8, 128, "bfloat16", 4)},
        # one long prompt of odd length, several kv heads
        {"name": "write_long", **_write(1, (0, 0), (32771, 32771), 32, 8, 128, "bfloat16", 5)},
        # a handful of short instructions, small heads: latency counts
        {"name": "prompt_short", **_prompt(4, (0, 0), (1, 50), 0, 4, 1, 64, "float16", 6)},
        # the prefixes of 32 observations, packed: 768 image tokens see each other, text is causal
        {"name": "prompt_prefix", **_prompt(32, (0, 0), (700, 968), 768, 8, 1, 256, "float16", 7)},
        # one long causal prompt with grouped heads
        {"name": "prompt_long", **_prompt(1, (0, 0), (8192, 8192), 0, 32, 8, 128, "bfloat16", 8)},
        # further chunks of eight prompts, each on thousands of earlier keys
        {"name": "prompt_chunk", **_prompt(8, (1000, 4000), (17, 300), 0, 16, 4, 128, "bfloat16", 9)},
        # one request answering, one observation in the cache: latency counts
        {"name": "paged_single", **_paged(1, (1005, 1005), 64, 8, 1, 256, "float16", 10)},
        # 32 requests answering together
        {"name": "paged_batch", **_paged(32, (700, 1100), 64, 8, 1, 256, "bfloat16", 11)},
        # long contexts of very different lengths, grouped heads, small pages
        {"name": "paged_long", **_paged(64, (1, 16384), 16, 32, 8, 128, "bfloat16", 12)},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["slots", "write", "prompt", "prompt", "paged", "paged"])
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["float16", "bfloat16"])
    page = rng.choice([16, 32, 64, 128])
    lens_seed = rng.randrange(1 << 30)
    if op in ("slots", "write"):
        batch = _log_int(rng, 1, 1024 if op == "slots" else 256)
        held = rng.choice([0, _log_int(rng, 1, 2000 if op == "slots" else 1000)])
        new = rng.choice([1, _log_int(rng, 1, max(2, min(8192, 32768 // batch)))])
        low = rng.choice([new, 1])
        if op == "slots":
            return _slots(batch, (0, held), (low, new), page, lens_seed)
        return _write(batch, (0, held), (low, new), page, min(kv_heads, 1024 // head_dim), head_dim,
                      dtype, lens_seed)
    if op == "prompt":
        # at most the pairs of the long prompt: batch * heads * queries * keys
        heads = kv_heads * group
        batch = _log_int(rng, 1, 32)
        room = (8192 * 8192 * 32 * 128) / (batch * heads * head_dim)
        new = _log_int(rng, 1, max(2, min(8192, int(math.sqrt(room)))))
        held = rng.choice([0, 0, _log_int(rng, 1, max(2, min(8192, int(room / new) - new)))])
        low = rng.choice([new, max(1, new // 2), 1])
        prefix = rng.choice([0, 0, rng.randrange(new + held + 1)])
        return _prompt(batch, (held // 2, held), (low, new), prefix, heads, kv_heads, head_dim,
                       dtype, lens_seed)
    batch = _log_int(rng, 1, 128)
    most = max(16, min(32768, (64 * 16384 * 8 * 128) // (batch * kv_heads * head_dim)))
    held = _log_int(rng, 1, most)
    low = rng.choice([held, max(1, held // 2), 0])
    return _paged(batch, (low, held), page, kv_heads * group, kv_heads, head_dim, dtype, lens_seed)


def _lens(case, what):
    """Lengths of the requests, from the case alone: cached tokens ("held") or new ones ("new")."""
    rng = random.Random(case["lens_seed"] * 2 + (what == "new"))
    low, high = case[what + "_min"], case[what + "_max"]
    return [rng.randint(low, high) for _ in range(case["batch"])]


# ---- inputs ---------------------------------------------------------------------------------------

def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages_of(tokens, page):
    return (tokens + page - 1) // page


def _table(lens, page, order):
    """[batch, columns] page numbers for requests of these lengths, taken from `order`."""
    counts = [_pages_of(n, page) for n in lens]
    columns = max(1, max(counts))
    table = np.full((len(lens), columns), -1, np.int64)
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        at += n
    return table


def _tokens(gen, rows, heads, head_dim, dtype):
    """Keys or values: normal entries, each token with a magnitude of its own."""
    x = torch.randn((rows, heads, head_dim), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, heads, 1), generator=gen, device="cuda"))
    return x.to(getattr(torch, dtype))


def _scale_of(amax):
    mantissa, exponent = torch.frexp(amax)
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    scale = torch.ldexp(torch.ones_like(amax), exponent)
    return torch.where(amax > 0, scale, torch.zeros_like(scale)).clamp_min(MIN_SCALE)


def _filled_cache(gen, pages, page, kv_heads, head_dim):
    """A cache whose pages all hold tokens: codes and scales of keys and of values."""
    out = []
    for _ in range(2):
        x = torch.randn((pages, kv_heads, page, head_dim), generator=gen, device="cuda",
                        dtype=torch.bfloat16)
        x *= torch.exp(0.5 * torch.randn((pages, kv_heads, 1, 1), generator=gen, device="cuda"))
        scale = _scale_of(x.abs().amax((2, 3)).float())
        x /= scale.to(x.dtype)[:, :, None, None]
        out += [x.to(torch.float8_e4m3fn), scale]
    return {"k": out[0], "v": out[2], "k_scale": out[1], "v_scale": out[3]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"op": case["op"], "case": case}
    held = _lens(case, "held")
    if case["op"] in ("slots", "write"):
        new, page = _lens(case, "new"), case["page"]
        total = [a + b for a, b in zip(held, new)]
        held_pages = sum(_pages_of(n, page) for n in held)
        # the pool: what the requests need, and some pages that stay free
        pages = sum(_pages_of(n, page) for n in total) + sum(_pages_of(n, page) for n in held) // 8 + 8
        order = np.random.RandomState(seed % (1 << 31)).permutation(pages)
        columns = max(_pages_of(n, page) for n in total)
        table = np.full((case["batch"], columns), -1, np.int64)
        first = _table(held, page, order)
        table[:, :min(columns, first.shape[1])] = first[:, :columns]
        state.update(kv_lens=_int32(held), new_lens=_int32(new), block_table=_int32(table),
                     free_pages=_int32(order[held_pages:]), free_pos=_int32([0]), page=page,
                     tokens=sum(new))
        if case["op"] == "write":
            # the slots are in hand: another operator made them
            state.update(_plain_slots(state))
            state["max_new"] = max(new)
            state["cache"] = _filled_cache(gen, pages, page, case["kv_heads"], case["head_dim"])
            size = (sum(new), case["kv_heads"], case["head_dim"], case["dtype"])
            state.update(k=_tokens(gen, *size), v=_tokens(gen, *size))
    elif case["op"] == "prompt":
        new = _lens(case, "new")
        keys = [a + b for a, b in zip(held, new)]
        state.update(q=_tokens(gen, sum(new), case["heads"], case["head_dim"], case["dtype"]),
                     k=_tokens(gen, sum(keys), case["kv_heads"], case["head_dim"], case["dtype"]),
                     v=_tokens(gen, sum(keys), case["kv_heads"], case["head_dim"], case["dtype"]),
                     cu_q=_int32(np.cumsum([0] + new)), cu_k=_int32(np.cumsum([0] + keys)),
                     prefix=_int32([min(case["prefix"], n) for n in keys]),
                     max_q=max(new), max_k=max(keys))
    else:
        page = case["page"]
        pages = sum(_pages_of(n, page) for n in held) + 8
        order = np.random.RandomState(seed % (1 << 31)).permutation(pages)
        state.update(cache=_filled_cache(gen, pages, page, case["kv_heads"], case["head_dim"]),
                     block_table=_int32(_table(held, page, order)), kv_lens=_int32(held),
                     q=_tokens(gen, case["batch"], case["heads"], case["head_dim"], case["dtype"]))
    return state


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_slots(s):
    """Tables and slots: a sum over the requests gives each its tokens and its new pages."""
    page, held, new, table = s["page"], s["kv_lens"].long(), s["new_lens"].long(), s["block_table"]
    have = (held + page - 1) // page
    need = (held + new + page - 1) // page - have
    offset = torch.cumsum(need, 0) - need
    cu = torch.zeros(len(held) + 1, dtype=torch.long, device=held.device)
    cu[1:] = torch.cumsum(new, 0)
    column = torch.arange(table.shape[1], device=held.device)
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    index = s["free_pos"].long() + offset[:, None] + column - have[:, None]
    taken = s["free_pages"][index.clamp(0, len(s["free_pages"]) - 1)]
    table = torch.where(fresh, taken, table)
    token = torch.arange(s["tokens"], device=held.device)
    request = torch.searchsorted(cu[1:], token, right=True)
    position = held[request] + token - cu[request]
    slot = table[request, position // page].long() * page + position % page
    return {"block_table": table, "cu_seqlens": cu.int(), "positions": position.int(),
            "slot_mapping": slot.int(), "kv_lens_new": (held + new).int(),
            "free_pos_new": s["free_pos"] + need.sum().int()}


def _plain_write_one(s, codes, scale, x):
    """Codes and scales of a pool after the tokens `x` have joined it at their slots."""
    page, slot = s["page"], s["slot_mapping"].long()
    x = x.float()
    where = (slot // page)[:, None].expand(-1, x.shape[1])
    amax = torch.full_like(scale, -1.0).scatter_reduce(0, where, x.abs().amax(2), "amax")
    # rows that the page of a request's first new token holds already
    first = s["cu_seqlens"][:-1].long().clamp(max=len(slot) - 1)
    rows = torch.zeros(len(scale), dtype=torch.long, device=x.device)
    rows = rows.scatter_reduce(0, slot[first] // page, s["kv_lens"].long() % page, "amax")
    fits = _scale_of(amax.clamp_min(0))
    after = torch.where((rows > 0)[:, None], torch.maximum(scale, fits), fits)
    after = torch.where(amax >= 0, after, scale)
    kept = torch.arange(page, device=x.device)[None, :] < rows[:, None]
    moved = (codes.float() * (scale / after)[:, :, None, None]).to(torch.float8_e4m3fn)
    grown = kept[:, None, :, None] & (after > scale)[:, :, None, None]
    bits = torch.where(grown, moved.view(torch.uint8), codes.view(torch.uint8))
    fresh = (x / after[slot // page][:, :, None]).to(torch.float8_e4m3fn)
    bits[slot // page, :, slot % page] = fresh.view(torch.uint8)
    return bits.view(torch.float8_e4m3fn), after


def _plain_write(s):
    k, k_scale = _plain_write_one(s, s["cache"]["k"], s["cache"]["k_scale"], s["k"])
    v, v_scale = _plain_write_one(s, s["cache"]["v"], s["cache"]["v_scale"], s["v"])
    return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


def _softmax_rows(scores, seen, values):
    """Sum of values weighted by the softmax over the seen keys; zeros where none is seen."""
    scores = torch.where(seen, scores, float("-inf"))
    most = scores.amax(-1, keepdim=True)
    scores -= torch.where(torch.isfinite(most), most, 0.0)
    weights = torch.exp_(scores)
    total = weights.sum(-1, keepdim=True)
    out = weights @ values
    return torch.where(total > 0, out / total, 0.0)


def _plain_prompt(s):
    """Each request padded to the longest: scores, mask, softmax, weighted sum."""
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    heads, kv_heads, head_dim = q.shape[1], k.shape[1], q.shape[2]
    n_q, n_k = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    i = torch.arange(s["max_q"], device=q.device)
    j = torch.arange(s["max_k"], device=q.device)
    row = (cu_q[:-1, None] + i).clamp(max=len(q) - 1)
    key = (cu_k[:-1, None] + j).clamp(max=len(k) - 1)
    # [batch, kv head, queries of its group or keys, head_dim]
    qp = q[row].float().view(len(n_q), len(i), kv_heads, -1, head_dim).permute(0, 2, 3, 1, 4)
    kp, vp = (x[key].float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    last = i[None, :] + (n_k - n_q)[:, None]
    seen = (j <= last[:, :, None]) | (j < s["prefix"].long()[:, None, None])
    seen &= (j < n_k[:, None])[:, None, :]
    vp = vp * (j < n_k[:, None])[:, None, None, :, None]
    out = _softmax_rows((qp / math.sqrt(head_dim)) @ kp.transpose(-1, -2), seen[:, None, None], vp)
    out = out.permute(0, 3, 1, 2, 4).reshape(len(n_q), len(i), heads, head_dim)
    token = torch.arange(len(q), device=q.device)
    request = torch.searchsorted(cu_q[1:], token, right=True)
    return out[request, token - cu_q[request]].to(q.dtype)


def _plain_paged(s):
    """The pages of each request side by side as numbers, then attention of its one token."""
    q, c, table, n = s["q"], s["cache"], s["block_table"].long(), s["kv_lens"].long()
    kv_heads, page, head_dim = c["k"].shape[1:]
    pages = table.clamp_min(0)

    def numbers(codes, scale):
        x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
        x *= scale[pages][:, :, :, None, None]
        return x.transpose(1, 2).reshape(len(q), kv_heads, -1, head_dim)

    seen = torch.arange(table.shape[1] * page, device=q.device) < n[:, None]
    k, v = numbers(c["k"], c["k_scale"]), numbers(c["v"], c["v_scale"])
    v *= seen[:, None, :, None]
    qf = q.float().view(len(q), kv_heads, -1, head_dim) / math.sqrt(head_dim)
    return _softmax_rows(qf @ k.transpose(-1, -2), seen[:, None, None], v).reshape(q.shape).to(q.dtype)


# ---- one pass -------------------------------------------------------------------------------------

def _paged_module():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlc-vla_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mlc_vla import paged
    return paged


def run(state):
    s = state
    if not own:
        return {"slots": _plain_slots, "write": _plain_write, "prompt": _plain_prompt,
                "paged": _plain_paged}[s["op"]](s)
    paged = sys.modules.get("mlc_vla.paged") or _paged_module()
    if s["op"] == "slots":
        r = paged.build_slots(s["kv_lens"], s["new_lens"], s["block_table"], s["free_pages"],
                              s["free_pos"], s["page"], s["tokens"])
        return {"block_table": s["block_table"], "cu_seqlens": r.cu_seqlens,
                "positions": r.positions, "slot_mapping": r.slot_mapping,
                "kv_lens_new": r.kv_lens, "free_pos_new": r.free_pos}
    if s["op"] == "prompt":
        return paged.attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"],
                                      prefix_lens=s["prefix"])
    cache = paged.KVCache8(**s["cache"])
    if s["op"] == "write":
        paged.write_kv(cache, s["k"], s["v"], s["cu_seqlens"], s["kv_lens"], s["slot_mapping"],
                       max_new=s["max_new"])
        return dict(s["cache"])
    return paged.attention_paged(s["q"], cache, s["block_table"], s["kv_lens"])


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    held = _lens(case, "held")
    if case["op"] == "slots":
        new, page = _lens(case, "new"), case["page"]
        fresh = sum(_pages_of(a + b, page) - _pages_of(a, page) for a, b in zip(held, new))
        # lengths in and out, a page number read and one written per new page, two numbers a token
        return {"bytes": 4 * (4 * case["batch"] + 2 * fresh + 2 * sum(new)), "flops": 4 * sum(new)}
    width = case["kv_heads"] * case["head_dim"]
    if case["op"] == "write":
        new, page = _lens(case, "new"), case["page"]
        pages = sum(_pages_of(a + b, page) - a // page for a, b in zip(held, new))
        tokens = sum(new)
        return {"bytes": 2 * tokens * width * 3 + 2 * pages * case["kv_heads"] * 4 + 4 * tokens,
                "flops": 4 * tokens * width}
    if case["op"] == "prompt":
        new = _lens(case, "new")
        pairs = 0
        for h, n in zip(held, new):
            prefix = min(case["prefix"], h + n)
            below = max(0, min(n, prefix - h))      # queries whose own key lies in the prefix
            pairs += below * prefix + (n * (n + 1) - below * (below + 1)) // 2 + (n - below) * h
        keys = sum(held) + sum(new)
        return {"bytes": 2 * (2 * sum(new) * case["heads"] * case["head_dim"] + 2 * keys * width),
                "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    pages = sum(_pages_of(n, case["page"]) for n in held)
    tokens, out = sum(held), case["batch"] * case["heads"] * case["head_dim"]
    return {"bytes": 2 * tokens * width + 2 * pages * case["kv_heads"] * 4 + 4 * pages + 4 * out,
            "flops": 4 * tokens * case["heads"] * case["head_dim"]}


# ---- in 64 bits -----------------------------------------------------------------------------------

def _exact_code(x, scale):
    """x / scale on the grid of e4m3 (3 bits after the point, smallest step 2^-9), ties to even."""
    y = x / scale
    _, exponent = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (exponent - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _exact_write(s):
    """Page by page, as the definition says."""
    page, out = s["page"], {}
    cu, held = s["cu_seqlens"].tolist(), s["kv_lens"].tolist()
    slot = s["slot_mapping"].tolist()
    for name in ("k", "v"):
        codes = s["cache"][name].double()
        scale = s["cache"][name + "_scale"].double()
        x = s[name].double()
        for r, start in enumerate(held):
            at, end = cu[r], cu[r + 1]
            while at < end:
                row = slot[at] % page
                n = min(page - row, end - at)
                p, part = slot[at] // page, x[at:at + n]
                most = part.abs().amax((0, 2))
                power = torch.ceil(torch.log2(most / FP8_MAX))
                power += (most > FP8_MAX * torch.exp2(power)).double()
                power -= (most <= FP8_MAX * torch.exp2(power - 1)).double()
                new = torch.exp2(power).clamp_min(MIN_SCALE)
                if row:
                    new = torch.maximum(new, scale[p])
                    old = codes[p, :, :row] * scale[p][:, None, None]
                    codes[p, :, :row] = _exact_code(old, new[:, None, None])
                scale[p] = new
                codes[p, :, row:row + n] = _exact_code(part.transpose(0, 1), new[:, None, None])
                at += n
        out[name], out[name + "_scale"] = codes, scale
    return {key: out[key] for key in ("k", "v", "k_scale", "v_scale")}


def _exact_rows(q, k, v, seen):
    """Attention of [heads, queries, d] on [heads, keys, d], in pieces of the queries."""
    out = torch.zeros_like(q)
    piece = max(1, (1 << 27) // max(1, k.shape[0] * k.shape[1]))
    for a in range(0, q.shape[1], piece):
        x = q[:, a:a + piece] @ k.transpose(1, 2) / math.sqrt(q.shape[2])
        x = x.masked_fill(~seen[a:a + piece], -math.inf)
        p = torch.softmax(x, -1).nan_to_num(0.0)
        out[:, a:a + piece] = p @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "slots":
        return None
    if case["op"] == "write":
        return _exact_write(s)
    q = s["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    if case["op"] == "prompt":
        k, v = s["k"].double(), s["v"].double()
        cu_q, cu_k, prefix = s["cu_q"].tolist(), s["cu_k"].tolist(), s["prefix"].tolist()
        for r in range(case["batch"]):
            a, b, c, d = cu_q[r], cu_q[r + 1], cu_k[r], cu_k[r + 1]
            i = torch.arange(b - a, device="cuda")[:, None] + (d - c) - (b - a)
            j = torch.arange(d - c, device="cuda")[None, :]
            seen = (j <= i) | (j < prefix[r])
            for g in range(case["kv_heads"]):
                h = slice(g * group, (g + 1) * group)
                kg, vg = (x[c:d, g].expand(group, -1, -1) for x in (k, v))
                out[a:b, h] = _exact_rows(q[a:b, h].transpose(0, 1), kg, vg, seen).transpose(0, 1)
        return out
    table, lens = s["block_table"].tolist(), s["kv_lens"].tolist()
    for r, n in enumerate(lens):
        if n == 0:
            continue
        p = torch.tensor(table[r][:_pages_of(n, case["page"])], device="cuda")
        k, v = (s["cache"][x].view(torch.uint8)[p].view(torch.float8_e4m3fn).double()
                * s["cache"][x + "_scale"][p].double()[:, :, None, None] for x in ("k", "v"))
        k, v = (x.transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, :n] for x in (k, v))
        x = q[r].view(case["kv_heads"], group, -1)
        seen = torch.ones((group, n), dtype=torch.bool, device="cuda")
        out[r] = _exact_rows(x, k, v, seen).reshape(case["heads"], -1)
    return out
