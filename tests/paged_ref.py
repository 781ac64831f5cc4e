"""Plain numpy restatements, in 64 bits, of the text-generation operators, and the error bounds their
outputs are held to. Written from the definitions: a request at a time, a page at a time."""

import numpy as np

# unit roundoff of the output types (half an ulp, relative)
UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def build_slots(kv_lens, new_lens, table, free_pages, free_pos, page, num_tokens):
    """(table, cu, positions, slots, kv_lens, free_pos): requests in order, pages from the list."""
    table = table.copy()
    cu, positions, slots, lens = [0], np.zeros(num_tokens, int), np.full(num_tokens, -1), []
    asked = taken = 0  # pages asked for so far (admitted or not), pages taken
    for r, (kv, new) in enumerate(zip(kv_lens, new_lens)):
        have, need = -(-kv // page), -(-(kv + new) // page) - -(-kv // page)
        fits = kv + new <= table.shape[1] * page
        need = need if fits else 0
        asked += need
        ok = fits and (need == 0 or free_pos + asked <= len(free_pages))
        if ok and need:
            table[r, have:have + need] = free_pages[free_pos + asked - need:free_pos + asked]
            taken = asked
        for i in range(new):
            t = cu[-1] + i
            positions[t] = kv + i
            if ok:
                slots[t] = table[r, (kv + i) // page] * page + (kv + i) % page
        lens.append(kv + new if ok else kv)
        cu.append(cu[-1] + new)
    return table, np.array(cu), positions, slots, np.array(lens), free_pos + taken


def e4m3(x):
    """x rounded to the e4m3 grid (3 fraction bits, smallest step 2^-9), ties to even; NaN stays."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        e = np.floor(np.log2(np.where(x == 0, 1.0, np.abs(x))))
        e = np.where(2.0 ** (e + 1) <= np.abs(x), e + 1, np.where(2.0 ** e > np.abs(x), e - 1, e))
        step = 2.0 ** (np.maximum(e, -6) - 3)
        return np.round(x / step) * step


def pow2_scale(amax):
    s = 2.0 ** -64
    while amax > 448.0 * s:
        s *= 2.0
    return s


def write_kv(codes, scales, x, cu, kv_lens, slots, page):
    """Codes [pages, heads, page, dim] and scales [pages, heads] (numbers) after the tokens joined."""
    codes, scales = codes.copy(), scales.copy()
    for r, start in enumerate(kv_lens):
        t = cu[r]
        while t < cu[r + 1]:
            row = (start + t - cu[r]) % page
            n = min(page - row, cu[r + 1] - t)
            if slots[t] >= 0:
                p = slots[t] // page
                for h in range(codes.shape[1]):
                    part = x[t:t + n, h].astype(np.float64)
                    finite = np.abs(part[np.isfinite(part)])
                    s = pow2_scale(finite.max() if finite.size else 0.0)
                    if row:
                        s = max(s, scales[p, h])
                        codes[p, h, :row] = e4m3(codes[p, h, :row] * (scales[p, h] / s))
                    codes[p, h, row:row + n] = e4m3(np.where(np.isfinite(part), part, np.nan) / s)
                    scales[p, h] = s
            t += n
    return codes, scales


def _attend(q, k, v, scale, dtype):
    """One query row over the keys it sees: the result and the bound on a kernel's error.

    With u the unit roundoff of the 16-bit type, n keys and d dimensions, a kernel may differ from
    the exact row by
      * u·|o|: the rounding of the result;
      * 2u·Σp|v|: weights held in the 16-bit type (u each) and their sum, held or rounded alike;
      * n·2^-25·max|v|: weights that fall below the 16-bit type's normal range, against a sum >= 1;
      * logits: d fp32 additions of the products, 2^-23 of Σ|q·k| each at most (tensor cores may
        truncate), and as much again for the scaling and the exponential (2^-21 of the logit's
        size, or 2^-20), in both numerator and denominator: a factor on Σp|v|;
      * n·2^-23·Σp|v|: the fp32 sum of the weighted values."""
    n, d = k.shape
    if n == 0:
        return np.zeros(v.shape[1]), np.zeros(v.shape[1])
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    o = p @ v
    spread = p @ np.abs(v)
    size = (np.abs(k) @ np.abs(q)).max() * abs(scale)
    u = UNIT[dtype]
    logit = 2 * (d * 2.0 ** -23 * size + 2.0 ** -21 * np.abs(s).max() + 2.0 ** -20)
    bound = (u * np.abs(o) + (2 * u + logit + n * 2.0 ** -23) * spread
             + n * 2.0 ** -25 * np.abs(v).max())
    return o, bound + 2.0 ** -24  # results below fp16's normal range round in steps of 2^-24


def attention_prompt(q, k, v, cu_q, cu_k, prefix, scale, dtype):
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    for r in range(len(cu_q) - 1):
        lq, lk = cu_q[r + 1] - cu_q[r], cu_k[r + 1] - cu_k[r]
        for i in range(lq):
            seen = [j for j in range(lk) if j <= i + lk - lq or j < prefix[r]]
            rows = cu_k[r] + np.array(seen, int)
            for h in range(q.shape[1]):
                t = cu_q[r] + i
                out[t, h], tol[t, h] = _attend(q[t, h], k[rows, h // group], v[rows, h // group],
                                               scale, dtype)
    return out, tol


def attention_paged(q, k, v, table, lens, scale, dtype):
    """k, v: the numbers [pages, heads, page, dim] that codes and scales stand for."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    group, page = q.shape[1] // k.shape[1], k.shape[2]
    for b, n in enumerate(lens):
        pages = table[b, :-(-n // page)]
        for h in range(q.shape[1]):
            kk, vv = (np.concatenate([x[p, h // group] for p in pages] or [x[0, 0, :0]])[:n]
                      for x in (k, v))
            out[b, h], tol[b, h] = _attend(q[b, h], kk, vv, scale, dtype)
    return out, tol
