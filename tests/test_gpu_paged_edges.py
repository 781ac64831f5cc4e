"""GPU: the text-generation operators (``mlc_vla.paged``) at the edges of their contracts: batches
without requests or tokens, slots left out within a page, error flags that hold an earlier call's
code, weights far below a row's largest. Restatements are written here, from the definitions."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).cuda()


# ---- block tables and slots -----------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [0, 1, 1024, 1025, 3000, 300000])
def test_slots_of_an_empty_batch(tokens):
    """More than 1024 tokens take several blocks."""
    from mlc_vla import paged

    none = dev(np.zeros(0, np.int32))
    table = torch.full((4, 5), -7, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = paged.build_slots(none, none, table[:0], dev([3, 1, 2]), dev([1]), 8, tokens, err=err)
    assert int(err.item()) == 0 and (table == -7).all()
    assert s.cu_seqlens.tolist() == [0] and s.kv_lens.numel() == 0 and s.free_pos.tolist() == [1]
    assert (s.slot_mapping == -1).all() and (s.positions == 0).all()
    assert len(s.slot_mapping) == len(s.positions) == tokens


@pytest.mark.parametrize("batch", [6127, 6128, 6136, 6143, 6144, 7000, 16384])
def test_slots_of_large_batches(batch):
    """The sums of up to 16384 requests lie in shared memory, beyond its default limit from 6128 on."""
    from mlc_vla import paged

    rng = np.random.default_rng(batch)
    page, columns = 4, 3
    kv, new = rng.integers(0, 6, batch), rng.integers(0, 4, batch)
    table = np.full((batch, columns), -1)
    have, need = -(-kv // page), -(-(kv + new) // page) - -(-kv // page)
    order = rng.permutation(int(have.sum() + need.sum()))
    at = 0
    for r in range(batch):
        table[r, :have[r]] = order[at:at + have[r]]
        at += have[r]
    free, want = order[at:], table.copy()
    cu = np.concatenate([[0], np.cumsum(new)])
    first = np.cumsum(need) - need
    positions, slots = [], []
    for r in range(batch):
        want[r, have[r]:have[r] + need[r]] = free[first[r]:first[r] + need[r]]
        for p in range(kv[r], kv[r] + new[r]):
            positions.append(p)
            slots.append(want[r, p // page] * page + p % page)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = dev(table)
    s = paged.build_slots(dev(kv), dev(new), got, dev(free), dev([0]), page, int(cu[-1]), err=err)
    assert int(err.item()) == 0
    for g, w in zip((got, *s), (want, cu, positions, slots, kv + new, [need.sum()])):
        assert np.array_equal(g.cpu().numpy(), np.array(w))


def test_slots_of_too_many_requests_are_refused():
    from mlc_vla import paged

    n = torch.zeros(16385, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        paged.build_slots(n, n, n[:, None].expand(16385, 1).contiguous(), n, n[:1], 8, 4)


def test_slots_of_lengths_beyond_31_bits():
    """A table row may have room for more tokens than a length can count."""
    from mlc_vla import paged

    page, columns = 1 << 20, 2100
    table = torch.zeros((2, columns), dtype=torch.int32, device="cuda")
    kv = [(1 << 31) - 648, 3]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = paged.build_slots(dev(kv), dev([1000, 2]), table, dev([5, 6, 7]), dev([0]), page, 1002, err=err)
    assert int(err.item()) == 17
    assert s.kv_lens.tolist() == [kv[0], 5] and s.free_pos.tolist() == [0]
    assert (s.slot_mapping[:1000] == -1).all() and s.slot_mapping[1000:].tolist() == [3, 4]
    assert not table.any()
    # up to the last length that it can
    err.zero_()
    s = paged.build_slots(dev(kv), dev([647, 2]), table, dev([5, 6, 7]), dev([0]), page, 649, err=err)
    assert int(err.item()) == 0 and s.kv_lens.tolist() == [(1 << 31) - 1, 5]
    assert s.positions[:647].tolist() == list(range(kv[0], kv[0] + 647))


# ---- the cache ------------------------------------------------------------------------------------

def e4m3_of(x):
    return torch.as_tensor(x, dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def joined(codes, scales, x, cu, lens, slots, page):
    """Codes (bytes) [pages, heads, page, dim] and scales after the tokens joined, token by token: a
    token is written if its slot is its row of a page of the pool, and of the page that the first
    such token of its run names. The scale is that of the written tokens and of the rows held before."""
    codes, scales, reported = codes.copy(), scales.copy(), False
    number = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    for r, start in enumerate(lens):
        t = cu[r]
        while t < cu[r + 1]:
            row = (start + t - cu[r]) % page
            n = min(page - row, cu[r + 1] - t)
            own = [i for i in range(n) if 0 <= slots[t + i] < len(codes) * page
                   and slots[t + i] % page == row + i]
            p = slots[t + own[0]] // page if own else -1
            put = [i for i in own if slots[t + i] // page == p]
            reported |= any(slots[t + i] >= 0 and i not in put for i in range(n))
            for h in range(codes.shape[1] if put else 0):
                part = x[[t + i for i in put], h]
                top = np.abs(part[np.isfinite(part)]).max(initial=0.0)
                s = 2.0 ** -64
                while top > 448.0 * s:
                    s *= 2.0
                if row:
                    s = max(s, scales[p, h])
                    if s > scales[p, h]:
                        codes[p, h, :row] = e4m3_of(number[codes[p, h, :row]] * (scales[p, h] / s))
                scales[p, h] = s
                for i, values in zip(put, part):
                    codes[p, h, row + i] = e4m3_of(np.where(np.isfinite(values), values, np.nan) / s)
            t += n
    return codes, scales, reported


@pytest.mark.parametrize("page,heads,dim,dtype", [
    (16, 2, 64, "float16"), (64, 1, 256, "bfloat16"), (128, 2, 256, "float16"), (24, 1, 72, "bfloat16"),
    (256, 1, 128, "float16"), (8, 3, 128, "bfloat16")])
@pytest.mark.parametrize("held", [0, 5])
@pytest.mark.parametrize("infinite", [False, True])
def test_cache_takes_each_token_by_its_own_slot(page, heads, dim, dtype, held, infinite):
    from mlc_vla import paged

    rng = np.random.default_rng(page + dim + held)
    new, pages = [page + 3, 2 * page, 4, 3, 1], 12
    lens = [held, held, 0, held, page - 1]
    cu = np.concatenate([[0], np.cumsum(new)])
    slots, at = [], 0
    for r, n in enumerate(new):
        first = lens[r]
        for p in range(first, first + n):
            slots.append((at + p // page) * page + p % page)
        at += -(-(first + n) // page)
    assert at <= pages
    right, slots = list(slots), np.array(slots)
    slots[2] = -1                       # within a page
    slots[cu[1]] = -1                   # the first token of a page's run
    slots[cu[1] + 2] = slots[cu[1] + 3]   # another's row
    slots[cu[2] - 1] = -1               # the last token of a page's run
    slots[cu[2] + 1] += page            # its row of another page
    slots[cu[3]:cu[4]] = -1             # a request that was not admitted
    x = [rng.standard_normal((cu[-1], heads, dim)) * np.exp(rng.standard_normal((cu[-1], heads, 1)))
         for _ in range(2)]
    for y in x:
        y[[2, cu[1], cu[2] - 1]] *= 1000.0  # what is left out must not count for the scale
        if infinite:
            y[1, 0, 3], y[cu[1] + 1, 0, 0], y[cu[1], 0, 0] = np.inf, np.nan, -np.inf
    x = [torch.as_tensor(y).to(getattr(torch, dtype)).cuda() for y in x]
    codes = rng.integers(0, 0x7E, (2, pages, heads, page, dim)).astype(np.uint8)
    scales = 2.0 ** rng.integers(-12, -6, (2, pages, heads))
    c = paged.KVCache8(*(torch.as_tensor(a).cuda().view(torch.float8_e4m3fn) for a in codes),
                       *(torch.as_tensor(a).float().cuda() for a in scales))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.write_kv(c, *x, dev(cu), dev(lens), dev(slots), max_new=max(new), err=err)
    for y, got, got_scale, a, b in zip(x, (c.k, c.v), (c.k_scale, c.v_scale), codes, scales):
        want, want_scale, reported = joined(a, b, y.double().cpu().numpy(), cu, lens, slots, page)
        assert reported and int(err.item()) == 19
        assert np.array_equal(got_scale.cpu().double().numpy(), want_scale)
        got = got.view(torch.uint8).cpu().numpy()
        nan = (got & 0x7F) == 0x7F
        assert np.array_equal(nan, (want & 0x7F) == 0x7F)
        assert np.array_equal(got[~nan], want[~nan])
    # all in their places: nothing is reported
    err.zero_()
    paged.write_kv(c, *x, dev(cu), dev(lens), dev(right), max_new=max(new), err=err)
    assert int(err.item()) == 0


@pytest.mark.parametrize("most", [0, 1, 1000])
def test_cache_writes_whatever_the_launch_was_sized_for(most):
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    k, v = (torch.as_tensor(rng.standard_normal((37, 2, 64))).half().cuda() for _ in range(2))
    cu, lens, slots = dev([0, 20, 37]), dev([0, 0]), dev(np.r_[16:36, 48:65])
    got, want = ([t.zero_() for t in paged.KVCache8.empty(6, 16, 2, 64)] for _ in range(2))
    paged.write_kv(paged.KVCache8(*got), k, v, cu, lens, slots, max_new=most)
    paged.write_kv(paged.KVCache8(*want), k, v, cu, lens, slots)
    paged.check()
    for g, w in zip(got, want):
        assert w.view(torch.uint8).any()
        assert torch.equal(g.view(torch.uint8), w.view(torch.uint8))


# ---- attention over the cache ---------------------------------------------------------------------

@pytest.mark.parametrize("batch", [1, 3, 193, 1000])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 1, 256, 64), (4, 2, 128, 16), (40, 2, 64, 8),
                                                     (3, 1, 72, 16)])
def test_paged_batch_without_any_token(batch, heads, kv_heads, dim, page):
    from mlc_vla import paged

    c = paged.KVCache8.empty(2, page, kv_heads, dim)
    for t in c:
        t.view(torch.uint8).fill_(0x7F)
    table = torch.full((batch, 3), -1, dtype=torch.int32, device="cuda")
    q = torch.ones((batch, heads, dim), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    paged.attention_paged(q, c, table, dev(np.zeros(batch, np.int32)), out=out)
    paged.check()
    assert not out.any()
    # the same without a token but in the last request
    lens = np.zeros(batch, np.int32)
    lens[-1] = 1
    c.k.view(torch.uint8).zero_()
    c.v.view(torch.uint8).fill_(0x38)  # 1.0
    c.k_scale.fill_(1.0)
    c.v_scale.fill_(0.5)
    table[-1] = 1
    paged.attention_paged(q, c, table, dev(lens), out=out)
    paged.check()
    assert not out[:-1].any() and (out[-1] == 0.5).all()


# ---- attention over prompts, and both ---------------------------------------------------------------

def filled_cache(rng, lens, page, heads, dim):
    """A cache of random codes in which requests hold `lens` tokens, with its table."""
    from mlc_vla import paged

    counts = [-(-n // page) for n in lens]
    order = rng.permutation(sum(counts) + 2)
    table, at = np.full((len(lens), max(counts)), -1), 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        at += n
    codes = [rng.integers(0, 256, (len(order), heads, page, dim)).astype(np.uint8) for _ in range(2)]
    for x in codes:
        x[(x & 0x7F) == 0x7F] = 0
    return paged.KVCache8(*(torch.as_tensor(x).cuda().view(torch.float8_e4m3fn) for x in codes),
                          *(torch.full((len(order), heads), 2.0 ** -7, device="cuda")
                            for _ in range(2))), table


@pytest.mark.parametrize("code", [1, 18, 1000])
def test_a_recorded_error_does_not_reach_later_calls(code):
    """`err` keeps the first code; waits that take long must not give up at one that is there already."""
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(0)

    def rows(*shape):
        return torch.randn(shape, generator=g, device="cuda").half()

    new, held = [300, 20, 700], [3800, 10, 0]
    cu_q, cu_k = dev(np.cumsum([0] + new)), dev(np.cumsum([0] + [a + b for a, b in zip(new, held)]))
    rng = np.random.default_rng(0)
    for heads, kv_heads, dim in ((4, 2, 128), (8, 1, 256), (2, 2, 64)):
        q, k, v = rows(1020, heads, dim), rows(4830, kv_heads, dim), rows(4830, kv_heads, dim)
        odd = v.clone()
        odd[4099, :, 5] = float("inf")  # the last key of the first request, seen by its last query
        lens = [3000, 5, 900, 129]
        c, table = filled_cache(rng, lens, 16, kv_heads, dim)
        qd = rows(4, heads, dim)
        for values in (v, odd):
            got = []
            for first in (0, code):
                err = dev([first])
                got.append((paged.attention_prompt(q, k, values, cu_q, cu_k, err=err),
                            paged.attention_paged(qd, c, dev(table), dev(lens), err=err)))
                assert int(err.item()) == first
            for a, b in zip(*got):
                assert torch.equal(a.nan_to_num(), b.nan_to_num())
                assert torch.equal(a.isnan(), b.isnan())
            clean = torch.isfinite(got[1][0])
            if values is odd:
                assert not clean[299, :, 5].any()
                clean[299, :, 5] = True
            assert clean.all() and torch.isfinite(got[1][1]).all()


@pytest.mark.parametrize("dim,page", [(128, 16), (256, 64), (64, 8)])
def test_a_bad_page_does_not_reach_other_requests(dim, page):
    from mlc_vla import paged

    rng = np.random.default_rng(dim)
    lens = [2000, 700, 1, 4000, 333] * 4
    c, table = filled_cache(rng, lens, page, 1, dim)
    q = torch.as_tensor(rng.standard_normal((20, 8, dim))).half().cuda()
    clean = paged.attention_paged(q, c, dev(table), dev(lens))
    paged.check()
    bad = table.copy()
    bad[3, 5], bad[8, 0] = len(c.k), -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = paged.attention_paged(q, c, dev(bad), dev(lens), err=err)
    assert int(err.item()) == 19
    good = [r for r in range(20) if r not in (3, 8)]
    assert torch.equal(out[good], clean[good])


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 1, 256, "float16"), (4, 2, 128, "bfloat16"),
                                                      (16, 1, 64, "float16"), (3, 3, 128, "float16")])
@pytest.mark.parametrize("new,held,prefix", [
    ([200], [69900], None), ([1500, 3, 260], [0, 20000, 4100], None), ([900, 700], [0, 0], [400, 768]),
    ([100], [5], None)])
def test_values_that_are_no_numbers_reach_their_rows_only(heads, kv_heads, dim, dtype, new, held, prefix):
    """Where some rows of a tile see such a value and others do not: the others, and the other
    dimensions, keep their bits, however long the request is."""
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(1)
    cu_q, cu_k = np.cumsum([0] + new), np.cumsum([0] + [a + b for a, b in zip(new, held)])

    def rows(n, h):
        return torch.randn((n, h, dim), generator=g, device="cuda").to(getattr(torch, dtype))

    q, k, v = rows(cu_q[-1], heads), rows(cu_k[-1], kv_heads), rows(cu_k[-1], kv_heads)

    def attend(values):
        out = paged.attention_prompt(q, k, values, dev(cu_q), dev(cu_k),
                                     prefix_lens=None if prefix is None else dev(prefix))
        paged.check()
        return out

    clean, inf = attend(v), float("inf")
    assert torch.isfinite(clean).all()
    odd = v.clone()
    marks = []  # request, key, dimension, value
    for r, (n, h) in enumerate(zip(new, held)):
        marks += [(r, h + j, d, x) for j, d, x in ((n - 1, 0, inf), (n // 2, 5, -inf), (n // 3, 33, inf),
                                                   (2 * n // 3, 33, -inf), (n // 2, dim - 1, inf - inf))]
    marks.append((0, 0, 40, -inf))  # seen by every row of the first request
    for r, j, d, x in marks:
        odd[cu_k[r] + j, :, d] = x
    got, want = attend(odd), clean.float()
    for r, n in enumerate(new):
        lk = n + held[r]
        sees = torch.arange(n, device="cuda") + held[r] + 1
        if prefix is not None:
            sees = sees.clamp_min(prefix[r]).clamp_max(lk)
        for m, j, d, x in marks:
            if m == r:
                want[cu_q[r]:cu_q[r + 1], :, d] += torch.where(sees > j, x, 0.0)[:, None]
    finite = torch.isfinite(want)
    assert torch.equal(got[finite], clean[finite])
    # an infinity whose weight is no longer a number above zero gives NaN
    rest = got[~finite].float()
    assert ((rest == want[~finite]) | rest.isnan()).all()
    assert (rest.isnan() | ~want[~finite].isnan()).all()


# ---- small weights --------------------------------------------------------------------------------

def sink_error(out, q, k, v, dtype, step):
    """Largest error, in parts of its bound, of rows [queries, dim] that see all keys: rounding of the
    result and of the weights (u each, and of their sum), fp32 logits (2^-23 of each product; 2^-21 of
    the logit and 2^-20 for the exponential, in numerator and denominator), the fp32 sum; and `step`,
    what a weight below the normal range of its form loses at most, in units of the row's largest."""
    q, k, v = q.double(), k.double(), v.double()
    n, dim = k.shape
    s = q @ k.T * dim ** -0.5
    p = torch.softmax(s, -1)
    o, spread = p @ v, p @ v.abs()
    size = (q.abs() @ k.abs().T).amax(1, True) * dim ** -0.5
    u = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]
    logit = 2 * (dim * 2.0 ** -23 * size + 2.0 ** -21 * s.abs().amax(1, True) + 2.0 ** -20)
    tol = (u * o.abs() + (2 * u + logit + n * 2.0 ** -23) * spread + n * step * v.abs().max()
           + 2.0 ** -25)  # half a step of fp16's results below its normal range
    return float(((out.double() - o).abs() / tol).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,dim,new", [(64, 256, 150), (32, 128, 600), (16, 64, 1200)])
@pytest.mark.parametrize("gap", [15, 20, 23, 25])
def test_prompt_one_key_above_all_others(heads, dim, new, dtype, gap):
    """A first key `gap` bits above the rest whose value is zero: the result is what thousands of
    small weights add up to. In fp16 weights are held in steps of 2^-24 below 2^-14, lifted by 2^7.
    Requests enough that a CTA takes all keys of some tiles."""
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(gap + dim)
    batch, n, kv_heads = 4, 4200, 8
    q = torch.randn((batch * new, heads, dim), generator=g, device="cuda")
    k = torch.randn((batch * n, kv_heads, dim), generator=g, device="cuda") * 0.5
    v = 1.0 + 0.1 * torch.randn((batch * n, kv_heads, dim), generator=g, device="cuda")
    q[:, :, 0], k[:, :, 0], k[::n], v[::n] = 8.0, 0.0, 0.0, 0.0
    k[::n, :, 0] = gap * np.log(2.0) * dim ** 0.5 / 8.0
    q, k, v = (x.to(getattr(torch, dtype)) for x in (q, k, v))
    out = paged.attention_prompt(q, k, v, dev(np.arange(batch + 1) * new), dev(np.arange(batch + 1) * n),
                                 prefix_lens=dev([n] * batch))
    paged.check()
    step = 2.0 ** -32 if dtype == "float16" else 0.0
    for r in range(batch):
        rows, keys = slice(r * new, (r + 1) * new), slice(r * n, (r + 1) * n)
        worst = max(sink_error(out[rows, h], q[rows, h], k[keys, h // (heads // kv_heads)],
                               v[keys, h // (heads // kv_heads)], dtype, step) for h in range(heads))
        assert worst <= 1.0, worst


@pytest.mark.parametrize("heads,kv_heads,dim,page,batch", [
    (8, 1, 256, 64, 320), (4, 1, 128, 16, 640), (8, 1, 64, 8, 640), (3, 1, 64, 128, 900),
    (16, 1, 128, 32, 320), (12, 1, 256, 16, 200)])
@pytest.mark.parametrize("gap", [18, 22, 23, 25])
def test_paged_one_key_above_all_others(heads, kv_heads, dim, page, batch, gap):
    """The same over the cache, where weights are held as sums of e4m3 parts, in steps of 2^-29 of the
    largest (half of that is lost at most). Many requests on the same pages, so that a CTA takes all
    keys of some of them. Values of page 0, the sink's, are zero."""
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(gap + dim)
    n, pages = 16384 + 5, -(-(16384 + 5) // page)
    k = (4.0 * torch.randn((pages, 1, page, dim), generator=g, device="cuda")).to(torch.float8_e4m3fn)
    v = torch.randint(0x58, 0x60, (pages, 1, page, dim), generator=g, device="cuda",
                      dtype=torch.uint8).view(torch.float8_e4m3fn)  # 16 to 30
    k.view(torch.uint8)[..., 0] = 0
    k.view(torch.uint8)[0, 0, 0] = 0
    v.view(torch.uint8)[0, 0, 0] = 0
    k[0, 0, 0, 0] = 256.0
    k_scale = torch.full((pages, 1), 2.0 ** -3, device="cuda")
    v_scale = torch.full((pages, 1), 2.0 ** -5, device="cuda")
    q = torch.randn((batch, heads, dim), generator=g, device="cuda")
    q[:, :, 0] = gap * np.log(2.0) * dim ** 0.5 / 32.0
    q = q.half()
    c = paged.KVCache8(k, v, k_scale, v_scale)
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, pages).contiguous()
    out = paged.attention_paged(q, c, table, dev([n] * batch))
    paged.check()
    kn, vn = (x.double().reshape(-1, dim)[:n] * s for x, s in ((k, 2.0 ** -3), (v, 2.0 ** -5)))
    rows, got = q.reshape(-1, dim), out.reshape(-1, dim)
    for a in range(0, len(rows), 640):
        worst = sink_error(got[a:a + 640], rows[a:a + 640], kn, vn, "float16", 2.0 ** -30)
        assert worst <= 1.0, worst


@pytest.mark.parametrize("heads,dim,page", [(8, 256, 64), (4, 128, 16), (16, 64, 32)])
@pytest.mark.parametrize("loud", [8, 14])
def test_paged_loud_page(heads, dim, page, loud):
    """A page whose scale is 2^`loud` above the others, because of one token of no weight: the weights
    of the others are taken relative to the page's scale and have as many bits less."""
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(loud + dim)
    batch, n = 640, 2048
    pages = n // page
    k = (8.0 * torch.randn((pages, 1, page, dim), generator=g, device="cuda")).to(torch.float8_e4m3fn)
    v = torch.randint(0x58, 0x60, (pages, 1, page, dim), generator=g, device="cuda",
                      dtype=torch.uint8).view(torch.float8_e4m3fn)
    k.view(torch.uint8)[..., 0] = 0
    k[1, 0, 3] = 0.0
    k[1, 0, 3, 0] = -448.0
    v[1] = 0.0
    v[1, 0, 3] = 448.0
    k_scale = torch.full((pages, 1), 2.0 ** -3, device="cuda")
    v_scale = torch.full((pages, 1), 2.0 ** -5, device="cuda")
    v_scale[1] = 2.0 ** (loud - 5)
    q = torch.randn((batch, heads, dim), generator=g, device="cuda")
    q[:, :, 0] = 60.0 * dim ** 0.5 / 56.0  # the loud token's logit: -60
    q = q.half()
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, pages).contiguous()
    out = paged.attention_paged(q, paged.KVCache8(k, v, k_scale, v_scale), table, dev([n] * batch))
    paged.check()
    kn = k.double().reshape(-1, dim) * 2.0 ** -3
    vn = (v.double() * v_scale.double()[:, :, None, None]).reshape(-1, dim)
    quiet = vn.clone()
    quiet[page + 3] = 0.0  # of weight e^-55 and less: not in the bound's largest value
    rows, got = q.reshape(-1, dim), out.reshape(-1, dim)
    for a in range(0, len(rows), 640):
        worst = sink_error(got[a:a + 640], rows[a:a + 640], kn, quiet, "float16", 2.0 ** (loud - 30))
        assert worst <= 1.0, worst


# ---- outputs and gradients --------------------------------------------------------------------------

def test_out_apart_from_the_inputs():
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(0)
    fused = torch.randn((300, 20, 64), generator=g, device="cuda").half()
    q, k, v, room = fused[:, :8], fused[:, 8:10], fused[:, 10:12], fused[:, 12:]
    cu = dev([0, 100, 300])
    want = paged.attention_prompt(q, k, v, cu)
    paged.attention_prompt(q, k, v, cu, out=room)  # between the rows of its inputs
    assert torch.equal(room, want)
    dense = torch.randn((301, 8, 64), generator=g, device="cuda").half()
    for out, query in ((q, q), (dense[1:], dense[:300]), (dense[:300], dense[1:])):
        with pytest.raises(ValueError, match="overlap"):
            paged.attention_prompt(query, k, v, cu, out=out)
    with pytest.raises(ValueError, match="overlap"):
        paged.attention_prompt(q, dense[:300], dense[:300].clone(), cu, out=dense[:300])
    # over the cache the result may replace the queries
    rng = np.random.default_rng(0)
    for dim in (64, 72):
        lens = [3000, 1, 700]
        c, table = filled_cache(rng, lens, 16, 2, dim)
        x = torch.randn((3, 8, dim), generator=g, device="cuda").half()
        want = paged.attention_paged(x, c, dev(table), dev(lens))
        assert torch.equal(paged.attention_paged(x, c, dev(table), dev(lens), out=x), want)
        paged.check()


def test_gradients_are_refused_where_they_are_asked_for():
    from mlc_vla import paged

    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn((20, h, 64), generator=g, device="cuda").half() for h in (4, 2, 2))
    cu = dev([0, 20])
    rng = np.random.default_rng(0)
    c, table = filled_cache(rng, [50] * 20, 16, 2, 64)
    calls = [lambda q, k, v, **kw: paged.attention_prompt(q, k, v, cu, **kw),
             lambda q, k, v, **kw: paged.attention_paged(q, c, dev(table), dev([50] * 20), **kw)]
    for call in calls:
        want = call(q, k, v)
        assert not want.requires_grad
        weight = torch.ones((), device="cuda", dtype=torch.float16, requires_grad=True)
        out = call(q * weight, k, v)
        assert torch.equal(out, want)  # forward as ever
        with pytest.raises(RuntimeError, match="not implemented"):
            out.float().sum().backward()
        room = torch.empty_like(q)
        with pytest.raises(RuntimeError, match="no_grad"):
            call(q * weight, k, v, out=room)
        with torch.no_grad():
            assert not call(q * weight, k, v).requires_grad
            call(q * weight, k, v, out=room)
        assert torch.equal(room, want)
    out = calls[0](q, k, v.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="not implemented"):
        out.float().sum().backward()
    with torch.inference_mode():
        assert torch.equal(calls[0](q, k, v), calls[0](q.clone(), k, v))


def test_calls_keep_no_memory():
    """Workspaces return to the allocator, whatever streams the calls were on."""
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    c, table = filled_cache(rng, [3000, 10], 16, 1, 256)
    x = torch.randn((200, 8, 256), device="cuda").half()
    args = (x[:2], c, dev(table), dev([3000, 10]))
    cu = dev([0, 200])
    want = paged.attention_paged(*args), paged.attention_prompt(x, x[:, :1], x[:, 1:2], cu)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(4):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = paged.attention_paged(*args), paged.attention_prompt(x, x[:, :1], x[:, 1:2], cu)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got
    assert torch.cuda.memory_allocated() == before
    paged.check()
