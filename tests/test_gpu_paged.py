"""GPU: block tables and slot maps, the 8-bit page cache, attention over packed prompts and over the
cache (``mlc_vla.paged``) against 64-bit restatements, at the sizes and masks where they can go
wrong. Tolerances come from the error bounds in ``paged_ref``."""

import numpy as np
import pytest

import paged_ref as R

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

NAN_CODE = 0x7F


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).cuda()


def num(t):
    return t.float().cpu().numpy().astype(np.float64)


def close(got, want, tol):
    got = num(got)
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) / np.maximum(tol, 1e-300))
    assert worst <= 1.0, f"error {worst:.3f} of the bound"


def rows(rng, *shape, dtype):
    x = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[:-1] + (1,)))
    return torch.as_tensor(x).to(getattr(torch, dtype)).cuda()


# ---- block tables and slots -----------------------------------------------------------------------

def run_slots(kv, new, page, columns, num_tokens, free, free_pos=0, seed=0, rows_of=None):
    from mlc_vla import paged

    rng = np.random.default_rng(seed)
    pages = len(free) + sum(-(-n // page) for n in kv if n > 0)
    order = rng.permutation(pages)
    table = np.full((len(kv), columns), -1)
    at = len(free)
    for r, n in enumerate(kv):
        c = min(columns, -(-max(n, 0) // page))
        table[r, :c] = order[at:at + c]
        at += -(-max(n, 0) // page)
    free = order[:len(free)]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    wide = torch.full((len(kv), columns + 3), -7, dtype=torch.int32, device="cuda")
    t = wide[:, :columns]
    t.copy_(dev(table))
    s = paged.build_slots(dev(kv), dev(new), t, dev(free), dev([free_pos]), page, num_tokens, err=err)
    assert (wide[:, columns:] == -7).all()
    want = R.build_slots(kv, new, table, free, free_pos, page, num_tokens)
    got = [t, s.cu_seqlens, s.positions, s.slot_mapping, s.kv_lens, s.free_pos]
    return [x.cpu().numpy() for x in got], want, int(err.item())


@pytest.mark.parametrize("batch,held,most,page", [
    (1, 0, 1, 16), (1, 15, 1, 16), (1, 16, 1, 16), (5, 40, 7, 1), (33, 100, 1, 64),
    (64, 300, 70, 24), (513, 90, 40, 16), (2000, 30, 5, 8), (7, 0, 3001, 128)])
def test_slots_against_the_definition(batch, held, most, page):
    rng = np.random.default_rng(batch * 7 + page)
    kv = rng.integers(0, held + 1, batch)
    new = rng.integers(0, most + 1, batch)
    new[0] = most
    if batch > 2:
        kv[1], new[1] = 0, 0
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(kv, new))
    columns = max(-(-(a + b) // page) for a, b in zip(kv, new)) + 1
    got, want, err = run_slots(kv, new, page, columns, int(new.sum()) + 5, range(need + 4), 2)
    assert err == 0
    for g, w in zip(got, want):
        assert np.array_equal(g.ravel(), np.ravel(w))


def test_slots_of_a_pool_that_runs_out():
    # requests 0 and 1 fit, 2 does not, 3 needs no page and fits, 4 no more
    kv, new = [0, 8, 0, 3, 0], [16, 9, 40, 5, 1]
    got, want, err = run_slots(kv, new, 8, 6, 71, range(5))
    for g, w in zip(got, want):
        assert np.array_equal(g.ravel(), np.ravel(w))
    assert err == 18 and list(got[4]) == [16, 17, 0, 8, 0] and got[5][0] == 4


def test_slots_of_a_request_longer_than_its_row():
    got, want, err = run_slots([30, 0], [3, 4], 8, 4, 7, range(6))
    for g, w in zip(got, want):
        assert np.array_equal(g.ravel(), np.ravel(w))
    assert err == 17 and list(got[4]) == [30, 4]


def test_slots_errors_and_empty_batch():
    from mlc_vla import _lib, paged

    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(8, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = paged.build_slots(dev([-3, 0]), dev([2, 1]), table, free, z[:1], 8, 3, err=err)
    assert int(err.item()) == 16 and s.slot_mapping.tolist() == [0, 1, 8]
    err.zero_()
    s = paged.build_slots(z, dev([2, 5]), table, free, z[:1], 8, 4, err=err)  # 7 tokens, room for 4
    assert int(err.item()) == 16 and s.cu_seqlens.tolist() == [0, 2, 7]
    # the flag of the device where no `err` is given
    paged.build_slots(z, dev([1, 1]), table, dev([99] * 4), z[:1], 8, 2, num_pages=8)
    with pytest.raises(_lib.Pi0Error):
        paged.check()
    paged.check()
    s = paged.build_slots(z[:0], z[:0], table[:0], free, z[:1], 8, 3)
    assert s.cu_seqlens.tolist() == [0] and s.slot_mapping.tolist() == [-1] * 3
    assert s.free_pos.tolist() == [0]


# ---- the cache ------------------------------------------------------------------------------------

def fresh_cache(pages, heads, page, dim, code=NAN_CODE):
    from mlc_vla import paged

    c = paged.KVCache8.empty(pages, page, heads, dim)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(code)
    for t in (c.k_scale, c.v_scale):
        t.fill_(float("nan"))
    return c


def same_numbers(got, want):
    got = num(got)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got, nan=0.0), np.nan_to_num(want, nan=0.0))


class Requests:
    """Requests on one cache, appended to step by step, beside the restatement's copy."""

    def __init__(self, batch, pages, heads, page, dim, columns, seed):
        self.rng = np.random.default_rng(seed)
        self.page, self.heads, self.dim = page, heads, dim
        self.cache = fresh_cache(pages, heads, page, dim)
        self.table = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")
        self.free = dev(self.rng.permutation(pages))
        self.pos = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.want = [(num(c), num(s)) for c, s in ((self.cache.k, self.cache.k_scale),
                                                   (self.cache.v, self.cache.v_scale))]

    def append(self, new, dtype, change=None, max_new=None):
        from mlc_vla import paged

        total = int(np.sum(new))
        s = paged.build_slots(self.lens, dev(new), self.table, self.free, self.pos, self.page, total)
        x = [rows(self.rng, total, self.heads, self.dim, dtype=dtype) for _ in range(2)]
        if change is not None:
            change(x)
        paged.write_kv(self.cache, *x, s.cu_seqlens, self.lens, s.slot_mapping, max_new=max_new)
        cu, slots, old = (t.cpu().numpy() for t in (s.cu_seqlens, s.slot_mapping, self.lens))
        self.want = [R.write_kv(c, sc, num(y), cu, old, slots, self.page)
                     for (c, sc), y in zip(self.want, x)]
        self.lens, self.pos = s.kv_lens, s.free_pos
        paged.check()

    def compare(self):
        for (codes, scales), c, s in zip(self.want, (self.cache.k, self.cache.v),
                                         (self.cache.k_scale, self.cache.v_scale)):
            same_numbers(s, scales)
            same_numbers(c, codes)


@pytest.mark.parametrize("page,heads,dim,dtype", [
    (16, 1, 256, "float16"), (64, 2, 128, "bfloat16"), (32, 3, 64, "float16"),
    (128, 1, 256, "bfloat16"), (24, 2, 72, "float16"), (1, 1, 16, "bfloat16"), (8, 4, 8, "float16"),
    (256, 1, 64, "bfloat16")])
def test_cache_after_prompts_and_single_tokens(page, heads, dim, dtype):
    columns = 4 + 350 // page  # room for the longest request of any page size
    r = Requests(4, 4 * columns, heads, page, dim, columns, page + dim)
    r.append([1, 0, page, 2 * page + 3], dtype)
    r.compare()
    for step in range(3):  # growing magnitudes: scales rise, codes are rounded again
        r.append([1, 1, 1, 1], dtype, lambda x: [y.mul_(4.0 ** step) for y in x], max_new=1)
        r.compare()
    r.append([5, 17, 0, 40], dtype, max_new=3)  # longer than the launch was sized for
    r.compare()


def test_cache_takes_what_has_no_code():
    r = Requests(2, 8, 2, 16, 64, 4, 3)

    def change(x):
        x[0][0, 0, 3], x[0][1, 1, 5], x[0][2, 0, 7] = float("inf"), float("nan"), float("-inf")
        x[1][:] = 0.0
        x[1][4, 1, 1] = 6e-8
    r.append([9, 4], "float16", change)
    r.compare()
    assert float(r.cache.v_scale[int(r.table[0, 0]), 0]) == 2.0 ** -64
    r.append([4, 4], "float16")
    r.compare()
    b = Requests(1, 2, 1, 16, 64, 2, 4)  # beyond what 2^-64 and fp16 reach
    b.append([3], "bfloat16", lambda x: (x[0].mul_(1e-30), x[1].mul_(1e36)))
    b.compare()


def test_cache_leaves_out_tokens_without_a_slot_and_reads_strided_rows():
    from mlc_vla import paged

    c = fresh_cache(4, 2, 16, 64)
    before = c.k.view(torch.uint8).clone()
    cu, lens = dev([0, 3, 8]), dev([0, 0])
    fused = rows(np.random.default_rng(0), 8, 6, 64, dtype="float16")
    k, v = fused[:, 2:4], fused[:, 4:6]
    slots = dev([-1, -1, -1, 32, 33, 34, 35, 36])
    paged.write_kv(c, k, v, cu, lens, slots)
    paged.check()
    changed = (c.k.view(torch.uint8) != before).flatten(1).any(1).tolist()
    assert changed == [False, False, True, False]
    want = R.write_kv(np.zeros((4, 2, 16, 64)), np.zeros((4, 2)), num(k), [0, 3, 8], [0, 0],
                      slots.tolist(), 16)
    same_numbers(c.k[2, :, :5], want[0][2, :, :5])
    # a slot that is not its token's row, and one outside the pool
    for bad in (33, 16 * 4):
        paged.write_kv(c, k[:1], v[:1], dev([0, 1]), dev([0]), dev([bad]))
        with pytest.raises(RuntimeError):
            paged.check()


# ---- attention over prompts -----------------------------------------------------------------------

def packed(new, held):
    return np.cumsum([0] + list(new)), np.cumsum([0] + [a + b for a, b in zip(new, held)])


def prompt_case(new, held, prefix, heads, kv_heads, dim, dtype, seed=0, pad=0):
    rng = np.random.default_rng(seed)
    cu_q, cu_k = packed(new, held)
    q = rows(rng, cu_q[-1] + pad, heads, dim, dtype=dtype)
    k = rows(rng, cu_k[-1] + pad, kv_heads, dim, dtype=dtype)
    v = rows(rng, cu_k[-1] + pad, kv_heads, dim, dtype=dtype)
    return q, k, v, cu_q, cu_k, prefix


def check_prompt(case, dtype, scale=None, **kw):
    from mlc_vla import paged

    q, k, v, cu_q, cu_k, prefix = case
    out = paged.attention_prompt(q, k, v, dev(cu_q), dev(cu_k),
                                 prefix_lens=None if prefix is None else dev(prefix), scale=scale, **kw)
    paged.check()
    n = int(cu_q[-1])
    want, tol = R.attention_prompt(num(q)[:n], num(k), num(v), cu_q, cu_k,
                                   [0] * (len(cu_q) - 1) if prefix is None else prefix,
                                   q.shape[2] ** -0.5 if scale is None else scale, dtype)
    close(out[:n], want, tol)
    assert not out[n:].any()
    return out


SHAPES = [(8, 1, 256, "float16"), (8, 1, 256, "bfloat16"), (4, 2, 128, "bfloat16"),
          (4, 1, 64, "float16"), (5, 1, 128, "float16"), (3, 3, 256, "float16"),
          (2, 2, 64, "bfloat16"), (16, 1, 128, "float16"), (6, 2, 256, "bfloat16"),
          (2, 1, 72, "float16"), (3, 1, 16, "bfloat16")]


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", SHAPES)
def test_prompt_causal_ragged(heads, kv_heads, dim, dtype):
    new = [1, 0, 2, 31, 129, 64, 200]
    check_prompt(prompt_case(new, [0] * 7, None, heads, kv_heads, dim, dtype, seed=dim + heads, pad=3),
                 dtype)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", SHAPES)
def test_prompt_prefix_and_earlier_keys(heads, kv_heads, dim, dtype):
    new, held = [5, 70, 1, 130, 33], [0, 61, 300, 127, 1]
    prefix = [3, 100, 0, 257, 34]  # inside the new tokens, reaching into them, none, all, all
    check_prompt(prompt_case(new, held, prefix, heads, kv_heads, dim, dtype, seed=dim), dtype)


@pytest.mark.parametrize("dim", [16, 64, 128, 256])
def test_prompt_rows_that_see_nothing(dim):
    # fewer keys than queries: the first ones see none; a request without keys; prefix beyond them
    new, held, prefix = [40, 7, 150, 3], [-30, -7, -149, -1], [0, 0, 0, 50]
    out = check_prompt(prompt_case(new, held, prefix, 4, 2, dim, "float16", seed=1), "float16")
    assert not out[:30].any() and not out[40:47].any()


@pytest.mark.parametrize("n", [127, 128, 129, 255, 256, 257, 385, 640])
@pytest.mark.parametrize("heads,dim", [(1, 128), (8, 256), (2, 64)])
def test_prompt_around_tile_edges(n, heads, dim):
    rng = np.random.default_rng(n)
    check = prompt_case([n], [0], None, heads, 1, dim, "bfloat16", seed=n)
    q, k, v, cu_q, cu_k, _ = check
    from mlc_vla import paged

    out = paged.attention_prompt(q, k, v, dev(cu_q))
    paged.check()
    some = sorted(set(rng.integers(0, n, 12)) | {0, n - 1, n // 2})
    want, tol = [], []
    for i in some:  # a single query with its leading keys
        w, t = R.attention_prompt(num(q)[i:i + 1], num(k)[:i + 1], num(v)[:i + 1], [0, 1], [0, i + 1],
                                  [0], dim ** -0.5, "bfloat16")
        want.append(w[0])
        tol.append(t[0])
    close(out[some], np.array(want), np.array(tol))


@pytest.mark.parametrize("new,held,prefix,heads,kv_heads,dim,dtype", [
    ([4096], [0], None, 16, 4, 128, "bfloat16"), ([3000, 1111], [0, 777], None, 8, 4, 64, "float16"),
    ([968, 700, 850, 901] * 3, [0] * 12, [768] * 12, 8, 1, 256, "float16"),
    ([200, 33, 170], [4000, 2500, 3777], None, 16, 4, 128, "float16"),
    ([1, 1, 1], [5000, 3, 9000], None, 8, 1, 256, "bfloat16"),
    ([2500, 1], [0, 1], [2500, 1], 5, 1, 128, "float16")])
def test_prompt_many_tiles(new, held, prefix, heads, kv_heads, dim, dtype):
    """Enough tiles that a CTA works on several and shares some with others."""
    from mlc_vla import paged

    q, k, v, cu_q, cu_k, prefix = prompt_case(new, held, prefix, heads, kv_heads, dim, dtype, seed=dim)
    out = paged.attention_prompt(q, k, v, dev(cu_q), dev(cu_k),
                                 prefix_lens=None if prefix is None else dev(prefix))
    paged.check()
    rng = np.random.default_rng(0)
    kn, vn = num(k), num(v)
    for r in range(len(new)):
        first, n = cu_k[r], cu_k[r + 1] - cu_k[r]
        some = sorted(set(rng.integers(0, new[r], 24)) | {0, new[r] - 1})
        for i in some:  # one query with the keys it sees
            t = cu_q[r] + i
            sees = min(n, max(i + n - new[r] + 1, 0 if prefix is None else prefix[r]))
            want, tol = R.attention_prompt(num(q[t:t + 1]), kn[first:first + sees],
                                           vn[first:first + sees], [0, 1], [0, sees], [0],
                                           dim ** -0.5, dtype)
            close(out[t:t + 1], want, tol)
    # every row, against a softmax in 64 bits on the GPU, within the bound of paged_ref._attend
    group, worst = heads // kv_heads, 0.0
    for r in range(len(new)):
        n, i = cu_k[r + 1] - cu_k[r], torch.arange(new[r], device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= i + n - new[r]) | (j < (0 if prefix is None else prefix[r]))
        for h in range(heads):
            kh, vh = (x[cu_k[r]:cu_k[r + 1], h // group].double() for x in (k, v))
            s = q[cu_q[r]:cu_q[r + 1], h].double() @ kh.T * dim ** -0.5
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            o, spread = p @ vh, p @ vh.abs()
            size = (q[cu_q[r]:cu_q[r + 1], h].double().abs() @ kh.abs().T).amax(1, True) * dim ** -0.5
            logit = 2 * (dim * 2.0 ** -23 * size + 2.0 ** -21 * s.abs().amax(1, True) + 2.0 ** -20)
            u = R.UNIT[dtype]
            tol = (u * o.abs() + (2 * u + logit + n * 2.0 ** -23) * spread
                   + n * 2.0 ** -25 * vh.abs().max() + 2.0 ** -24)
            worst = max(worst, float(((out[cu_q[r]:cu_q[r + 1], h].double() - o).abs() / tol).max()))
    assert worst <= 1.0, worst


def test_prompt_large_logits_and_scales():
    for scale in (1.0, 0.01, -0.3, 0.0):
        check_prompt(prompt_case([90, 33], [0, 100], None, 4, 1, 128, "float16", seed=5), "float16",
                     scale=scale)
    case = prompt_case([300], [0], None, 2, 1, 256, "bfloat16", seed=6)
    case[1].mul_(20.0)  # near one-hot rows, running maxima that jump
    check_prompt(case, "bfloat16")


def test_prompt_strided_rows_out_and_stream():
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    fused = rows(rng, 150, 12, 128, dtype="float16")  # q, k and v of one projection
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    wide = torch.full((150, 16, 128), 7.0, dtype=torch.float16, device="cuda")
    cu = np.array([0, 20, 150])
    out = check_prompt((q, k, v, cu, cu, None), "float16", out=wide[:, 4:12])
    assert (wide[:, :4] == 7).all() and (wide[:, 12:] == 7).all()
    heads_first = fused.transpose(0, 1).contiguous().transpose(0, 1)  # [heads, tokens, dim] storage
    again = paged.attention_prompt(heads_first[:, :8], heads_first[:, 8:10], heads_first[:, 10:],
                                   dev(cu))
    assert torch.equal(again, out)
    cu_d = dev(cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = paged.attention_prompt(q, k, v, cu_d)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(third, out)


@pytest.mark.parametrize("heads,dim,dtype", [(8, 256, "float16"), (4, 128, "bfloat16"),
                                             (2, 64, "float16"), (2, 24, "float16")])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_prompt_unseen_keys_do_not_reach_a_row(heads, dim, dtype, what):
    from mlc_vla import paged

    q, k, v, cu, _, _ = prompt_case([60, 140, 50], [0, 0, 0], None, heads, 1, dim, dtype, seed=9, pad=4)
    clean = paged.attention_prompt(q, k, v, dev(cu))
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[150:152] = what      # inside the second request: rows 150.. see it
        t[200:201] = what      # the first key of the third request
        t[250:] = what         # behind the last request
    out = paged.attention_prompt(q, k2, v2, dev(cu))
    paged.check()
    assert torch.equal(out[:150], clean[:150])
    assert out[150:200].isnan().all() and out[200:250].isnan().all()
    only = v.clone()
    only[199] = what           # the last key of the second request, seen by its last query alone
    out = paged.attention_prompt(q, k, only, dev(cu))
    assert torch.equal(out[:199], clean[:199]) and torch.equal(out[200:], clean[200:])
    assert not torch.isfinite(out[199]).any()


def test_prompt_repeats_bit_for_bit():
    from mlc_vla import paged

    q, k, v, cu_q, cu_k, _ = prompt_case([700, 40, 968], [0, 500, 0], None, 8, 1, 256, "float16")
    a = paged.attention_prompt(q, k, v, dev(cu_q), dev(cu_k))
    for _ in range(3):
        assert torch.equal(a, paged.attention_prompt(q, k, v, dev(cu_q), dev(cu_k)))
    empty = paged.attention_prompt(q[:0], k[:0], v[:0], dev([0, 0]))
    assert empty.shape == (0, 8, 256)


# ---- attention over the cache ---------------------------------------------------------------------

def filled(rng, lens, page, heads, dim, spare=3, columns=None):
    """A cache whose requests hold `lens` tokens; everything else in it is NaN."""
    from mlc_vla import paged

    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = rng.permutation(pages)
    columns = columns or max(1, max(counts))
    table = np.full((len(lens), columns), -1)
    codes = [np.full((pages, heads, page, dim), np.nan) for _ in range(2)]
    scales = [np.full((pages, heads), np.nan) for _ in range(2)]
    at = 0
    for r, n in enumerate(lens):
        for c in range(counts[r]):
            p = order[at]
            at += 1
            table[r, c] = p
            m = min(page, n - c * page)
            for i in range(2):
                x = rng.standard_normal((heads, m, dim)) * np.exp(0.5 * rng.standard_normal((heads, m, 1)))
                amax = np.abs(x).max((1, 2))
                s = 2.0 ** np.ceil(np.log2(amax / 448.0))
                scales[i][p] = s
                codes[i][p, :, :m] = R.e4m3(x / s[:, None, None])
    c = paged.KVCache8(*(torch.as_tensor(x).float().cuda().to(torch.float8_e4m3fn) for x in codes),
                       *(torch.as_tensor(x).float().cuda() for x in scales))
    return c, table, [x * s[:, :, None, None] for x, s in zip(codes, scales)]


def check_paged(lens, page, heads, kv_heads, dim, dtype, seed=0, scale=None, columns=None):
    from mlc_vla import paged

    rng = np.random.default_rng(seed)
    c, table, (k, v) = filled(rng, lens, page, kv_heads, dim, columns=columns)
    q = rows(rng, len(lens), heads, dim, dtype=dtype)
    out = paged.attention_paged(q, c, dev(table), dev(lens), scale=scale)
    paged.check()
    want, tol = R.attention_paged(num(q), k, v, table, lens, dim ** -0.5 if scale is None else scale,
                                  dtype)
    close(out, want, tol)
    return q, c, table, out


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", SHAPES + [(40, 1, 128, "bfloat16"),
                                                               (64, 2, 256, "float16")])
@pytest.mark.parametrize("page", [16, 64, 24])
def test_paged_ragged(heads, kv_heads, dim, dtype, page):
    lens = [1, 0, page - 1, page, page + 1, 127, 128, 129, 700]
    check_paged(lens, page, heads, kv_heads, dim, dtype, seed=page + dim)


@pytest.mark.parametrize("page", [1, 8, 32, 128, 256, 384])
def test_paged_page_sizes(page):
    check_paged([257, 3, 640], page, 8, 1, 256, "bfloat16", seed=page)
    check_paged([257, 3, 640], page, 4, 2, 64, "float16", seed=page)


@pytest.mark.parametrize("batch,n", [(1, 5000), (2, 2500), (3, 1), (160, 130)])
def test_paged_few_and_many_requests(batch, n):
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(max(1, n // 2), n + 1, batch)]
    lens[-1] = n
    check_paged(lens, 64, 8, 1, 128, "bfloat16", seed=batch, columns=-(-n // 64) + 5)
    check_paged(lens[:5], 16, 2, 2, 256, "float16", seed=batch)


def test_paged_scales_and_magnitudes():
    from mlc_vla import paged

    for scale in (1.0, -0.2, 0.0):
        check_paged([300, 20], 32, 8, 2, 128, "float16", scale=scale)
    # pages of very different magnitude, and scales that are no powers of two
    rng = np.random.default_rng(2)
    c, table, (k, v) = filled(rng, [200, 90], 16, 1, 128)
    f = np.exp(rng.uniform(-12, 3, c.v_scale.shape)).astype(np.float32)
    c.v_scale.mul_(torch.as_tensor(f).cuda())
    g = np.exp(rng.uniform(-1, 1, c.k_scale.shape)).astype(np.float32)
    c.k_scale.mul_(torch.as_tensor(g).cuda())
    k = num(c.k) * num(c.k_scale)[:, :, None, None]
    v = num(c.v) * num(c.v_scale)[:, :, None, None]
    q = rows(rng, 2, 8, 128, dtype="float16")
    out = paged.attention_paged(q, c, dev(table), dev([200, 90]))
    want, tol = R.attention_paged(num(q), k, v, table, [200, 90], 128 ** -0.5, "float16")
    close(out, want, tol)


def test_paged_after_write_strides_stream_and_repeats():
    from mlc_vla import paged

    r = Requests(3, 40, 1, 64, 256, 12, 5)
    r.append([500, 1, 130], "float16")
    r.append([1, 1, 1], "float16", max_new=1)
    k, v = (c * s[:, :, None, None] for c, s in r.want)
    wide = rows(r.rng, 3, 16, 256, dtype="float16")
    q = wide[:, 4:12]
    out = paged.attention_paged(q, r.cache, r.table, r.lens)
    want, tol = R.attention_paged(num(q), k, v, r.table.cpu().numpy(), r.lens.tolist(), 1 / 16, "float16")
    close(out, want, tol)
    room = torch.full_like(wide, 3.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            paged.attention_paged(q, r.cache, r.table, r.lens, out=room[:, 8:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(room[:, 8:], out) and (room[:, :8] == 3).all()


def test_paged_in_a_graph_follows_its_inputs():
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    lens = [900, 40, 333]
    c, table, _ = filled(rng, lens, 64, 1, 256)
    q, t, n = rows(rng, 3, 8, 256, dtype="bfloat16"), dev(table), dev(lens)
    out = torch.empty_like(q)
    paged.attention_paged(q, c, t, n, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention_paged(q, c, t, n, out=out)
    n.copy_(dev([850, 40, 12]))
    graph.replay()
    replayed = out.clone()
    assert torch.equal(replayed, paged.attention_paged(q, c, t, n))
    paged.check()


def test_paged_on_two_streams_at_once():
    """Calls on different streams overlap: each has a workspace of its own, also beside prompts."""
    from mlc_vla import paged

    rng = np.random.default_rng(1)
    work = []
    for lens, page in (([1900, 10, 900, 77], 64), ([1000, 1200, 2000], 16)):
        c, table, _ = filled(rng, lens, page, 1, 128)
        q = rows(rng, len(lens), 8, 128, dtype="float16")
        k = rows(rng, 2000, 1, 128, dtype="float16")
        work.append((q, c, dev(table), dev(lens), rows(rng, 500, 8, 128, dtype="float16"), k,
                     dev([0, 500]), dev([0, 2000])))

    def calls(w):
        return (paged.attention_paged(*w[:4]), paged.attention_prompt(w[4], w[5], w[5], *w[6:]),
                paged.attention_paged(*w[:4]))

    want = [calls(w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(calls(w))
    torch.cuda.synchronize()
    paged.check()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_paged_nan_tokens_stay_with_their_request():
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    c, table, _ = filled(rng, [200, 150, 1], 16, 1, 128)
    q = rows(rng, 3, 4, 128, dtype="float16")
    t, n = dev(table), dev([200, 150, 1])
    clean = paged.attention_paged(q, c, t, n)
    p = int(table[1, 3])
    c.v.view(torch.uint8)[p, 0, 5, 9] = NAN_CODE
    out = paged.attention_paged(q, c, t, n)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert out[1, :, 9].isnan().all() and torch.equal(out[1, :, 10:], clean[1, :, 10:])
    c.k.view(torch.uint8)[p, 0, 5, 9] = NAN_CODE
    assert paged.attention_paged(q, c, t, n)[1].isnan().all()


@pytest.mark.parametrize("dim", [128, 24])
def test_paged_bad_tables_are_reported(dim):
    from mlc_vla import paged

    rng = np.random.default_rng(0)
    lens = [100, 300, 60]
    c, table, _ = filled(rng, lens, 32, 1, dim)
    q = rows(rng, 3, 4, dim, dtype="float16")
    clean = paged.attention_paged(q, c, dev(table), dev(lens))
    for what, at, number in ((19, 4, c.k.shape[0]), (19, 0, -1)):
        bad = table.copy()
        bad[1, at] = number
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = paged.attention_paged(q, c, dev(bad), dev(lens), err=err)
        assert int(err.item()) == what
        assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    for n in (-5, 32 * table.shape[1] + 1):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = paged.attention_paged(q, c, dev(table), dev([100, n, 60]), err=err)
        assert int(err.item()) == 17
        assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    paged.check()


def test_paged_pool_beyond_32_bits():
    """Codes more than 2^32 bytes into the pool: written there, and read back."""
    from mlc_vla import paged

    page, dim, pages = 128, 256, (1 << 32) // (128 * 256) + 6
    c = paged.KVCache8.empty(pages, page, 1, dim)
    rng = np.random.default_rng(0)
    table = dev([[pages - 1, pages - 4], [0, pages - 2]])
    lens = [200, 131]
    cu = dev([0, 200, 331])
    x = [rows(rng, 331, 1, dim, dtype="bfloat16") for _ in range(2)]
    slots = np.concatenate([table.cpu().numpy()[r][np.arange(n) // page] * page + np.arange(n) % page
                            for r, n in enumerate(lens)])
    paged.write_kv(c, *x, cu, dev([0, 0]), dev(slots))
    q = rows(rng, 2, 8, dim, dtype="bfloat16")
    out = paged.attention_paged(q, c, table, dev(lens))
    paged.check()
    small = paged.KVCache8.empty(4, page, 1, dim)
    slots = np.concatenate([np.arange(200), 256 + np.arange(131)])
    paged.write_kv(small, *x, cu, dev([0, 0]), dev(slots))
    assert torch.equal(out, paged.attention_paged(q, small, dev([[0, 1], [2, 3]]), dev(lens)))


# ---- refusals -------------------------------------------------------------------------------------

def test_refusals_on_the_device():
    from mlc_vla import paged

    f16 = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    q, k = f16(4, 8, 64), f16(4, 2, 64)
    cu = dev([0, 4])
    bad = [(q.float(), k, k, cu), (q, f16(4, 3, 64), f16(4, 3, 64), cu), (q, k, f16(5, 2, 64), cu),
           (q, k, k, cu.long()), (q, k.bfloat16(), k.bfloat16(), cu), (q, k, k, dev([])),
           (q, k[:, :1].expand(4, 2, 64), k, cu), (f16(4, 8, 65)[:, :, 1:], k, k, cu),
           (f16(4, 8, 128)[:, :, ::2], k, k, cu), (f16(4, 8, 12), f16(4, 2, 12), f16(4, 2, 12), cu),
           (f16(4, 8, 264), f16(4, 2, 264), f16(4, 2, 264), cu), (q, k.cpu(), k, cu)]
    for args in bad:
        with pytest.raises(ValueError):
            paged.attention_prompt(*args)
    with pytest.raises(ValueError):
        paged.attention_prompt(q, k, k, cu, prefix_lens=dev([1, 2]))
    with pytest.raises(ValueError):
        paged.attention_prompt(q, k, k, cu, out=f16(4, 8, 128))
    c = paged.KVCache8.empty(4, 16, 2, 64)
    table, n = dev(np.zeros((4, 2))), dev([1, 1, 1, 1])
    for args in [(f16(4, 8, 128), c, table, n), (f16(4, 7, 64), c, table, n), (q, c, table[:3], n),
                 (q, c, table, n[:3]), (q, c._replace(k=c.k.view(torch.uint8)), table, n),
                 (q, c._replace(v_scale=c.v_scale[:2]), table, n), (q, c, table.t(), n),
                 (q, c._replace(v=c.v[:, :1]), table, n)]:
        with pytest.raises(ValueError):
            paged.attention_paged(*args)
    for args in [(c, k, f16(4, 2, 128), cu, dev([0]), dev([0] * 4)), (c, k, k, cu, dev([0, 0]), dev([0] * 4)),
                 (c, k, k, cu, dev([0]), dev([0] * 3))]:
        with pytest.raises(ValueError):
            paged.write_kv(*args)
    with pytest.raises(ValueError):
        paged.write_kv(c, k, k, cu, dev([0]), dev([0] * 4), max_new=-1)
    with pytest.raises(ValueError):
        paged.build_slots(n, n, table, n, dev([0]), 0, 4)
    with pytest.raises(ValueError):
        paged.build_slots(n, n, table, n, dev([0, 0]), 8, 4)
    with pytest.raises(ValueError):
        paged.build_slots(n, n, table, n, dev([0]), 64, 4, num_pages=1 << 26)
    paged.check()
