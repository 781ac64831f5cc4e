"""CPU: what the text-generation operators refuse before any kernel runs, at the Python functions and
at the C entry points, and the restatements that their GPU tests compare with."""

import ctypes

import numpy as np
import pytest

import paged_ref as R

torch = pytest.importorskip("torch")


def test_python_functions_refuse_host_tensors():
    from mlc_vla import paged

    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    n = torch.zeros(4, dtype=torch.int32)
    c = paged.KVCache8.empty(2, 16, 2, 64, device="cpu")
    for call in (lambda: paged.attention_prompt(x, x, x, n), lambda: paged.write_kv(c, x, x, n, n, n),
                 lambda: paged.attention_paged(x, c, n[:, None], n),
                 lambda: paged.build_slots(n, n, n[:, None], n, n[:1], 8, 4)):
        with pytest.raises(ValueError):
            call()


def test_c_entry_points_refuse():
    from mlc_vla import _lib

    lib = _lib.load()
    one = ctypes.c_void_p(4096)  # never read: every call below is refused before a launch
    bad = _lib.PI0_ERR_INVALID
    kv = _lib.Pi0Kv8C(4096, 4096, 4096, 4096, 4, 16, 2, 64)

    def cache(**kw):
        c = _lib.Pi0Kv8C(4096, 4096, 4096, 4096, 4, 16, 2, 64)
        for name, value in kw.items():
            setattr(c, name, value)
        return ctypes.byref(c)

    def slots(batch=2, table=one, columns=4, page=16, tokens=3, pages=8, stride=4):
        return lib.pi0_build_slots(batch, one, one, table, stride, columns, one, 4, one, pages, page,
                                   tokens, one, one, one, one, one, None, None)

    assert [slots(batch=-1), slots(table=None), slots(columns=0), slots(page=0), slots(tokens=-1),
            slots(pages=1 << 30), slots(stride=3)] == [bad] * 7
    assert slots(batch=1 << 20) == _lib.PI0_ERR_UNSUPPORTED

    def write(dtype=0, k=one, stride=128, cu=one, c=ctypes.byref(kv), batch=1):
        return lib.pi0_write_kv(dtype, k, stride, 64, one, 128, 64, 5, batch, cu, one, one, 5, c, None,
                                None)

    assert [write(dtype=2), write(k=None), write(k=ctypes.c_void_p(4104)), write(stride=100),
            write(cu=None), write(c=None), write(c=cache(head_dim=60)), write(c=cache(k=None)),
            write(c=cache(num_pages=1 << 30)), write(c=cache(head_dim=512))] == [bad] * 10
    assert write(batch=70000) == _lib.PI0_ERR_UNSUPPORTED

    def prompt(dtype=1, q=one, heads=8, kv_heads=2, dim=64, cu=one, total=4, out=one, tok=512, batch=1):
        return lib.pi0_attention_prompt(dtype, q, tok, 64, one, 128, 64, one, 128, 64, total, 4, heads,
                                        kv_heads, dim, batch, cu, one, None, 0.125, out, 512, 64, None, 0,
                                        None, None)

    assert [prompt(dtype=3), prompt(q=None), prompt(heads=7), prompt(kv_heads=0), prompt(dim=12),
            prompt(dim=264), prompt(cu=None), prompt(total=-1), prompt(out=ctypes.c_void_p(4100)),
            prompt(tok=4), prompt(batch=0)] == [bad] * 11
    assert prompt(total=0) == 0

    def decode(dtype=0, q=one, heads=8, c=ctypes.byref(kv), table=one, stride=4, columns=4, batch=1):
        return lib.pi0_attention_paged(dtype, q, 512, 64, batch, heads, c, table, stride, columns, one,
                                       0.125, one, 512, 64, None, 0, None, None)

    assert [decode(dtype=2), decode(q=None), decode(heads=7), decode(c=None), decode(table=None),
            decode(stride=3), decode(columns=0), decode(batch=-1)] == [bad] * 8
    assert decode(batch=0) == 0


def test_restatement_of_codes():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    finite = np.unique(codes[np.isfinite(codes)])
    assert np.array_equal(R.e4m3(finite), finite)
    x = np.random.default_rng(0).uniform(-448, 448, 20000) * 10.0 ** np.random.default_rng(1).uniform(-6, 0, 20000)
    want = torch.as_tensor(x.astype(np.float32)).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(R.e4m3(x.astype(np.float32)), want)
    assert [R.pow2_scale(a) for a in (448.0, 449.0, 0.0, 7.0)] == [1.0, 2.0, 2.0 ** -64, 2.0 ** -6]


def test_restatement_of_slots():
    table = np.full((2, 3), -1)
    table[0, 0] = 9
    t, cu, pos, slots, lens, free = R.build_slots([3, 0], [2, 5], table, [4, 5, 6, 7], 0, 4, 8)
    assert t.tolist() == [[9, 4, -1], [5, 6, -1]] and cu.tolist() == [0, 2, 7]
    assert pos.tolist() == [3, 4, 0, 1, 2, 3, 4, 0]
    assert slots.tolist() == [39, 16, 20, 21, 22, 23, 24, -1]
    assert lens.tolist() == [5, 5] and free == 3
