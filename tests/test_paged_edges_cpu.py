"""CPU: refusals and host-side parts of the text-generation operators that need no GPU."""

import ctypes

import pytest

torch = pytest.importorskip("torch")


def test_build_slots_refuses_outputs_over_its_inputs():
    """The kernel's blocks read lengths and the free list while others write the results."""
    from mlc_vla import _lib

    lib = _lib.load()
    names = ("kv_lens", "new_lens", "free_pages", "free_pos", "cu", "positions", "slots", "kv_out",
             "pos_out")
    at = {n: 4096 * (i + 1) for i, n in enumerate(names)}  # never read: every call is refused

    def call(**over):
        p = {n: ctypes.c_void_p(a) for n, a in {**at, **over}.items()}
        return lib.pi0_build_slots(2, p["kv_lens"], p["new_lens"], ctypes.c_void_p(1 << 20), 4, 4,
                                   p["free_pages"], 4, p["free_pos"], 8, 16, 3, p["cu"],
                                   p["positions"], p["slots"], p["kv_out"], p["pos_out"], None, None)

    for over in ({"kv_out": at["kv_lens"]}, {"kv_out": at["kv_lens"] + 4},
                 {"kv_out": at["new_lens"] - 4}, {"pos_out": at["free_pos"]},
                 {"pos_out": at["free_pages"] + 12}, {"cu": at["kv_lens"] - 8},
                 {"slots": at["positions"] + 8}, {"kv_out": at["cu"]}, {"pos_out": at["kv_out"] + 4}):
        assert call(**over) == _lib.PI0_ERR_INVALID, over
