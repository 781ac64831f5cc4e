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


def test_compare_paged_rotates_every_position_that_it_reaches():
    """The rotation table is as long as the answers: a position behind its end would be read out of
    range on the GPU."""
    from mlc_vla.compare_paged import Stack
    from mlc_vla.model.pi0.pi0_config import GemmaExpertConfig

    cfg = GemmaExpertConfig.from_variant("dummy")
    stack = Stack(cfg, 1, 10, torch.float32, 0, device="cpu", positions=5000)
    x = torch.randn(3, cfg.width)
    at = torch.tensor([0, 4096, 4999])
    q, k, v = stack.project(stack.layers[0], x, at)
    plain = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)) @ stack.layers[0].qkv.T
    plain = plain.view(3, -1, cfg.head_dim)[:, :cfg.num_heads]
    half = cfg.head_dim // 2
    angle = at[:, None].double() * 10_000.0 ** (-torch.arange(half).double() / half)
    a, b = plain.double().chunk(2, -1)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    want = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    # an fp32 table (2^-25), two products and a sum in fp32; the projections may add in another order
    assert (q.double() - want).abs().max() <= 2.0 ** -20 * plain.abs().max() + 1e-5
    with pytest.raises(IndexError):
        stack.project(stack.layers[0], x, torch.tensor([0, 1, 5000]))
    from mlc_vla.compare_paged import PagedSession

    with pytest.raises(ValueError, match="positions"):
        PagedSession(stack, 2, 5001)
    session = PagedSession(stack, 2, 40)
    session.longest = 40
    with pytest.raises(ValueError, match="beyond the session's 40"):
        session.step(x[:2])
    with pytest.raises(ValueError, match="beyond the session's 40"):
        PagedSession(stack, 2, 40).prompts(x, torch.tensor([1, 2]), torch.tensor([0, 0]), 41)


def test_attention_prompt_refuses_out_over_its_inputs():
    from mlc_vla import _lib

    lib = _lib.load()

    def call(out, tok=512, k_tok=128, total=4):
        p = ctypes.c_void_p
        return lib.pi0_attention_prompt(1, p(1 << 20), tok, 64, p(2 << 20), k_tok, 64, p(3 << 20), k_tok,
                                        64, total, total, 8, 2, 64, 1, p(4096), p(4096), None, 0.125,
                                        p(out), tok, 64, None, 0, None, None)

    for out in (1 << 20, 2 << 20, 3 << 20, (1 << 20) + 1024, (1 << 20) - 1024, (3 << 20) + 1008,
                (2 << 20) - 4 * 1024 + 16):
        assert call(out) == _lib.PI0_ERR_INVALID
    assert call(1 << 20, tok=1024) == _lib.PI0_ERR_INVALID
