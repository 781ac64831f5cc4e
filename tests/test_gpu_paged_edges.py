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
