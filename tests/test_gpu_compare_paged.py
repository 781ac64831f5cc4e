"""GPU: the four text-generation operators together, as a serving loop uses them
(``mlc_vla.compare_paged``): prompts and greedy steps of a small stack against dense attention."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant,dtype,lens", [
    ("mini_vlm", "float16", [70, 33, 129, 1]), ("mini_vlm", "bfloat16", [5, 64, 200]),
    ("gemma_2b", "float16", [300, 17, 64]), ("dummy", "float16", [40, 3])])
def test_compare_paged(variant, dtype, lens):
    from mlc_vla import compare_paged
    from mlc_vla.model.pi0.pi0_config import GemmaExpertConfig

    assert compare_paged.run(GemmaExpertConfig.from_variant(variant), dtype, lens, steps=8)
