"""The widest rows that the 8-bit form allows (2^26 features), each type and
direction: their column tiles stay within a grid's limits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("features", [65535 * 1024, 65535 * 1024 + 8, (1 << 26) - 3, 1 << 26])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_widest_rows_are_saved_and_loaded(features, dt):
    import rollfast_b200 as rf

    # Whole numbers below 127 with a 127 in each block: the codes are the values.
    x = (torch.arange(features, device="cuda") % 251 - 125).clamp(-126, 126).to(dt).reshape(1, features)
    x[:, ::32] = 127
    saved = rf.save_activation(x)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(rf.load_activation(saved, dtype=out), x.to(out))
    h, sg, su = rf.swiglu_forward(x, x)
    assert torch.equal(rf.load_activation(sg), x) and torch.equal(rf.load_activation(su), x) and h.isfinite().all()
    dg, du, _ = rf.swiglu_backward(x, sg, su)
    assert dg.isfinite().all() and du.isfinite().all()
