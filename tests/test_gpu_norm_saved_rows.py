"""Norms' 8-bit copies are those of ``save_activation`` to the last byte also
in rows that are not finite, the blocks behind the last feature included."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [33, 40, 136, 1000, 4104, 8200])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16)], ids=["typed", "mixed"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_copies_of_rows_that_are_not_finite(d, kind, types, fmt):
    import rollfast_b200 as rf

    g = torch.Generator("cuda").manual_seed(1)
    x, b = (torch.randn(9, d, device="cuda", generator=g).to(t) for t in types)
    x[1, 2], b[2, 3], x[3, 4], b[4, 5] = float("nan"), float("nan"), float("inf"), -float("inf")
    x[5], b[5], b[6] = 0.0, 0.0, 0.0  # 0 / 0 without an epsilon
    r = rf.block_norm_forward(x, b, kind=kind, eps=0.0, save=fmt)
    for t, got in ((r.x, r.saved_x), (b, r.saved_branch), (r.y, r.saved_y)):
        want = rf.save_activation(t, fmt)
        assert torch.equal(got.codes, want.codes)
        assert torch.equal(got.scales[:, :9], want.scales[:, :9])
