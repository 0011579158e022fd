"""``embedding.lookup`` refuses scales that float32, in which it multiplies, does not hold."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -4e38])
def test_scales_past_float32_are_refused(pkg, scale):
    tokens, table = torch.tensor([1, -1], device=DEV), torch.ones(3, 32, device=DEV)
    for t in (table, table.bfloat16(), pkg.mx.quantize(table)):
        with pytest.raises(ValueError, match="scale"):
            pkg.embedding.lookup(tokens, t, scale=scale)


def test_the_largest_scale(pkg):
    top = torch.finfo(torch.float32).max
    y = pkg.embedding.lookup(torch.tensor([1, -1], device=DEV), torch.ones(3, 32, device=DEV), scale=top)
    assert torch.equal(y[0], torch.full_like(y[0], top)) and not bool(y[1].any())
