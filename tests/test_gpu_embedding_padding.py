"""Padding rows of ``embedding.lookup`` hold +0 (all bits zero) whatever the scale, for every kind of table and row length."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("scale", [-1.0, -0.25, 12.0])
@pytest.mark.parametrize("width", [1, 33, 64, 256, 1001, 2056])
def test_padding_is_positive_zero(pkg, width, scale):
    g = torch.Generator(device=DEV).manual_seed(width)
    table = torch.randn(40, width, device=DEV, generator=g)
    tokens = torch.tensor([-1, 3, 40, -7, 39], device=DEV)
    for t in (table, table.bfloat16(), pkg.mx.quantize(table)):
        y = pkg.embedding.lookup(tokens, t, scale=scale)
        bits = y.view(torch.int32 if y.dtype == torch.float32 else torch.int16)
        assert not bool(bits[[0, 2, 3]].any()) and bool(bits[1].any()) and bool(bits[4].any())
