"""CPU checks of what the mixture-of-experts layer refuses."""
import importlib

import pytest
import torch

from conftest import PKG_NAME


@pytest.fixture(scope="module")
def moe():
    u = torch.uint8
    cls = importlib.import_module(PKG_NAME + ".mxfp4_moe").Mxfp4MoE
    E, D, F = 3, 64, 96
    return cls(torch.zeros(E, 2 * F, D // 2, dtype=u), torch.zeros(E, 2 * F, D // 32, dtype=u),
               torch.zeros(E, D, F // 2, dtype=u), torch.zeros(E, D, F // 32, dtype=u))


@pytest.mark.parametrize("x,ids,weights", [((8, 64), (8, 2), (4, 4)), ((8, 64), (8, 2), (2, 8)), ((2, 4, 64), (2, 4, 2), (4, 2, 2)),
                                           ((2, 4, 64), (4, 2, 2), (2, 4, 2)), ((2, 4, 64), (8, 2), (8, 2)), ((8, 64), (8, 2), (16,)),
                                           ((64,), (), ())])
def test_shapes_that_only_count_alike(moe, x, ids, weights):
    """As many weights or slots as there are, but not the tokens' own."""
    with pytest.raises(ValueError, match="do not fit"):
        moe(torch.zeros(x), torch.zeros(ids, dtype=torch.int64), torch.ones(weights))
