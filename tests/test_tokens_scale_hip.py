"""The scale of a lookup is a number: a tensor that asks for a gradient would
not get one."""
import pytest
import torch

from xrdslam_amd import _lib
from xrdslam_amd.engine import tokens

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def test_a_scale_that_wants_a_gradient_is_refused():
    table = torch.randn(5, 8, device=DEV)
    ids = torch.tensor([4, 0, 4], device=DEV)
    scale = torch.tensor(2.0, device=DEV, requires_grad=True)
    with pytest.raises(_lib.XrdError, match='scale'):
        tokens.lookup(table, ids, scale=scale)
    want = table[ids] * 2
    assert torch.equal(tokens.lookup(table, ids, scale=scale.detach()), want)
    assert torch.equal(tokens.lookup(table, ids, scale=2), want)
    with torch.no_grad():
        assert torch.equal(tokens.lookup(table, ids, scale=scale), want)
    # the way to a gradient of the scale
    (tokens.lookup(table, ids) * scale).sum().backward()
    assert torch.allclose(scale.grad, table[ids].sum())
