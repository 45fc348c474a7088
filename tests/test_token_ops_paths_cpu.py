"""What the token operators refuse, where that shows without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from conftest import pkg


def test_forward_mode_tangents_are_refused():
    like = pkg().ops._like
    t = torch.zeros(3)
    with forward_ad.dual_level():
        like(t, "t", -1, torch.float32)
        like(t.int(), "t", -1, torch.int32)
        with pytest.raises(ValueError, match="tangent"):
            like(forward_ad.make_dual(t, t), "t", -1, torch.float32)


def test_tracing_is_refused():
    ops, x = pkg().ops, torch.zeros(4, 8)
    for f in (lambda t: ops.linear(t, t), lambda t: ops.layer_norm(t)):
        with pytest.raises(pkg().YKError, match="jit.trace"):
            torch.jit.trace(f, (x,))
