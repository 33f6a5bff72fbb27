"""An update whose gradient lies where a weight or momentum does: both are written while it is read."""
import pytest
import torch

from cbm4gnn_b200.optim import orthogonal_step


def test_a_gradient_that_is_written_is_refused():
    w, g, m = (torch.full((3, 4), float(i)) for i in range(1, 4))
    for ws, gs, ms in (([w], [m], [m]), ([w], [w], [m]), ([w, g], [m, w], [m, torch.zeros(3, 4)])):
        with pytest.raises(RuntimeError, match="a gradient is a weight or a momentum"):
            orthogonal_step(ws, gs, ms, lr=0.1)
    assert w.eq(1).all() and g.eq(2).all() and m.eq(3).all()
