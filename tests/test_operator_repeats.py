"""One update that is given a tensor twice: every weight and momentum is written once."""
import pytest
import torch

from cbm4gnn_b200.optim import orthogonal_step


def test_written_twice_is_refused():
    w, g, m = torch.ones(2, 3), torch.ones(2, 3), torch.zeros(2, 3)
    for ws, ms in (([w, w], [m, torch.zeros(2, 3)]), ([w, torch.ones(2, 3)], [m, m]), ([w], [w])):
        with pytest.raises(RuntimeError, match="twice"):
            orthogonal_step(ws, [g] * len(ws), ms, lr=0.1)
    assert w.eq(1).all() and m.eq(0).all()
    orthogonal_step([w, torch.ones(2, 3)], [g, g], [m, torch.zeros(2, 3)], lr=0.1)   # a gradient may be
    orthogonal_step([torch.ones(0, 3)] * 2, [torch.ones(0, 3)] * 2, [torch.ones(0, 3)] * 2, lr=0.1)
