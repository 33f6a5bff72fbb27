"""The operators around a stack on the GPU at the edges of what their documentation allows, against their 64-bit forms."""
import pytest
import torch

from cbm4gnn_b200.classify import class_log_probs

from operators64 import assert_within, classes64

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=_gen(seed))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("c,top", [(1, 1), (3, 3), (3, 2), (32, 32), (47, 5), (200, 32), (600, 7), (1300, 3), (2000, 32), (20_000, 20)])
def test_undefined_classes_are_listed_like_others(kind, c, top):
    """NaN comes first, the lower class before the higher, also at class 0 and where all classes are undefined; rows beside such ones are as ever."""
    n = 12
    for pitch, first in ((c, 0), (c + 3, 1)):   # aligned rows, and rows out of line
        wide = torch.zeros((n, pitch), dtype=kind, device="cuda")
        wide[:, first:first + c] = _normal(c, n, c).to(kind)
        x = wide[:, first:first + c]
        x[0] = torch.nan
        x[2, 0] = torch.nan
        x[4, 0] = x[4, c - 1] = torch.nan
        x[6, c // 2:] = torch.nan
        x[8, 0], x[8, c - 1] = torch.nan, torch.inf
        x[10] = torch.nan
        x[11] = torch.nan
        x = x.detach().requires_grad_(True)
        labels = torch.arange(n, device="cuda") % c
        r = class_log_probs(x, labels, top=top)
        gt = _normal(3, n, top)
        want, bound = classes64(x, labels, top, None, None, gt)
        assert torch.equal(r.top_classes, want["classes"])
        assert_within(r.top_log_probs.detach(), want["top"], bound["top"], "top")
        gx, = torch.autograd.grad(r.top_log_probs, x, gt)
        assert_within(gx, want["gx"], bound["gx"], "gx")
