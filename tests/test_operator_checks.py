"""Operators around a stack on the CPU: what they refuse, their forms for CPU tensors, the optimiser's bookkeeping."""
import math

import pytest
import torch

from cbm4gnn_b200.classify import class_log_probs
from cbm4gnn_b200.gcn import GCNModel
from cbm4gnn_b200.norm import GroupNorm, group_norm
from cbm4gnn_b200.optim import OrthogonalSGD, orthogonal_step, orthogonalise

from operators64 import assert_within, classes64, norm64, ortho64


def _labels(*v, t=torch.int64):
    return torch.tensor(v, dtype=t)


@pytest.mark.parametrize("call,error", [
    (lambda: class_log_probs(torch.ones(4, 3), _labels(0, 1)), "shape mismatch"),
    (lambda: class_log_probs(torch.ones(4), _labels(0, 1, 2, 0)), "shape mismatch"),
    (lambda: class_log_probs(torch.ones(4, 0), _labels(0, 1, 2, 0)), "shape mismatch"),
    (lambda: class_log_probs(torch.ones(2, 3).double(), _labels(0, 1)), "fp32, bf16 or fp16"),
    (lambda: class_log_probs(torch.ones(2, 3), _labels(0, 1, t=torch.int16)), "int64 or int32"),
    (lambda: class_log_probs(torch.ones(2, 3), torch.zeros(2, dtype=torch.int64, device="meta")), "logits on cpu and labels on meta"),
    (lambda: class_log_probs(torch.ones(2, 3), _labels(0, 1), top=4), "between 0 and 3"),
    (lambda: class_log_probs(torch.ones(2, 40), _labels(0, 1), top=33), "between 0 and 32"),
    (lambda: class_log_probs(torch.ones(2, 3), _labels(0, 1), top=-1), "between 0 and 3"),
    (lambda: group_norm(torch.ones(4, 6), 4), "do not make 4 groups"),
    (lambda: group_norm(torch.ones(4, 6), 0), "do not make 0 groups"),
    (lambda: group_norm(torch.ones(6), 2), "expected"),
    (lambda: group_norm(torch.ones(2, 3, 6), 2, ptr=_labels(0, 2)), "expected"),
    (lambda: group_norm(torch.ones(4, 6).double(), 2), "fp32, bf16 or fp16"),
    (lambda: group_norm(torch.ones(4, 6), 2, activation="gelu"), "activation"),
    (lambda: group_norm(torch.ones(4, 6), 2, eps=-1.0), "eps"),
    (lambda: group_norm(torch.ones(4, 6), 2, eps=math.nan), "eps"),
    (lambda: group_norm(torch.ones(4, 6), 2, torch.ones(5)), "shape mismatch"),
    (lambda: group_norm(torch.ones(4, 6), 2, None, torch.ones(6, device="meta")), "shape mismatch"),
    (lambda: group_norm(torch.ones(4, 6), 2, torch.ones(6).bfloat16()), "parameters of x's type or fp32"),
    (lambda: group_norm(torch.ones(4, 6).half(), 2, torch.ones(6).half(), torch.ones(6)), "one type"),
    (lambda: group_norm(torch.ones(4, 6), 2, ptr=torch.ones(2)), "ptr"),
    (lambda: group_norm(torch.ones(4, 6), 2, ptr=_labels()), "ptr"),
    (lambda: group_norm(torch.ones(4, 6), 2, ptr=_labels(0, 4).to("meta")), "ptr"),
    (lambda: GroupNorm(4, 6), "do not make 4 groups"),
    (lambda: orthogonalise(torch.ones(4)), r"\[m, n\]"),
    (lambda: orthogonalise(torch.ones(4, 4).half()), "fp32 expected"),
    (lambda: orthogonalise(torch.ones(4, 4), steps=0), "steps"),
    (lambda: orthogonalise(torch.ones(4, 4), steps=65), "steps"),
    (lambda: orthogonalise(torch.ones(4, 4), eps=-1.0), "eps"),
    (lambda: orthogonal_step([torch.ones(2, 3)], [], [torch.ones(2, 3)], lr=1.0), "1 weights, 0 gradients"),
    (lambda: orthogonal_step([torch.ones(2, 3)], [torch.ones(3, 2)], [torch.ones(2, 3)], lr=1.0), "shape mismatch"),
    (lambda: orthogonal_step([torch.ones(6)], [torch.ones(6)], [torch.ones(6)], lr=1.0), "shape mismatch"),
    (lambda: orthogonal_step([torch.ones(2, 3)], [torch.ones(2, 3).half()], [torch.ones(2, 3)], lr=1.0), "dense fp32"),
    (lambda: orthogonal_step([torch.ones(2, 3)], [torch.ones(2, 3, device="meta")], [torch.ones(2, 3)], lr=1.0), "operands on cpu and meta"),
    (lambda: OrthogonalSGD([torch.nn.Parameter(torch.ones(3))]), "fp32 matrices"),
    (lambda: OrthogonalSGD([torch.nn.Parameter(torch.ones(3, 3))], momentum=1.0), "momentum"),
    (lambda: OrthogonalSGD([torch.nn.Parameter(torch.ones(3, 3))], lr=-1.0), "lr"),
    (lambda: GCNModel([8, 6, 3], norm_groups=4), "do not make 4 groups"),
    (lambda: GCNModel([8, 6, 3], activation="silu"), "activation"),
    (lambda: GCNModel([8, 6, 3])(torch.ones(4, 8), None, ptr=_labels(0, 4)), "norm_groups"),
])
def test_refused(call, error):
    with pytest.raises((RuntimeError, ValueError), match=error):
        call()


def test_classes_on_the_host():
    g = torch.Generator().manual_seed(1)
    x = torch.randn((40, 9), generator=g) * 3
    x[3, 2:7] = -torch.inf
    x[4] = -torch.inf
    x[5, 1] = torch.nan
    x[6, 1] = torch.inf
    x[7] = torch.finfo(torch.float32).min
    x[8, 3:] = 5.0
    labels = torch.randint(0, 9, (40,), generator=g)
    labels[10], labels[11], labels[3] = -100, 9, 4
    x.requires_grad_(True)
    gl, ge, gt = (torch.randn(s, generator=g) for s in ((40,), (40,), (40, 4)))
    r = class_log_probs(x, labels, top=4)
    want, bound = classes64(x, labels, 4, gl, ge, gt)
    gx, = torch.autograd.grad(r[:3], x, (gl, ge, gt))
    # (the host form takes log(sum) of a sum that holds the largest term, and p * lp as it is: an absolute error of some U more)
    assert_within(r.log_prob, want["log_prob"], bound["log_prob"] * 4)
    assert_within(r.entropy, want["entropy"], bound["entropy"] * 4)
    assert_within(r.top_log_probs, want["top"], bound["top"] * 4)
    fine = torch.ones(40, dtype=torch.bool)
    fine[[3, 5, 6, 11]] = False  # (torch's own derivatives of masked and undefined rows go by other rules)
    assert torch.equal(r.top_classes[fine], want["classes"][fine])
    assert_within(gx[fine], want["gx"][fine], bound["gx"][fine] * 4 + 1e-6)


@pytest.mark.parametrize("activation", [None, "relu", "silu"])
@pytest.mark.parametrize("ptr", [[0, 30], [0, 7, 7, 20, 30], [2, 9, 25]])
def test_norm_on_the_host(activation, ptr):
    g = torch.Generator().manual_seed(2)
    x = torch.randn((30, 12), generator=g).requires_grad_(True)
    w, b = (torch.randn(12, generator=g).requires_grad_(True) for _ in range(2))
    gy = torch.randn((30, 12), generator=g)
    y = group_norm(x, 3, w, b, torch.tensor(ptr, dtype=torch.int32) if ptr != [0, 30] else None, activation=activation)
    want, bound = norm64(x, 3, w, b, ptr, 1e-5, activation, gy, y)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, (x, w, b), gy)), y=y)
    for k in want:
        assert_within(got[k], want[k], bound[k] * 2, k)
    assert_within(group_norm(x.view(5, 6, 12), 3, w, b).reshape(30, 12), norm64(x, 3, w, b, [0, 6, 12, 18, 24, 30], 1e-5, None)[0]["y"], 1e-5)


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (5, 8), (8, 5), (6, 6)])
def test_orthogonalised_on_the_host(shape):
    u = torch.randn(shape, generator=torch.Generator().manual_seed(3))
    want, bound = ortho64(u, 5)
    assert (orthogonalise(u).double() - want).norm() <= bound
    assert orthogonalise(torch.zeros(shape)).eq(0).all()
    assert orthogonalise(torch.stack([u, 2 * u])).shape == (2, *shape)


def test_norm_and_classes_by_differences():
    """The 64-bit formulas that the GPU tests go by, against differences of their own results."""
    g = torch.Generator().manual_seed(5)
    x, w, b = torch.randn((6, 4), generator=g).double(), torch.randn(4, generator=g).double(), torch.randn(4, generator=g).double()
    gy, h = torch.randn((6, 4), generator=g).double(), 1e-6
    for act in (None, "relu", "silu"):
        want, _ = norm64(x, 2, w, b, [0, 4, 6], 1e-5, act, gy)
        f = lambda x, w, b: (norm64(x, 2, w, b, [0, 4, 6], 1e-5, act)[0]["y"] * gy).sum()  # noqa: E731
        for key, at in (("gx", 0), ("gw", 1), ("gb", 2)):
            for e in range(min(8, (x, w, b)[at].numel())):
                up, down = ([t.clone() for t in (x, w, b)] for _ in range(2))
                up[at].view(-1)[e] += h
                down[at].view(-1)[e] -= h
                assert abs((f(*up) - f(*down)) / (2 * h) - want[key].reshape(-1)[e]) < 1e-6
    labels, gl, ge, gt = torch.tensor([0, 1, 2, 3, -1, 2]), gy[:, 0], gy[:, 1], gy[:, 2:]
    want, _ = classes64(x, labels, 2, gl, ge, gt)

    def f(x):
        r, _ = classes64(x, labels, 2)
        return (r["log_prob"] * gl).sum() + (r["entropy"] * ge).sum() + (r["top"] * gt).sum()

    for e in range(x.numel()):
        up, down = x.clone(), x.clone()
        up.view(-1)[e] += h
        down.view(-1)[e] -= h
        assert abs((f(up) - f(down)) / (2 * h) - want["gx"].reshape(-1)[e]) < 1e-6


def test_optimiser_keeps_momentum_and_skips_missing_gradients():
    g = torch.Generator().manual_seed(4)
    a, b = (torch.nn.Parameter(torch.randn((4, 6), generator=g)) for _ in range(2))
    opt = OrthogonalSGD([a, b], lr=0.1, momentum=0.5, nesterov=False, weight_decay=0.2)
    first = a.detach().clone()
    before, version = b.detach().clone(), a._version
    for k in (1.0, 3.0):
        a.grad = torch.full((4, 6), k) + torch.eye(4, 6)
        opt.step()
    assert torch.equal(b.detach(), before) and b not in opt.state and a._version > version
    m = (torch.ones(4, 6) + torch.eye(4, 6)) * 0.5 + torch.full((4, 6), 3.0) + torch.eye(4, 6)
    assert torch.allclose(opt.state[a]["momentum"], m)
    want = first * 0.98 - 0.1 * orthogonalise(torch.ones(4, 6) + torch.eye(4, 6))
    want = want * 0.98 - 0.1 * orthogonalise(m)
    assert torch.allclose(a.detach(), want, atol=1e-6)
    again = OrthogonalSGD([a, b])
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[a]["momentum"], opt.state[a]["momentum"]) and again.param_groups[0]["momentum"] == 0.5


def test_models_without_norms_hold_what_they_held():
    torch.manual_seed(0)
    plain = GCNModel([8, 6, 3])
    assert sorted(plain.state_dict()) == ["layers.0.lin.weight", "layers.1.lin.weight"]
    normed = GCNModel([8, 6, 6, 3], norm_groups=2, activation="silu")
    assert [n for n, _ in normed.named_parameters() if "norms" in n] == ["norms.0.weight", "norms.0.bias", "norms.1.weight", "norms.1.bias"]
