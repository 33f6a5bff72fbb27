"""The operators around a stack on the GPU over the lengths, layouts and lists at which their ways change, against their 64-bit forms."""
import pytest
import torch

from cbm4gnn_b200.classify import class_log_probs
from cbm4gnn_b200.norm import group_norm
from cbm4gnn_b200.optim import orthogonal_step, orthogonalise

from operators64 import assert_within, classes64, half_step, norm64, ortho64

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=_gen(seed))


def _pointers(n, longest, seed):
    """Samples of 0 to `longest` rows that cover n rows."""
    sizes = torch.randint(0, longest + 1, (3 * n // longest + 8,), generator=torch.Generator().manual_seed(seed))
    ends = sizes.cumsum(0)
    return [0] + [int(e) for e in ends if e < n] + [n]


def _check(x, groups, w, b, ptr, activation, gy):
    on = None if ptr is None else torch.tensor(ptr, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = group_norm(leaves[0], groups, *leaves[1:], ptr=on, activation=activation)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, gy)))
    want, bound = norm64(x, groups, w, b, [0, x.size(0)] if ptr is None else ptr, 1e-5, activation, gy, y.detach())
    assert_within(y.detach(), want["y"], bound["y"], "y")
    assert_within(got["gx"], want["gx"], bound["gx"], "gx")
    for k in ("gw", "gb"):  # (rounded to the parameter's type: half a step of the value)
        assert_within(got[k], want[k], bound[k] + half_step(got[k].dtype) * want[k].abs(), k)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,groups,longest", [(20_000, 4, 1, 6), (9_000, 5, 1, 20), (12_000, 16, 2, 40), (12_000, 64, 8, 60), (3_000, 512, 8, 12), (4_001, 300, 150, 30),
                                                (30_000, 48, 3, 9_000), (40_000, 24, 2, 39_000), (20_000, 130, 13, 700)])
def test_norm_of_samples_of_many_lengths(kind, n, c, groups, longest):
    x = (_normal(n, n, c) * 1.5 + 0.4).to(kind)
    _check(x, groups, (_normal(1, c) + 1).to(kind), _normal(2, c).to(kind), _pointers(n, longest, c), "silu", _normal(3, n, c).to(kind))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,groups", [(60_000, 32, 4), (50_001, 20, 2), (30_000, 256, 32), (40_000, 9, 3), (9_001, 600, 2)])
def test_norm_of_one_long_sample(kind, n, c, groups):
    x = (_normal(n, n, c) - 1.2).to(kind)
    _check(x, groups, _normal(1, c) + 1, _normal(2, c), None, "relu", _normal(3, n, c).to(kind))


@pytest.mark.parametrize("kind", TYPES)
def test_norm_of_rows_apart_and_out_of_line(kind):
    n, c = 3000, 64
    wide, gwide = _normal(1, n, 200).to(kind), _normal(2, n, 150).to(kind)
    ptr = _pointers(n, 50, 3)
    for a, b in ((0, 0), (8, 16), (4, 2), (1, 0), (0, 1), (2, 8)):   # offsets of 16 bytes and less, in x and in the gradient
        _check(wide[:, a:a + c], 8, _normal(4, c), _normal(5, c), ptr, None, gwide[:, b:b + c])


def test_norm_where_a_short_sample_follows_a_long_one():
    """Rows of samples that a thread keeps from one pass to the next, beside those that it does not."""
    ptr = [0, 2, 5, 105, 106, 110, 3110, 3112, 3116, 3120, 3200, 3300]
    for c, groups in ((32, 4), (64, 2), (512, 4)):
        for kind in TYPES:
            x = _normal(c, 3300, c).to(kind)
            _check(x, groups, _normal(1, c), _normal(2, c), ptr, "silu", _normal(3, 3300, c).to(kind))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,top", [(400, 1100, 5), (400, 2000, 32), (350, 4097, 1), (320, 8191, 9), (320, 8193, 3), (310, 16_500, 20), (150, 12_345, 7)])
def test_classes_of_middling_rows(kind, n, c, top):
    for pitch, first in ((c, 0), (c + 3, 1)):
        wide = torch.zeros((n, pitch), dtype=kind, device="cuda")
        wide[:, first:first + c] = _normal(c, n, c).to(kind)
        wide[0] = -torch.inf
        wide[1, ::2] = -torch.inf
        wide[2, c // 2] = torch.nan
        wide[3] = 1.5   # all alike: the lowest classes are listed
        x = wide[:, first:first + c].detach().requires_grad_(True)
        labels = torch.randint(-1, c, (n,), device="cuda", generator=_gen(n))
        labels[4:8] = torch.tensor([0, c - 1, c // 2, 1], device="cuda")
        gl, ge, gt = _normal(1, n), _normal(2, n), _normal(3, n, top)
        r = class_log_probs(x, labels, top=top)
        want, bound = classes64(x, labels, top, gl, ge, gt)
        assert_within(r.log_prob.detach(), want["log_prob"], bound["log_prob"], "log_prob")
        assert_within(r.entropy.detach(), want["entropy"], bound["entropy"], "entropy")
        assert_within(r.top_log_probs.detach(), want["top"], bound["top"], "top")
        defined = torch.arange(n, device="cuda") != 2
        assert torch.equal(r.top_classes[defined], want["classes"][defined])
        gx, = torch.autograd.grad(r[:3], x, (gl, ge, gt))
        assert_within(gx[defined], want["gx"][defined], bound["gx"][defined], "gx")
        assert gx[2].isnan().all()


def _step64(w, g, m, lr, momentum, decay):
    m1 = momentum * m.double() + g.double()
    o, bound = ortho64(g.double() + momentum * m1, 5)
    f = lr * max(1.0, w.size(0) / w.size(1)) ** 0.5
    # (u and the new weight are rounded to fp32: 2^-23 of the weight, and of u what five steps make of it, some hundreds of times)
    return m1, (1 - lr * decay) * w.double() - f * o, f * (bound + 2e-4 * 2.0 ** -3) + 2.0 ** -23 * w.double().norm()


@pytest.mark.parametrize("shapes", [
    [(64, 100)] * 4 + [(47, 256), (128, 1024), (1, 7), (1024, 128), (16, 16), (33, 200), (128, 130)],           # all small, two lists
    [(64, 100), (300, 200), (47, 256), (256, 256), (16, 600), (129, 1000), (7, 7), (500, 64), (1, 300), (260, 140), (64, 64)],
    [(400, 300)] * 9])
def test_long_lists_captured_and_replayed(shapes):
    start = [[_normal(100 * k + i, *s) for i, s in enumerate(shapes)] for k in range(3)]
    ws, gs, ms = ([t.clone() for t in ts] for ts in start)
    step = lambda: orthogonal_step(ws, gs, ms, lr=0.05, momentum=0.9, weight_decay=0.01)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    wants = [_step64(*a, 0.05, 0.9, 0.01) for a in zip(*start)]
    for w, m, (m1, w1, bound) in zip(ws, ms, wants):
        assert torch.allclose(m.double(), m1, atol=1e-6, rtol=1e-6)
        assert (w.double() - w1).norm() <= bound
    after = [t.clone() for t in ws + ms]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):   # a replay from the start, with the operands' values of now
        for to, of in zip(ws + gs + ms, start[0] + start[1] + start[2]):
            to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(after, ws + ms))


def test_two_captured_graphs_and_an_eager_call_side_by_side():
    us = [_normal(i, 300, 420) for i in range(3)]
    want = [orthogonalise(u) for u in us]
    outs, graphs = [], []
    for u in us[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(orthogonalise(u))
        graphs.append(graph)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        last = orthogonalise(us[2])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(last, want[2])


def test_norm_of_more_groups_than_a_grid_is_wide():
    c = 140_000
    x = _normal(1, 2, 40, c).bfloat16().requires_grad_(True)
    gy = _normal(2, 2, 40, c).bfloat16()
    y = group_norm(x, c // 2)
    gx, = torch.autograd.grad(y, x, gy)
    want, bound = norm64(x.detach().reshape(80, c), c // 2, None, None, [0, 40, 80], 1e-5, None, gy.reshape(80, c), y.detach().reshape(80, c))
    assert_within(y.detach().reshape(80, c), want["y"], bound["y"], "y")
    assert_within(gx.reshape(80, c), want["gx"], bound["gx"], "gx")
    with pytest.raises(RuntimeError, match="bad sizes"):
        group_norm(torch.zeros((2, (1 << 22) + 2), device="cuda"), 2)
