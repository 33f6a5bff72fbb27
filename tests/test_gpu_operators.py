"""The operators around a stack on the GPU against their 64-bit forms (operators64.py has the bounds)."""
import math

import pytest
import torch

from cbm4gnn_b200 import graphs
from cbm4gnn_b200.cbm import cbm_matrix
from cbm4gnn_b200.classify import class_log_probs
from cbm4gnn_b200.gcn import GCNModel
from cbm4gnn_b200.norm import GroupNorm, group_norm
from cbm4gnn_b200.optim import OrthogonalSGD, orthogonal_step, orthogonalise
from cbm4gnn_b200.utility import add_self_loops, normalize_edge_index

from operators64 import assert_within, classes64, half_step, norm64, ortho64

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=_gen(seed))


# ------------------------------------------------------------------------------------------------ classes
def _check_classes(x, labels, top, grads=(True, True, True)):
    n = x.size(0)
    given = [_normal(9 + i, *s) if on else None for i, (on, s) in enumerate(zip(grads, ((n,), (n,), (n, top))))]
    x = x.detach().requires_grad_(True)
    r = class_log_probs(x, labels, top=top)
    used = [(o, g) for o, g in zip(r[:3], given) if g is not None and g.numel()]
    want, bound = classes64(x, labels, top, *given)
    assert_within(r.log_prob.detach(), want["log_prob"], bound["log_prob"], "log_prob")
    assert_within(r.entropy.detach(), want["entropy"], bound["entropy"], "entropy")
    assert_within(r.top_log_probs.detach(), want["top"], bound["top"], "top")
    assert torch.equal(r.top_classes, want["classes"])
    if used:
        gx, = torch.autograd.grad([o for o, _ in used], x, [g for _, g in used])
        assert gx.dtype == x.dtype and gx.shape == x.shape
        assert_within(gx, want["gx"], bound["gx"], "gx")
    return r


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,top", [(1, 1, 1), (1, 2, 0), (5, 7, 3), (4097, 7, 7), (1000, 31, 5), (999, 32, 32), (333, 33, 2), (257, 47, 3),
                                     (130, 64, 1), (77, 172, 10), (65, 256, 4), (33, 500, 32), (9, 1000, 5), (6, 1025, 3), (5, 4099, 20),
                                     (3, 16_411, 32), (2, 50_257, 8), (1, 128_256, 20)])
def test_classes_of_every_width(kind, n, c, top):
    x = (_normal(c, n, c) * torch.linspace(0.3, 6.0, n, device="cuda")[:, None]).to(kind)
    labels = torch.randint(-1, c, (n,), device="cuda", generator=_gen(n))
    _check_classes(x, labels if n % 2 else labels.int(), top)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("c", [5, 40, 200, 1300, 20_000])
def test_masked_infinite_and_undefined_logits(kind, c):
    x = (_normal(3, 16, c) * 3).to(kind)
    low = torch.finfo(kind).min
    x[1] = -torch.inf                      # nothing is open
    x[2, 1:] = -torch.inf                  # one class
    x[3] = low                             # a mask of the lowest value on everything
    x[4, : c - 1] = low
    x[5, 2] = torch.nan
    x[6, 3] = torch.inf
    x[7, 1] = x[7, 4] = torch.inf
    x[8, ::2] = -torch.inf
    x[9] = 0.0
    x[10, ::2] = -0.0
    x[10, 1::2] = 0.0
    x[11, 0] = 60.0 if kind != torch.float16 else 40.0  # decided
    x[12] = x[12, 0]                       # ties
    x[13, c // 2:] = 7.0
    labels = torch.arange(16, device="cuda") % c
    labels[8] = 0                          # a closed class
    labels[14], labels[15] = -100, c       # none, and one that does not exist
    for grads in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        _check_classes(x, labels, min(c, 5), grads)


def test_classes_of_strided_rows_and_no_rows():
    wide = _normal(4, 300, 90)
    labels = torch.randint(0, 41, (300,), device="cuda", generator=_gen(2))
    for x in (wide[:, 3:44], wide[:, :41], _normal(5, 41, 300).t(), _normal(6, 300, 48)[:, :41], wide[::2, :41].repeat(2, 1), wide[:1, :41].expand(300, 41)):
        _check_classes(x, labels, 3)
    strided = torch.arange(600, device="cuda")[::2] % 41
    _check_classes(wide[:, :41], strided, 2)
    r = class_log_probs(wide[:0], labels[:0], top=2)
    assert r.log_prob.shape == (0,) and r.top_classes.shape == (0, 2)
    assert torch.autograd.grad(class_log_probs(x0 := wide[:0].requires_grad_(True), labels[:0]).log_prob.sum(), x0)[0].shape == (0, 90)


def test_classes_through_broadcast_gradients_and_only_once():
    x = _normal(7, 50, 12).requires_grad_(True)
    labels = torch.arange(50, device="cuda") % 12
    gx, = torch.autograd.grad(class_log_probs(x, labels).log_prob.sum(), x)
    want, bound = classes64(x, labels, 0, torch.ones(50, device="cuda"))
    assert_within(gx, want["gx"], bound["gx"])
    gx, = torch.autograd.grad(class_log_probs(x, labels).log_prob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_offsets_past_32_bits():
    """Rows whose offsets, in values, do not fit 32 bits."""
    n, c = 70_000, 32_768
    x = torch.zeros((n, c), dtype=torch.bfloat16, device="cuda")
    x[-3:] = _normal(8, 3, c).bfloat16()
    x.requires_grad_(True)
    labels = torch.arange(n, device="cuda") % c
    r = class_log_probs(x, labels, top=2)
    gl = _normal(1, n)
    gx, = torch.autograd.grad(r.log_prob, x, gl)
    want, bound = classes64(x[-3:], labels[-3:], 2, gl[-3:])
    assert_within(r.log_prob[-3:].detach(), want["log_prob"], bound["log_prob"])
    assert torch.equal(r.top_classes[-3:], want["classes"])
    assert_within(gx[-3:], want["gx"], bound["gx"])
    assert (r.log_prob[:-3].double() + math.log(c)).abs().max() < 1e-5


# --------------------------------------------------------------------------------------------------- norm
def _check_norm(x, groups, w, b, ptr, activation, three=False, train=True):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(train and t.is_leaf)
    n, c = x.reshape(-1, x.size(-1)).shape
    gy = _normal(11, *x.shape).to(x.dtype)
    on = None if ptr is None else torch.tensor(ptr, device="cuda")
    y = group_norm(x, groups, w, b, ptr=on, activation=activation)
    assert y.dtype == x.dtype and y.shape == x.shape
    rows = list(range(0, n + 1, x.size(1))) if three else [0, n] if ptr is None else ptr
    want, bound = norm64(x.detach().reshape(n, c), groups, w, b, rows, 1e-5, activation, gy.reshape(n, c) if train else None, y.detach().reshape(n, c))
    assert_within(y.detach().reshape(n, c), want["y"], bound["y"], "y")
    if train:
        for k, g in zip([k for k, t in zip(("gx", "gw", "gb"), (x, w, b)) if t is not None], torch.autograd.grad(y, leaves, gy)):
            # (a parameter's gradient is rounded to its own type: half a step, eps / 2 of the value)
            rounded = half_step(g.dtype) * want[k].abs() if k != "gx" else 0.0
            assert_within(g.reshape(want[k].shape), want[k], bound[k] + rounded, k)
        with torch.no_grad():
            assert torch.equal(group_norm(x, groups, w, b, ptr=on, activation=activation), y)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("activation", [None, "relu", "silu"])
@pytest.mark.parametrize("n,c,groups", [(1, 1, 1), (1, 4, 4), (3, 6, 2), (100, 64, 8), (257, 100, 10), (1000, 33, 11), (63, 500, 5), (65, 256, 32),
                                        (31, 1100, 4), (5000, 8, 1), (2, 2056, 8), (700, 48, 48), (129, 36, 3)])
def test_norm_of_one_graph(kind, activation, n, c, groups):
    x = (_normal(n, n, c) * 2 + 0.7).to(kind)
    _check_norm(x, groups, _normal(1, c) + 1, _normal(2, c), None, activation)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,groups,ptr", [
    (300, 64, 8, [0, 1, 1, 1, 5, 70, 71, 300]), (300, 100, 10, [0, 0, 0, 150, 150, 290]), (200, 33, 3, [13, 50, 60, 190]), (64, 12, 4, [0, 0]),
    (64, 12, 4, [64, 64]), (50, 24, 6, list(range(51))), (5000, 20, 5, [0, 17, 4000, 4001, 5000]), (4096, 40, 2, list(range(0, 4097, 3))),
    (130, 516, 2, [5, 6, 100, 130])])
def test_norm_of_uneven_graphs(kind, n, c, groups, ptr):
    x = (_normal(n, n, c) - 0.3).to(kind)
    _check_norm(x, groups, (_normal(1, c) + 1).to(kind), _normal(2, c).to(kind), ptr, "silu")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("b,n,c,groups", [(7, 1, 64, 8), (1000, 1, 256, 16), (5, 1, 33, 3), (3, 1, 3000, 5), (4, 9, 100, 10), (2, 300, 48, 6), (65, 2, 12, 1),
                                          (4097, 1, 47, 1), (10, 1, 1100, 50), (300, 1, 6, 3)])
def test_norm_of_equal_graphs(kind, b, n, c, groups):
    x = (_normal(n, b, n, c) * 3 + 1).to(kind)
    _check_norm(x, groups, _normal(1, c) + 1, _normal(2, c), None, "relu", three=True)
    _check_norm(x, groups, None, None, None, None, three=True)


def test_norm_keeps_digits_beside_a_large_mean():
    """Values of 1000 and a spread of 1: sums of squares would leave nothing of the variance."""
    for ptr in (None, [0, 40, 4000]):
        x = 1000.0 + _normal(5, 4000, 32)
        _check_norm(x, 4, _normal(1, 32), _normal(2, 32), ptr, "silu")
    _check_norm(1000.0 + _normal(5, 400, 1, 32), 4, _normal(1, 32), _normal(2, 32), None, "silu", three=True)


def test_norm_of_constant_rows_infinities_and_nan():
    x = torch.full((6, 8), 3.0, device="cuda")
    assert torch.equal(group_norm(x, 2, bias=torch.ones(8, device="cuda")), torch.ones(6, 8, device="cuda"))
    x[4, 1] = torch.nan
    x[5, 6] = torch.inf
    y = group_norm(x, 2, ptr=torch.tensor([0, 4, 5, 6], device="cuda"), activation="relu")
    assert y[:4].eq(0).all() and y[4, :4].isnan().all() and y[4, 4:].eq(0).all() and y[5, :4].eq(0).all() and y[5, 4:].isnan().all()


def test_norm_of_strided_rows_and_no_rows():
    wide = _normal(6, 400, 80)
    for x in (wide[:, 8:72], wide[:, 3:67], wide[::2, :64], _normal(7, 64, 300).t(), wide[:1, :64].expand(50, 64), _normal(8, 200, 67)[:, :64]):
        _check_norm(x.detach(), 8, _normal(1, 64), _normal(2, 64), None, "silu")
        _check_norm(x.detach(), 8, _normal(1, 128)[::2], _normal(2, 64), [0, 3, 30, x.size(0) - 1], "relu")
    three = _normal(9, 6, 10, 48)[:, :, :40]
    _check_norm(three, 4, _normal(1, 40), _normal(2, 40), None, "silu", three=True)
    _check_norm(_normal(9, 10, 6, 40).transpose(0, 1), 4, _normal(1, 40), _normal(2, 40), None, "silu", three=True)
    w, b = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
    for x, ptr in ((_normal(1, 0, 8), None), (_normal(1, 0, 8), torch.zeros(3, dtype=torch.int64, device="cuda")), (_normal(1, 0, 5, 8), None), (_normal(1, 5, 0, 8), None)):
        x.requires_grad_(True)
        y = group_norm(x, 2, w, b, ptr=ptr)
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == x.shape == gx.shape and gw.eq(0).all() and gb.eq(0).all()


def test_norm_pointers_that_leave_the_rows_stay_inside():
    """Their values cannot be looked at without a wait; what they say is cut off at the rows there are."""
    x = _normal(3, 100, 16)
    y = group_norm(x, 4, ptr=torch.tensor([-5, 40, 1000], device="cuda"))
    assert torch.equal(y, group_norm(x, 4, ptr=torch.tensor([0, 40, 100], device="cuda")))
    assert group_norm(x, 4, ptr=torch.tensor([50, 20, 10], device="cuda")).eq(0).all()


def test_norm_gradients_of_some():
    x, w, b = _normal(1, 60, 24), _normal(2, 24), _normal(3, 24)
    gy = _normal(4, 60, 24)
    want, bound = norm64(x, 3, w, b, [0, 60], 1e-5, "silu", gy)
    for k, t in (("gx", x), ("gw", w), ("gb", b)):
        t.requires_grad_(True)
        assert_within(torch.autograd.grad(group_norm(x, 3, w, b, activation="silu"), t, gy)[0], want[k], bound[k], k)
        t.requires_grad_(False)


# ------------------------------------------------------------------------------------------------- update
@pytest.mark.parametrize("m,n", [(1, 1), (1, 50), (50, 1), (7, 64), (64, 500), (100, 256), (256, 100), (47, 256), (128, 128), (129, 127), (130, 700),
                                 (256, 256), (257, 513), (500, 333), (640, 640), (1000, 1030), (513, 2050), (2050, 65)])
def test_orthogonalised(m, n):
    u = _normal(m * n, m, n)
    u[: m // 3] *= 0.01
    for steps in (1, 5):
        want, bound = ortho64(u, steps)
        got = orthogonalise(u, steps=steps)
        assert got.shape == u.shape and (got.double() - want).norm() <= bound, ((got.double() - want).norm().item(), bound.item())


def test_orthogonalised_batches_and_layouts():
    for b, m, n in ((3, 40, 60), (5, 300, 200), (2, 1, 1), (2, 700, 900)):
        u = _normal(b, b, m, n) * torch.tensor([10.0 ** (3 * i) for i in range(b)], device="cuda")[:, None, None]
        for v in (u, u.transpose(1, 2), u[:, : m // 2 + 1, : n // 2 + 1], u.transpose(0, 1).contiguous().transpose(0, 1), u[:1].expand(b, m, n)):
            got = orthogonalise(v)
            for i in range(b):
                want, bound = ortho64(v[i], 5)
                assert (got[i].double() - want).norm() <= bound
    assert orthogonalise(torch.zeros((2, 0, 5), device="cuda")).shape == (2, 0, 5)
    assert orthogonalise(_normal(1, 0, 5, 5)).shape == (0, 5, 5)


@pytest.mark.parametrize("m,n", [(20, 30), (200, 300), (600, 520)])
def test_orthogonalised_extremes(m, n):
    assert orthogonalise(torch.zeros((m, n), device="cuda")).eq(0).all()
    u = _normal(1, m, n)
    want, bound = ortho64(u, 5)
    for scale in (2.0 ** 90, 2.0 ** -10):   # squares that fp32 does not hold; near eps only the division counts
        got = orthogonalise(u * scale, eps=0.0)
        assert (got.double() - ortho64(u * scale, 5, 0.0)[0]).norm() <= bound
    one = _normal(2, m, 1) @ _normal(3, 1, n)   # of rank one, its rounding beside it
    want, bound = ortho64(one, 5)
    assert (orthogonalise(one).double() - want).norm() <= bound
    u[3, 4] = torch.nan
    assert orthogonalise(u).isnan().any()
    u[3, 4] = torch.inf
    assert orthogonalise(u).isnan().any()


@pytest.mark.parametrize("nesterov", [True, False])
def test_step_of_a_list(nesterov):
    shapes = [(64, 500), (7, 64), (256, 100), (300, 700), (5, 1), (0, 4), (600, 16), (129, 129)]
    ws = [_normal(i, *s) for i, s in enumerate(shapes)]
    wide = _normal(50, 64, 600)
    ws[0] = wide[:, 20:520]   # rows at a pitch
    outside = wide[:, 520:].clone()
    gs, ms = [_normal(10 + i, *s) for i, s in enumerate(shapes)], [_normal(20 + i, *s) for i, s in enumerate(shapes)]
    gs[3] = _normal(13, 700, 300).t()
    want = []
    for w, g, m in zip(ws, gs, ms):
        m1 = 0.9 * m.double() + g.double()
        u = g.double() + 0.9 * m1 if nesterov else m1
        o, bound = ortho64(u, 5) if u.numel() else (u, torch.zeros((), device="cuda"))
        f = 0.03 * max(1.0, w.size(0) / max(1, w.size(1))) ** 0.5
        want.append((m1, (1 - 0.03 * 0.1) * w.double() - f * o, f * (bound + 2e-4 * 2.0 ** -3) + 2.0 ** -23 * w.double().norm()))
    orthogonal_step(ws, gs, ms, lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    for w, m, (m1, w1, bound) in zip(ws, ms, want):
        assert torch.allclose(m.double(), m1, atol=1e-6, rtol=1e-6)
        assert (w.double() - w1).norm() <= bound + 1e-12
    assert torch.equal(wide[:, 520:], outside)


# --------------------------------------------------------------------------------- streams, graphs, together
def _calls():
    x = _normal(1, 3000, 40).requires_grad_(True)
    logits = _normal(2, 500, 47).requires_grad_(True)
    labels = torch.arange(500, device="cuda") % 47
    ptr = torch.tensor([0, 100, 100, 2000, 2900], device="cuda")
    u, w, m = _normal(3, 300, 200), _normal(4, 64, 128), _normal(5, 64, 128)
    small = _normal(6, 64, 128)

    def call():
        y = group_norm(x, 4, activation="silu", ptr=ptr)
        z = group_norm(x, 4, activation="silu")
        r = class_log_probs(logits, labels, top=3)
        gx, = torch.autograd.grad(y.sum() + (z * z).sum(), x)
        gl, = torch.autograd.grad(r.log_prob.mean() + r.entropy.mean(), logits)
        wc, mc = w.clone(), m.clone()
        orthogonal_step([wc], [small], [mc], lr=0.1)
        return [y.detach(), z.detach(), gx, gl, r.log_prob.detach(), r.entropy.detach(), r.top_classes, orthogonalise(u), wc, mc]

    return call, [x, logits, u, w, m, small]


def test_results_do_not_change_between_calls_or_streams():
    call, _ = _calls()
    first = call()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in side:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_calls_see_new_operands():
    call, inputs = _calls()
    call()
    torch.cuda.synchronize()
    graphs_, outs = [], []
    pool = None
    for _ in range(2):   # two graphs of one pool
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(call())
        pool = g.pool()
        graphs_.append(g)
    for k in range(2):
        with torch.no_grad():
            for i, t in enumerate(inputs):
                t.copy_(_normal(100 * k + i, *t.shape))
        want = [t.clone() for t in call()]
        for g, out in zip(graphs_, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def _graph(n=600):
    ei = add_self_loops(torch.from_numpy(graphs.make_graph("c1", scale=n / 4096)))
    c = cbm_matrix(ei.to(torch.int32), torch.ones(ei.shape[1]), alpha=2, normalized=True)
    a = torch.sparse_coo_tensor(ei.flip(0), normalize_edge_index(ei), (c.num_rows, c.num_rows)).to_dense().double().cuda()
    return ei, c, a


@pytest.mark.parametrize("activation", ["relu", "silu"])
def test_a_training_step_of_a_normed_model(activation):
    """Norms between the layers, the loss with its gradient, the update: against the same step in 64 bits."""
    ei, c, a = _graph()
    n = c.num_rows
    torch.manual_seed(0)
    model = GCNModel([40, 64, 24, 7], structure=c, norm_groups=4, activation=activation).cuda()
    assert isinstance(model.norms[0], GroupNorm)
    x = _normal(1, n, 40)
    labels = torch.randint(-1, 7, (n,), device="cuda", generator=_gen(3))
    cut = n // 3
    ptr = torch.tensor([0, cut, n], device="cuda")
    r = model.log_probs(x, ei, labels, top=2, ptr=ptr)
    loss = -r.log_prob.mean() + 0.01 * r.entropy.mean()
    weights = [layer.lin.weight for layer in model.layers]
    before = [w.detach().double() for w in weights]
    opt = OrthogonalSGD(weights, lr=0.1, momentum=0.9)
    loss.backward()

    leaves = [w.detach().double().requires_grad_(True) for w in weights]
    h = x.double()
    for i, w in enumerate(leaves):
        h = a @ (h @ w.t())
        if i < 2:
            parts = [h[:cut], h[cut:]]
            h = torch.cat([((p.view(len(p), 4, -1) - p.view(len(p), 4, -1).mean((0, 2), keepdim=True))
                            / (p.view(len(p), 4, -1).var((0, 2), keepdim=True, correction=0) + 1e-5).sqrt()).reshape(p.shape) for p in parts])
            h = h.relu() if activation == "relu" else torch.nn.functional.silu(h)
    lp = torch.log_softmax(h, 1)
    picked = torch.where(labels >= 0, lp.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0.0)
    want = -picked.mean() + 0.01 * -(lp.exp() * lp).sum(1).mean()
    grads = torch.autograd.grad(want, leaves)
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())   # the framework's tolerance for its layers
    for w, g in zip(weights, grads):
        assert (w.grad.double() - g).norm() <= 1e-4 * g.norm()
    opt.step()
    for w, w0, g in zip(weights, before, grads):
        # of the update itself: the gradients' error is led through the products by at most 3.4445^5
        m = w.grad.double()
        o, bound = ortho64(m + 0.9 * m, 5)
        f = 0.1 * max(1.0, w.size(0) / w.size(1)) ** 0.5
        assert (w.detach().double() - (w0 - f * o)).norm() <= f * bound + 2.0 ** -23 * w0.norm()


def test_a_normed_model_by_itself_is_one_graph():
    ei, c, _ = _graph()
    model = GCNModel([40, 64, 7], structure=c, norm_groups=8).cuda()
    x = _normal(1, c.num_rows, 40)
    with torch.no_grad():
        y = model(x, ei)
        h = group_norm(model.layers[0](x, ei), 8, activation="relu")
        assert torch.equal(y, model.layers[1](h, ei))
        # given as a list of one graph it goes another way, whose sums are ordered otherwise: each is within its bound of the same values
        first = model.layers[0](x, ei)
        ptr = torch.tensor([0, c.num_rows], device="cuda")
        listed = group_norm(first, 8, activation="relu", ptr=ptr)
        for got in (h, listed):
            want, bound = norm64(first, 8, None, None, [0, c.num_rows], 1e-5, "relu", y=got)
            assert_within(got, want["y"], bound["y"])
        assert torch.equal(model(x, ei, ptr=ptr), model.layers[1](listed, ei))
