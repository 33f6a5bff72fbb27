"""The operators around a stack on the GPU at the edges of what their documentation allows, against their 64-bit forms."""
import pytest
import torch

from cbm4gnn_b200.classify import class_log_probs
from cbm4gnn_b200.norm import group_norm
from cbm4gnn_b200.optim import OrthogonalSGD, orthogonal_step, orthogonalise

from operators64 import SUM, U, assert_within, classes64, half_step, norm64, ortho64, smallest

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


# --------------------------------------------------------------------------------- groups wider than a block
def _check_norm(x, groups, ptr, activation, kind=None, close=False):
    """``close``: of a mean far from 0 no more may be lost than its one rounding, and that of x - mean."""
    c = x.size(-1)
    leaves = [t.to(kind or x.dtype).requires_grad_(True) for t in (_normal(1, c) + 1, _normal(2, c))]
    x = x.detach().requires_grad_(True)
    gy = _normal(3, *x.shape).to(x.dtype)
    on = None if ptr is None or x.dim() == 3 else torch.tensor(ptr, device="cuda")
    y = group_norm(x, groups, *leaves, ptr=on, activation=activation)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, (x, *leaves), gy)))
    n = x.numel() // c
    flat = x.detach().reshape(n, c)
    rows = ptr or [0, n]
    want, bound = norm64(flat, groups, *leaves, rows, 1e-5, activation, gy.reshape(n, c), y.detach().reshape(n, c))
    assert_within(y.detach().reshape(n, c), want["y"], bound["y"], "y")
    assert_within(got["gx"].reshape(n, c), want["gx"], bound["gx"], "gx")
    for k in ("gw", "gb"):  # (rounded to the parameter's type: half a step of the value, 2^-25 below the normal numbers of fp16)
        assert_within(got[k], want[k], bound[k] + half_step(got[k].dtype) * want[k].abs() + smallest(got[k].dtype), k)
    if close:
        assert activation is None and rows == [0, n] and x.dtype == torch.float32
        v = flat.double().view(n, groups, -1)
        mean, r = v.mean((0, 2), keepdim=True), (v.var((0, 2), keepdim=True, correction=0) + 1e-5).rsqrt()
        w, b = (t.detach().double().view(1, groups, -1) for t in leaves)
        xh = (v - mean) * r
        near = w.abs() * (r * 2 * U * mean.abs() + (SUM + 8 * U) * xh.abs()) + 4 * U * ((xh * w + b).abs() + b.abs())
        assert_within(y.detach().view(n, groups, -1), xh * w + b, near, "y beside a large mean")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,groups,ptr", [
    (1, 2049, 1, None), (300, 2049, 1, None), (150, 4100, 2, None), (90, 8200, 2, None), (40, 12_300, 3, [0, 0, 7, 7, 30, 40]), (64, 4096, 1, [3, 20, 20, 50]),
    (30, 2051, 1, [30, 30]), (30, 2500, 1, [0, 0]), (33, 9000, 1, list(range(34)))])
def test_norm_of_wide_groups(kind, n, c, groups, ptr):
    _check_norm((_normal(n, n, c) * 1.5 + 0.4).to(kind), groups, ptr, "silu", kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("b,n,c,groups", [(50, 1, 1100, 1), (37, 1, 4096, 1), (9, 1, 8200, 2), (7, 1, 9000, 1), (5, 1, 4095, 1), (6, 9, 4100, 1), (3, 20, 5000, 2)])
def test_norm_of_equal_samples_of_wide_groups(kind, b, n, c, groups):
    _check_norm((_normal(b, b, n, c) - 0.7).to(kind), groups, list(range(0, b * n + 1, n)), "relu")


@pytest.mark.parametrize("n,c,groups,mean", [(6000, 4096, 1, 1000.0), (10_000, 2304, 1, 100.0), (3000, 5000, 2, -3.0)])
def test_norm_of_wide_groups_keeps_digits_beside_a_large_mean(n, c, groups, mean):
    _check_norm(mean + _normal(5, n, c), groups, None, None, close=True)


@pytest.mark.parametrize("n,c,groups,ptr", [(40, 24, 6, [3, 10, 10, 30]), (5000, 64, 8, [100, 4000, 4010, 4500]), (60, 2500, 1, [2, 30, 50])])
def test_norm_rows_of_no_sample_may_hold_anything(n, c, groups, ptr):
    x = _normal(1, n, c)
    x[:ptr[0]], x[ptr[-1]:] = torch.nan, torch.inf
    clean = x.clone()
    clean[:ptr[0]] = clean[ptr[-1]:] = 0.0
    on, gy = torch.tensor(ptr, device="cuda"), _normal(4, n, c)
    found = []
    for t in (x, clean):
        leaves = [t.requires_grad_(True), _normal(2, c).requires_grad_(True), _normal(3, c).requires_grad_(True)]
        y = group_norm(leaves[0], groups, *leaves[1:], ptr=on, activation="silu")
        found.append((y.detach(), *torch.autograd.grad(y, leaves, gy)))
    for a, b in zip(*found):
        assert torch.equal(a, b)
    for t in found[0][:2]:
        assert t[:ptr[0]].eq(0).all() and t[ptr[-1]:].eq(0).all()


@pytest.mark.parametrize("n,c,groups", [(9, 12, 4), (3000, 64, 8), (40, 2500, 1)])
def test_norm_of_rows_without_samples(n, c, groups):
    """A list of no graphs: no row belongs to one."""
    x, w, b = (t.requires_grad_(True) for t in (_normal(1, n, c), _normal(2, c), _normal(3, c)))
    y = group_norm(x, groups, w, b, ptr=torch.zeros(1, dtype=torch.int64, device="cuda"), activation="silu")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), _normal(4, n, c))
    assert y.shape == x.shape and all(t.eq(0).all() for t in (y, gx, gw, gb))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("c,top", [(2, 1), (7, 3), (47, 0), (200, 2), (600, 5), (1300, 3), (20_000, 4)])
@pytest.mark.parametrize("grads", [(True, False, False), (True, True, True), (False, False, True)])
def test_gradients_of_decided_rows_keep_their_digits(kind, c, top, grads):
    """Where one class has all but 1e-9 to 1e-3 of a row, what is left of its own gradient is a product with 1 - p, not a difference."""
    n = 16
    lead = torch.linspace(7.0, 20.0, n, device="cuda") + torch.tensor(float(c)).log().cuda()
    lead = lead.clamp_max(27.0)
    for pitch, first in ((c, 0), (c + 3, 1)):
        wide = torch.zeros((n, pitch), dtype=kind, device="cuda")
        wide[:, first:first + c] = (0.5 * _normal(c, n, c)).to(kind)
        x = wide[:, first:first + c]
        labels = torch.arange(n, device="cuda") * 7 % c
        x[torch.arange(n), labels] = lead.to(kind)
        x = x.detach().requires_grad_(True)
        given = [_normal(9 + i, *s) if on and s[-1] else None for i, (on, s) in enumerate(zip(grads, ((n,), (n,), (n, top))))]
        r = class_log_probs(x, labels, top=top)
        used = [(o, g) for o, g in zip(r[:3], given) if g is not None]
        if not used:
            continue
        gx, = torch.autograd.grad([o for o, _ in used], x, [g for _, g in used])
        want, bound = classes64(x, labels, top, *given)
        # terms of 1 - p: arguments of up to 30 rounded once, exp's 2 steps and as many of its own argument, the sum, some operations more
        d = x.detach().double() - x.detach().double().gather(1, labels[:, None])
        left = torch.exp(d).scatter(1, labels[:, None], 0.0).sum(1)
        left, own = left / (1 + left), labels[:, None]
        zero = torch.zeros(n, dtype=torch.float64, device="cuda")
        gl, ge = (zero if g is None else g.double() for g in given[:2])
        gt = zero[:, None] if given[2] is None else given[2].double()
        near = (SUM + 128 * U) * (gl.abs() * left + gt[:, 0].abs() * left + ge.abs() * (want["entropy"] + left)) + 8 * U * gt[:, 1:].abs().sum(1)
        near = near + 2 * half_step(kind) * want["gx"].gather(1, own)[:, 0].abs() + smallest(kind)
        assert_within(gx, want["gx"], bound["gx"].scatter(1, own, near[:, None]), "gx")


# ------------------------------------------------------------------------------------------------- update
def test_step_of_a_turned_row():
    """A weight of one column may have any column stride: torch calls it contiguous, whatever it was made from."""
    for m in (5, 300):
        w, g, mom = (_normal(i, 1, m).t() for i in range(3))
        assert w.stride() == (1, m) and w.is_contiguous()
        m1 = 0.9 * mom.double() + g.double()
        o, bound = ortho64(g.double() + 0.9 * m1, 5)
        want = w.double() - 0.1 * m ** 0.5 * o
        orthogonal_step([w], [g], [mom], lr=0.1, momentum=0.9)
        assert (w.double() - want).norm() <= 0.1 * m ** 0.5 * bound + 2.0 ** -23 * want.norm()
        assert torch.allclose(mom.double(), m1, atol=1e-6, rtol=1e-6)
        assert (orthogonalise(g).double() - ortho64(g, 5)[0]).norm() <= ortho64(g, 5)[1]
    p = torch.nn.Parameter(_normal(7, 1, 40).t())
    p.grad = _normal(8, 40, 1)
    before = p.detach().clone()
    OrthogonalSGD([p], lr=0.1).step()
    assert (p.detach() - before).norm() > 0.1
    with pytest.raises(RuntimeError, match="unit column stride"):
        orthogonal_step([_normal(1, 6, 4).t()], [_normal(2, 4, 6)], [_normal(3, 4, 6)], lr=0.1)


# ------------------------------------------------------------------------------------------------- limits
def test_sizes_past_the_limits_are_refused_by_name():
    """Before anything is copied or counted in 32 bits; the operands are broadcasts of one value."""
    one = torch.ones((1, 1), device="cuda")
    labels = torch.zeros(1, dtype=torch.int64, device="cuda")
    for c in ((1 << 22) + 4, (1 << 32) + 4):
        with pytest.raises(RuntimeError, match=f"{c} channels, at most {1 << 22}"):
            group_norm(one.expand(1, c), 2)
        with pytest.raises(RuntimeError, match=f"{c} channels, at most {1 << 22}"):
            group_norm(one.expand(1, c), 2, ptr=labels)
    for c in ((1 << 30) + 1, (1 << 32) + 4):
        with pytest.raises(RuntimeError, match=f"{c} classes, at most {1 << 30}"):
            class_log_probs(one.expand(1, c), labels)
    for m, n in ((65_537, 3), (3, 65_537), ((1 << 32) + 5, 7), (7, (1 << 32) + 5)):
        with pytest.raises(RuntimeError, match="65536"):
            orthogonalise(one.expand(m, n))
        with pytest.raises(ValueError, match=f"{m} x {n}, sides of at most 65536"):
            OrthogonalSGD([torch.nn.Parameter(one.expand(m, n))])
    with pytest.raises(RuntimeError, match="stacks of at most 32768"):
        orthogonalise(one.expand(32_769, 2, 2))
    w, fine = torch.zeros((65_537, 2), device="cuda"), torch.ones((4, 4), device="cuda")
    with pytest.raises(RuntimeError, match="65537 x 2"):
        orthogonal_step([fine, w], [fine.clone(), w.clone()], [torch.zeros_like(fine), w.clone()], lr=0.1)
    assert fine.eq(1).all()
    tall = _normal(1, 65_536, 2)
    want, bound = ortho64(tall, 5)
    assert (orthogonalise(tall).double() - want).norm() <= bound


def _low_update(seed, m, n, by_rows, powers):
    """A random update of which an eighth of the rows (or columns) lies lower, for each of the powers."""
    u = _normal(seed, m, n)
    side = m if by_rows else n
    scale = torch.ones(side, device="cuda")
    for k, power in enumerate(powers):
        scale[k * side // 8:(k + 1) * side // 8] = power
    return u * (scale[:, None] if by_rows else scale[None, :])


def _stretch_bound(u, by_rows, floor):
    """The result in 64 bits, and how far each row (or column) of it may be off.

    A step: what is there grows by at most a.  New: values stored, products without their smallest part, and their sums, each some 2^-22
    of a row of |X| or |B| times |X|, whose norm is at most that of the row times the root of the shorter side (16 of them); and where
    two fp16 terms hold the operands the floor of 2^-37 under a row's entries, and under those of A (b and 2 c times, times X,
    whose norm is 1.21) and B."""
    m, n = u.shape
    turned = m > n
    x = u.double()
    x = x / (x.norm() + 1e-7)
    x = x.t() if turned else x
    along = 1 if by_rows != turned else 0   # rows, or columns, of x
    a, b, c = 3.4445, -4.7750, 2.0315
    short, length = min(m, n), x.size(along)
    off = torch.zeros(x.size(1 - along), dtype=torch.float64, device="cuda")
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * g @ g) @ x
        off = a * off + 16 * 2.0 ** -22 * short ** 0.5 * x.norm(dim=along)
        if floor:
            off = off + 2.0 ** -37 * (2 * length ** 0.5 + (12 * short ** 0.5 if along == 1 else 0.0))
    return (x.t() if turned else x), off


@pytest.mark.parametrize("m,n", [(128, 512), (100, 900), (30, 20), (300, 700), (500, 400), (1600, 1500), (65, 1100), (129, 129)])
@pytest.mark.parametrize("by_rows", [True, False])
@pytest.mark.parametrize("powers", [(1e-3,), (1e-4, 1e-5), (1e-7,), (1e-5, 1e-9, 1e-20), (0.0, 1e-12)])
def test_low_rows_and_columns_of_an_update_keep_their_digits(m, n, by_rows, powers):
    """Whatever lies beside them: down to 2^-24 of the norm in two fp16 terms, whose floor is 2^-37 of it, below that in fp32."""
    u = _low_update(m + n, m, n, by_rows, powers)
    along = 1 if by_rows else 0
    got = orthogonalise(u).double()
    want, off = _stretch_bound(u, by_rows, floor=min(p for p in powers if p) > 1e-6)
    wrong = (got - want).norm(dim=along)
    assert (wrong <= off).all(), (wrong / off).max()


def test_low_blocks_stacks_lists_and_replays():
    """Matrices that go by fp32 products beside others that do not."""
    stack = torch.stack([_low_update(i, 200, 330, True, (1e-9,) if i in (1, 4) else ()) for i in range(5)])
    got = orthogonalise(stack)
    for i in range(5):
        want, off = _stretch_bound(stack[i], True, floor=False)
        assert ((got[i].double() - want).norm(dim=1) <= off + (0 if i in (1, 4) else 2.0 ** -30)).all()
        assert torch.equal(got[i], orthogonalise(stack[i]))
    small = torch.stack([_low_update(i, 90, 60, False, (1e-9,) if i == 2 else ()) for i in range(4)])
    for i, o in enumerate(orthogonalise(small)):
        assert torch.equal(o, orthogonalise(small[i]))
    tiny = _normal(9, 40, 300) * 1e-13     # all of it far below eps
    for u in (tiny, _normal(8, 400, 300) * 1e-13):
        want, off = _stretch_bound(u, True, floor=False)
        assert ((orthogonalise(u).double() - want).norm(dim=1) <= off).all()
    shapes = [(64, 100), (300, 200), (128, 128), (16, 600), (500, 64), (90, 1000)]
    for chosen in (shapes, [s for s in shapes if min(s) <= 128 and max(s) <= 1024]):   # tiles beside one another, clusters
        ws = [_normal(i, *s) for i, s in enumerate(chosen)]
        gs = [_low_update(10 + i, *s, i % 2 == 0, (1e-10, 1e-6) if i % 3 else ()) for i, s in enumerate(chosen)]
        ms = [_low_update(30 + i, *s, i % 2 == 0, (1e-10, 1e-6) if i % 3 else ()) for i, s in enumerate(chosen)]
        start = [t.clone() for t in ws + ms]
        graph = torch.cuda.CUDAGraph()
        step = lambda: orthogonal_step(ws, gs, ms, lr=0.05, momentum=0.9)  # noqa: E731, B023
        step()
        after = [t.clone() for t in ws + ms]
        for w, w0, g, m0 in zip(ws, start, gs, start[len(ws):]):
            m1 = 0.9 * m0.double() + g.double()
            o, bound = ortho64(g.double() + 0.9 * m1, 5)
            f = 0.05 * max(1.0, w.size(0) / w.size(1)) ** 0.5
            assert (w.double() - (w0.double() - f * o)).norm() <= f * (bound + 2e-4 * 2.0 ** -3) + 2.0 ** -23 * w0.double().norm()
        with torch.cuda.graph(graph):
            step()
        for to, of in zip(ws + ms, start):
            to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(after, ws + ms))
