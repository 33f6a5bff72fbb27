"""The operators around a stack in 64 bits, and how far 32-bit arithmetic may be off them.

Bounds are sums of roundings.  U = 2^-24 is half a step of fp32.  A sum of L terms in fp32 is off by at most L U times the sum of
their magnitudes; the kernels add at most a few hundred terms one after the other in one register, whose errors are
independent, so 64 U stands for the square root of a depth of up to 4 096.  An output in fewer bits is off by half a step of its type more.
"""
import torch

U = 2.0 ** -24
SUM = 64 * U


def half_step(t):
    return torch.finfo(t).eps / 2


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound element by element; infinities and NaN have to be the same."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(same | (off <= bound))
    assert not bad.any(), (what, int(bad.sum()), off[bad][:4].tolist(), torch.as_tensor(bound, device=off.device).expand_as(off)[bad][:4].tolist(),
                           bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------ classes
def classes64(logits, labels, top, g_log=None, g_entropy=None, g_top=None):
    """Results and gradient, and their bounds."""
    x = logits.detach().double()
    n, c = x.shape
    m = x.max(1, keepdim=True).values
    closed = (m == -torch.inf)[:, 0]
    d = x - m  # (first: a logsumexp of the lowest values would be rounded to their magnitude)
    lp = d - torch.logsumexp(d, 1, keepdim=True)
    lp = torch.where(closed[:, None], -torch.inf, lp)
    lp = torch.where((x.isnan() | (x == torch.inf)).any(1, keepdim=True), torch.nan, lp)
    p = torch.exp(lp)
    entropy = -(p * torch.where(p == 0, 0.0, lp)).sum(1)
    known, wrong = labels >= 0, labels >= c
    at = labels.long().clamp(0, c - 1)[:, None]
    log_prob = torch.where(known, lp.gather(1, at)[:, 0], 0.0)
    log_prob = torch.where(wrong, torch.nan, log_prob)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    best = lp.gather(1, order)
    # x - m rounds once, log1p(s) twice; s is a sum of terms that are off by exp's 2 steps and their argument's rounding, of which
    # only the terms that count weigh (entropy).
    depth = SUM + U * (8 + 4 * entropy.nan_to_num(0.0))
    out = dict(log_prob=log_prob, entropy=entropy, top=best, classes=order)
    near = lambda v: 4 * U * torch.where(v.isfinite(), v.abs(), 0.0)  # noqa: E731
    bound = dict(log_prob=near(log_prob) + depth, entropy=4 * depth * (1 + entropy.nan_to_num(0.0)), top=near(best) + depth[:, None])
    if g_log is None and g_entropy is None and g_top is None:
        return out, bound
    zero = x.new_zeros(n)
    gl = torch.where(wrong, torch.nan, torch.where(known, g_log.double(), 0.0)) if g_log is not None else zero
    ge = g_entropy.double() if g_entropy is not None else zero
    gt = g_top.double() if g_top is not None else x.new_zeros((n, top))
    safe = torch.where(p == 0, 0.0, lp)
    gx = -p * (gl + gt.sum(1) + ge * entropy)[:, None] - ge[:, None] * p * safe
    gx = gx.scatter_add(1, at, gl[:, None]).scatter_add(1, order, gt)
    gx = torch.where(closed[:, None], 0.0, gx)
    size = gl.abs() + gt.abs().sum(1) + ge.abs() * (1 + entropy)
    relative = 2 * depth[:, None] + 8 * U * (1 + safe.abs())
    extra = torch.zeros_like(x).scatter_add(1, at, gl.abs()[:, None]).scatter_add(1, order, gt.abs())
    bound["gx"] = relative * p * (size[:, None] + ge.abs()[:, None] * safe.abs()) + 8 * U * extra + 2 * half_step(logits.dtype) * gx.abs() + smallest(logits.dtype)
    out["gx"] = gx
    return out, bound


def smallest(t):
    """Half a step below the normal numbers, where steps no longer shrink (and 32-bit products of exp go to 0)."""
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -126


# --------------------------------------------------------------------------------------------------- norm
def segments(x, ptr):
    """Sample of every row (their number: none), in the order that ptr gives."""
    n = x.shape[0]
    row = torch.full((n,), len(ptr) - 1, dtype=torch.int64, device=x.device)
    for s, (a, b) in enumerate(zip(ptr[:-1], ptr[1:])):
        row[a:b] = s
    return row


def norm64(x, groups, weight, bias, ptr, eps, activation, gy=None, y=None):
    """``ptr``: a list.  Results, gradients and their bounds; the ReLU's mask is taken from ``y`` where that is given and z is
    within its own bound of 0."""
    kind, row, samples = x.dtype, segments(x, ptr), len(ptr) - 1
    n, c = x.shape
    width = c // groups
    v = x.detach().double()
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
    size = (torch.bincount(row, minlength=samples + 1)[:, None] * width).clamp_min(1).double()

    def mean(t):
        s = t.reshape(n, groups, width).sum(2)
        return (torch.zeros((samples + 1, groups), dtype=torch.float64, device=x.device).index_add(0, row, s) / size)[row].repeat_interleave(width, 1)

    inside = (row < samples)[:, None]
    d = v - mean(v)
    r = (mean(d * d) + eps).rsqrt()
    xh = d * r
    z = xh * w + b
    # mean, then variance (a sum of squares around the mean), then four roundings
    d_xh = r * (SUM * mean(v.abs()) + 2 * U * v.abs()) + (SUM + 8 * U) * xh.abs()
    d_z = w.abs() * d_xh + 4 * U * (z.abs() + b.abs())
    sg = torch.sigmoid(z)
    if activation == "silu":
        out, slope = z * sg, sg * (1 + z * (1 - sg))
        d_out, d_slope = 1.1 * d_z + 8 * U * out.abs(), 0.5 * d_z + 16 * U * (1 + z.abs()) * sg
    elif activation == "relu":
        mask = z > 0 if y is None else torch.where(z.abs() <= d_z, y > 0, z > 0)
        out, slope, d_out, d_slope = torch.where(mask, z, 0.0), mask.double(), d_z, torch.zeros_like(z)
        if y is not None:
            d_out = d_out + torch.where(mask != (z > 0), z.abs(), 0.0)
    else:
        out, slope, d_out, d_slope = z, torch.ones_like(z), d_z, torch.zeros_like(z)
    res = dict(y=torch.where(inside, out, 0.0))
    bound = dict(y=d_out + half_step(kind) * out.abs() * 1.01 + smallest(kind))
    if gy is None:
        return res, bound
    gy = torch.where(inside, gy.double(), 0.0)
    g = gy * slope
    u, d_g = g * w, gy.abs() * d_slope + 2 * U * g.abs()
    d_u = d_g * w.abs()
    mu, mux = mean(u), mean(u * xh)
    res["gx"] = r * (u - mu - xh * mux)
    inner = d_u + SUM * mean(u.abs()) + mean(d_u) + xh.abs() * (SUM * mean((u * xh).abs()) + mean(d_u * xh.abs() + u.abs() * d_xh)) + d_xh * mux.abs()
    bound["gx"] = r * inner + (SUM + 8 * U + 2 * half_step(kind)) * r * (u.abs() + mu.abs() + (xh * mux).abs()) + smallest(kind)
    res["gw"], res["gb"] = (g * xh).sum(0), g.sum(0)
    bound["gw"] = ((SUM + 8 * U) * (g * xh).abs() + d_g * xh.abs() + g.abs() * d_xh).sum(0) + 1e-30
    bound["gb"] = (SUM * g.abs() + d_g).sum(0) + 1e-30
    return res, bound


# ------------------------------------------------------------------------------------------------- update
QUINTIC = (3.4445, -4.7750, 2.0315)


def ortho64(u, steps, eps=1e-7):
    """The result for one matrix, and a bound on the 2-norm of its error: what a step rounds (8 U of its result, as its products have
    sums of up to a few thousand terms) grows by at most |a| = 3.4445, the steepest slope of the quintic, with every step that follows."""
    a, b, c = QUINTIC
    turned = u.shape[0] > u.shape[1]
    x = (u.t() if turned else u).double()
    x = x / (x.norm() + eps)
    bound = 8 * U * x.norm()
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * g @ g) @ x
        bound = a * bound + 8 * U * x.norm()
    return (x.t() if turned else x), bound
