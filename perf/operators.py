"""Performance cases of the operators around a GCN stack: what lies between two layers (group norm with an activation),
what its logits are turned into (class log probabilities with entropy and runner-up classes, and their gradient), and
what its weight gradients are turned into (the orthogonalised update).

``listed()`` names the fixed cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one pass, ``work`` the bytes and operations that it cannot do without,
``exact`` the same outputs from the definitions in 64 bits.  Where ``own`` is false, ``run`` computes the plain form.
"""
from __future__ import annotations

import math

import torch

own = False

STEPS = 5
QUINTIC = (3.4445, -4.7750, 2.0315)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A graph of a thousand nodes between two narrow layers: only latency counts.
        dict(name="norm_small", op="norm", n=1000, c=64, groups=8, samples="one", act="relu", type="fp32", train=False),
        # Hidden layer of the 128-256-64 training configuration: one graph, both directions.
        dict(name="norm_graph_train", op="norm", n=235_868, c=256, groups=32, samples="one", act="silu", type="fp32", train=True),
        # A batch of small graphs of uneven sizes, some empty, padded behind the last; 100 channels by tens.
        dict(name="norm_batch_train", op="norm", n=262_147, c=100, groups=10, samples="ragged", mean_rows=30, act="silu", type="bf16",
             train=True),
        # Inference over the nodes of the 100-256-256-47 configuration, every node by itself.
        dict(name="norm_nodes", op="norm", n=2_449_029, c=256, groups=16, samples="rows", act="relu", type="fp16", train=False),
        # Scores of a small citation graph's nodes: 7 classes, the 3 best of them.
        dict(name="classes_small", op="classes", n=4096, c=7, top=3, type="fp32", masked=False, train=False),
        # Loss and its gradient over all nodes of the 100-256-256-47 configuration, a part of them without a label.
        dict(name="classes_train", op="classes", n=2_449_029, c=47, top=0, type="fp32", masked=False, train=True),
        # A few rows over a very large vocabulary, with alternatives: the scores of one step of an answer.
        dict(name="classes_long", op="classes", n=16, c=128_256, top=20, type="bf16", masked=True, train=False),
        # Loss and gradient over a large vocabulary, odd sizes, rows that are not 16-byte aligned.
        dict(name="classes_wide_train", op="classes", n=4099, c=50_257, top=0, type="bf16", masked=True, train=True),
        # Update of the 500-64-7 stack: latency.
        dict(name="update_small", op="update", shapes="64x500,7x64"),
        # Update of the 100-256-256-47 stack.
        dict(name="update_gcn", op="update", shapes="256x100,256x256,47x256"),
        # A stack of equal matrices, taller than wide, odd sizes.
        dict(name="ortho_batch", op="ortho", b=12, m=777, n=500),
        # One large matrix.
        dict(name="ortho_large", op="ortho", b=1, m=2048, n=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "classes", "classes", "update", "ortho"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.5
    if op == "norm":
        c, samples = _log(rng, 4, 1100), rng.choice(["one", "ragged", "rows"])
        n = min(_log(rng, 100, 400_000), 60_000_000 // c)
        groups = rng.choice([g for g in range(1, c + 1) if c % g == 0 and g <= 64 and c // g > 1])
        case = dict(op=op, n=n, c=c, groups=groups, samples=samples, act="silu" if train else rng.choice(["none", "relu", "silu"]),
                    type=kind, train=train)
        if samples == "ragged":
            case["mean_rows"] = _log(rng, 4, 5000)
        return case
    if op == "classes":
        c = _log(rng, 2, 140_000)
        n = max(1, min(_log(rng, 1, 400_000), 100_000_000 // c))
        return dict(op=op, n=n, c=c, top=min(c, rng.choice([0, 1, 3, 10, 32])), type=kind, masked=rng.random() < 0.5, train=train)
    if op == "update":
        widths = [_log(rng, 16, 600) for _ in range(rng.randint(1, 3))] + [_log(rng, 4, 64)]
        widths = [_log(rng, 16, 600)] + widths
        return dict(op=op, shapes=",".join("%dx%d" % (b, a) for a, b in zip(widths[:-1], widths[1:])))
    m, n = _log(rng, 16, 2048), _log(rng, 16, 2048)
    return dict(op=op, b=rng.choice([1, 1, 2, 5]), m=m, n=n)


# --------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _shapes(case):
    return [tuple(map(int, s.split("x"))) for s in case["shapes"].split(",")]


def _gradient(g, m, n):
    """A weight gradient as training gives it: a few strong directions over noise."""
    r = max(1, min(m, n) // 8)
    strong = _normal(g, m, r) @ (_normal(g, r, n) * torch.linspace(2.0, 0.2, r, device="cuda")[:, None])
    return (strong / math.sqrt(r) + 0.5 * _normal(g, m, n)) * 1e-3


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "norm":
        n, c, kind = case["n"], case["c"], TYPES[case["type"]]
        channel = 0.5 * _normal(g, c)
        x = (_normal(g, n, c) * (1.0 + 0.3 * _normal(g, c).abs()) + channel).to(kind)
        state = dict(case=case, weight=1.0 + 0.2 * _normal(g, c), bias=0.2 * _normal(g, c), ptr=None)
        if case["samples"] == "rows":
            x = x.view(n, 1, c)
        elif case["samples"] == "ragged":
            mean = case["mean_rows"]
            count = max(1, n // mean)
            size = (torch.exp(0.8 * _normal(g, count) - 0.32) * mean).long().clamp_min(1)
            size[torch.rand(count, device="cuda", generator=g) < 0.03] = 0
            state["ptr"] = torch.cat([size.new_zeros(1), size.cumsum(0)]).clamp_max(n - n // 64)
        state["x"] = x
        if case["train"]:
            state["gy"] = _normal(g, *x.shape).to(kind)
            for leaf in ("x", "weight", "bias"):
                state[leaf].requires_grad_(True)
        return state
    if op == "classes":
        n, c, kind = case["n"], case["c"], TYPES[case["type"]]
        sure = torch.exp(0.7 * _normal(g, n, 1) + 0.5)  # some rows are nearly decided, some are flat
        logits = (_normal(g, n, c) * sure).to(kind)
        labels = torch.randint(0, c, (n,), device="cuda", generator=g)
        if case["masked"]:
            closed = torch.rand((n, c), device="cuda", generator=g) < 0.1
            closed.scatter_(1, labels[:, None], False)
            logits.masked_fill_(closed, -math.inf)
            del closed
        labels[torch.rand(n, device="cuda", generator=g) < 0.1] = -100
        state = dict(case=case, logits=logits, labels=labels)
        if case["train"]:
            logits.requires_grad_(True)
            state["g_log_prob"] = torch.full((n,), -1.0 / n, device="cuda")
            state["g_entropy"] = torch.full((n,), -0.01 / n, device="cuda")
            state["g_top"] = _normal(g, n, case["top"]) / n
        return state
    if op == "update":
        shapes = _shapes(case)
        return dict(case=case, weights=[_normal(g, *s) / math.sqrt(s[1]) for s in shapes], grads=[_gradient(g, *s) for s in shapes],
                    momenta=[5.0 * _gradient(g, *s) for s in shapes])
    update = torch.stack([_gradient(g, case["m"], case["n"]) for _ in range(case["b"])])
    return dict(case=case, update=update if case["b"] > 1 else update[0])


# ------------------------------------------------------------------------------------------ plain forms
def _samples(state, n):
    """For every row its sample, for every sample its rows; rows of no sample get the last number."""
    ptr = state["ptr"]
    count = ptr.numel() - 1
    row = torch.searchsorted(ptr, torch.arange(n, device=ptr.device), right=True) - 1
    row[(row < 0) | (row >= count)] = count
    return row, torch.cat([ptr[1:] - ptr[:-1], ptr.new_zeros(1)])


def _plain_norm(state):
    case = state["case"]
    x, c, groups, act = state["x"].detach().float(), case["c"], case["groups"], case["act"]
    width = c // groups
    weight, bias = state["weight"].detach(), state["bias"].detach()
    if state["ptr"] is None:
        by = x.reshape(-1 if x.dim() == 3 else 1, 1 if x.dim() == 3 else x.size(0), groups, width)

        def mean(v):
            return v.reshape(by.shape).mean(dim=(1, 3), keepdim=True).expand(by.shape).reshape(x.shape)
    else:
        row, rows = _samples(state, x.size(0))
        size = (rows.double() * width).clamp_min(1.0)[:, None]

        def mean(v):
            of_row = v.view(-1, groups, width).sum(2, dtype=torch.float64)
            of_sample = torch.zeros((rows.numel(), groups), dtype=torch.float64, device=v.device).index_add_(0, row, of_row)
            return (of_sample / size).float()[row].repeat_interleave(width, dim=1)
    inside = 1.0 if state["ptr"] is None else (row < rows.numel() - 1).float()[:, None]
    centred = x - mean(x)
    r = torch.rsqrt(mean(centred * centred) + 1e-5)
    xh = centred * r
    z = xh * weight + bias
    s = torch.sigmoid(z) if act == "silu" else None
    y = z * s if act == "silu" else z.clamp_min(0.0) if act == "relu" else z
    y = (y * inside).to(state["x"].dtype)
    if not case["train"]:
        return dict(y=y)
    g = state["gy"].float() * inside
    g = g * (s * (1.0 + z * (1.0 - s))) if act == "silu" else g * (z > 0) if act == "relu" else g
    u = g * weight
    gx = r * (u - mean(u) - xh * mean(u * xh))
    flat = (-1, c)
    return dict(y=y, gx=gx.to(y.dtype), gw=(g * xh).reshape(flat).sum(0), gb=g.reshape(flat).sum(0))


def _plain_classes(state):
    case, k = state["case"], state["case"]["top"]
    x, labels = state["logits"].detach().float(), state["labels"]
    known = labels >= 0
    at = labels.clamp_min(0)[:, None]
    top = x.max(dim=1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lp = (x - top) - torch.log(total)
    p = e / total
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plp.sum(1)
    log_prob = torch.where(known, lp.gather(1, at)[:, 0], 0.0)
    if k:
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    else:
        best = labels.new_empty((x.size(0), 0))
    out = dict(log_prob=log_prob, entropy=entropy, top=lp.gather(1, best), classes=best)
    if case["train"]:
        gl = torch.where(known, state["g_log_prob"], 0.0)[:, None]
        ge, gt = state["g_entropy"][:, None], state["g_top"]
        gx = -p * (gl + gt.sum(1, keepdim=True) + ge * entropy[:, None]) - ge * plp
        gx.scatter_add_(1, at, gl)
        gx.scatter_add_(1, best, gt)
        out["gx"] = gx.to(state["logits"].dtype)
    return out


def _plain_ortho(u):
    a, b, c = QUINTIC
    tall = u.size(-2) > u.size(-1)
    x = u.transpose(-1, -2) if tall else u
    x = x / (x.square().sum(dim=(-1, -2), keepdim=True).sqrt() + 1e-7)
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if tall else x


LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def _plain_update(state):
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        m.mul_(MOMENTUM).add_(g)
        o = _plain_ortho(g + MOMENTUM * m)
        w.mul_(1.0 - LR * DECAY).add_(o, alpha=-LR * math.sqrt(max(1.0, w.size(0) / w.size(1))))
    return dict(weights=state["weights"], momenta=state["momenta"])


# ------------------------------------------------------------------------------------------------ run
def _own(state):
    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        from cbm4gnn_b200.norm import group_norm
        y = group_norm(state["x"], case["groups"], state["weight"], state["bias"], ptr=state["ptr"],
                       activation=None if case["act"] == "none" else case["act"])
        if not case["train"]:
            return dict(y=y)
        gx, gw, gb = torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["gy"])
        return dict(y=y, gx=gx, gw=gw, gb=gb)
    if op == "classes":
        from cbm4gnn_b200.classify import class_log_probs
        r = class_log_probs(state["logits"], state["labels"], top=case["top"])
        out = dict(log_prob=r.log_prob, entropy=r.entropy, top=r.top_log_probs, classes=r.top_classes)
        if case["train"]:
            given = [(r.log_prob, state["g_log_prob"]), (r.entropy, state["g_entropy"])]
            if case["top"]:
                given.append((r.top_log_probs, state["g_top"]))
            out["gx"], = torch.autograd.grad([v for v, _ in given], state["logits"], [v for _, v in given])
        return out
    if op == "update":
        from cbm4gnn_b200.optim import orthogonal_step
        orthogonal_step(state["weights"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS)
        return dict(weights=state["weights"], momenta=state["momenta"])
    from cbm4gnn_b200.optim import orthogonalise
    return dict(x=orthogonalise(state["update"], steps=STEPS))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op == "norm":
            return _plain_norm(state)
        if op == "classes":
            return _plain_classes(state)
        if op == "update":
            return _plain_update(state)
        return dict(x=_plain_ortho(state["update"]))


# ----------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    size = {"fp32": 4, "bf16": 2, "fp16": 2}.get(case.get("type"), 4)
    if op == "norm":
        params = 8 * case["c"] * (2 if case["train"] else 1)
        return dict(bytes=(4 if case["train"] else 2) * size * case["n"] * case["c"] + params, flops=0)
    if op == "classes":
        rows = 8 + 4 + 4 + 12 * case["top"] + ((8 + 4 * case["top"]) if case["train"] else 0)
        return dict(bytes=(2 if case["train"] else 1) * size * case["n"] * case["c"] + rows * case["n"], flops=0)
    shapes = _shapes(case) if op == "update" else [(case["m"], case["n"])] * case["b"]
    values = flops = 0
    for rows, cols in shapes:
        m, n = min(rows, cols), max(rows, cols)
        values += m * n
        # the two symmetric products need one half and the diagonal
        flops += STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)
    return dict(bytes=4 * values * (5 if op == "update" else 2), flops=flops)


# ---------------------------------------------------------------------------------------------- exact
def _exact_norm(case, state):
    leaves = [state[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias")]
    x, weight, bias = leaves
    n, c, groups = case["n"], case["c"], case["groups"]
    v = x.reshape(n, groups, c // groups)
    if case["samples"] == "rows":
        var, mean = torch.var_mean(v, dim=2, keepdim=True, correction=0)
    elif case["samples"] == "one":
        var, mean = torch.var_mean(v, dim=(0, 2), keepdim=True, correction=0)
    else:
        ptr = state["ptr"]
        count = ptr.numel() - 1
        where = torch.bucketize(torch.arange(n, device="cuda"), ptr[1:], right=True)  # `count`: behind the last
        size = (torch.bincount(where, minlength=count + 1).double() * (c // groups)).clamp_min(1.0)[:, None]

        def over(t):
            return (torch.zeros((count + 1, groups), dtype=torch.float64, device="cuda").index_add(0, where, t.sum(2)) / size)[where][..., None]
        mean = over(v)
        var = over((v - mean).square())
    y = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(n, c) * weight + bias
    if case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif case["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    if case["samples"] == "ragged":
        y = torch.where((where < count)[:, None], y, 0.0)
    y = y.reshape(state["x"].shape)
    if not case["train"]:
        return dict(y=y.detach())
    gx, gw, gb = torch.autograd.grad(y, leaves, state["gy"].double())
    return dict(y=y.detach(), gx=gx, gw=gw, gb=gb)


def _exact_classes(case, state):
    """By blocks of rows: 64-bit copies of the largest cases would not fit three times over."""
    k, parts = case["top"], []
    logits, labels = state["logits"].detach(), state["labels"]
    for first in range(0, case["n"], max(1, 60_000_000 // case["c"])):
        rows = slice(first, first + max(1, 60_000_000 // case["c"]))
        x = logits[rows].double().requires_grad_(case["train"])
        lse = torch.logsumexp(x, dim=1)
        lp = x - lse[:, None]
        label = labels[rows]
        picked = torch.where(label >= 0, lp.gather(1, label.clamp_min(0)[:, None])[:, 0], 0.0)
        open_ = x.detach() > -math.inf
        safe = torch.where(open_, lp, 0.0)
        entropy = -(torch.exp(safe) * safe * open_).sum(1)
        best = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :k]
        top = lp.gather(1, best)
        part = dict(log_prob=picked.detach(), entropy=entropy.detach(), top=top.detach(), classes=best)
        if case["train"]:
            loss = (picked * state["g_log_prob"][rows].double()).sum() + (entropy * state["g_entropy"][rows].double()).sum()
            loss = loss + (top * state["g_top"][rows].double()).sum()
            part["gx"], = torch.autograd.grad(loss, x)
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _exact_ortho(u):
    a, b, c = QUINTIC
    u = u.double()
    # the same polynomial of the singular values, by products with the smaller Gram matrix on either side
    x = u / (torch.linalg.vector_norm(u) + 1e-7)
    for _ in range(STEPS):
        if x.size(0) <= x.size(1):
            gram = torch.mm(x, x.t())
            x = torch.mm(a * torch.eye(x.size(0), dtype=x.dtype, device=x.device) + b * gram + c * torch.mm(gram, gram), x)
        else:
            gram = torch.mm(x.t(), x)
            x = torch.mm(x, a * torch.eye(x.size(1), dtype=x.dtype, device=x.device) + b * gram + c * torch.mm(gram, gram))
    return x


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(case, state)
    if op == "classes":
        return _exact_classes(case, state)
    if op == "ortho":
        u = state["update"]
        return dict(x=_exact_ortho(u) if u.dim() == 2 else torch.stack([_exact_ortho(v) for v in u]))
    weights, momenta = [], []
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        m = MOMENTUM * m.double() + g.double()
        o = _exact_ortho(g.double() + MOMENTUM * m)
        weights.append((1.0 - LR * DECAY) * w.double() - LR * max(1.0, w.size(0) / w.size(1)) ** 0.5 * o)
        momenta.append(m)
    return dict(weights=weights, momenta=momenta)
