"""The router's losses, counts, weights and their gradient against float64.

Tolerances, derived before the first run.  u = 2^-24 is fp32's rounding.  An
exponential's argument l - m is off by |l - m| u and the exponential by a few u
itself, a row's sum of non-negative terms by at most 26 u (16 in a lane, six
joins, the rest for the division), so a probability or score is off by
R = (|l - m| + 40) u relative, with |l - m| up to D, the largest spread of a row.
A mean of p over rows adds at most (rows of a lane + 64) u <= 2^-17 relative
(the rest is in fp64), so P and the balance loss are off by R + 2^-17 relative (all terms
are non-negative).  lse is off by (|m| + log E + 40) u, z by 2 |lse| of that, plus its
sums.  A gradient's terms p (h_j - sum p h + z' - c) and w (g_k - sum w g) are
each off by 2 R + 16 u of the sum of their terms' magnitudes; 1 - s <= 1
multiplies them.  bf16 outputs: 2^-8 more.
"""
import math

import pytest
import torch

from xtu_moe_amd.layer import route
from xtu_moe_amd.router import router_losses

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24


def _inputs(T, E, K, seed=0, dtype=F32, std=1.5, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    lg = (torch.randn((T, E), generator=g) * std).to(dtype)
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :K].to(torch.int32)
    if drop:
        ids = torch.where(torch.rand((T, K), generator=g) < drop, -1, ids)
    gw = torch.randn((T, K), generator=g)
    return lg.to(DEV), ids.contiguous().to(DEV), gw.to(DEV)


def _formula(lg, ids, starts, scoring, renorm, f, gw, gb, gz):
    """Everything in 64 bits, the gradient written out; with the magnitudes that
    its terms have."""
    lg, ids = lg.double(), ids.long()
    T, E = lg.shape
    K = ids.shape[1]
    soft = scoring == "softmax"
    m = lg.amax(1, keepdim=True) if T else lg[:, :1]
    m = torch.where(m == -float("inf"), torch.zeros_like(m), m)
    if soft:
        s = torch.exp(lg - m)
        rest = torch.ones_like(s)
    else:
        s, rest = torch.sigmoid(lg), torch.sigmoid(-lg)
    tot = s.sum(1, keepdim=True)
    p = torch.where(tot > 0, s / tot, torch.zeros_like(s))
    lse = torch.where(tot > 0, m + torch.log(tot), torch.zeros_like(m))[:, 0]
    ok = (ids >= 0) & (ids < E)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    sel = (p if soft else s).gather(1, at) * ok
    u = sel
    if renorm:
        n = sel.sum(1, keepdim=True)
        u = torch.where(n > 0, sel / n, torch.zeros_like(sel))
    w = f * u
    S = len(starts) - 1
    counts = torch.zeros((S, E), dtype=torch.int32, device=lg.device)
    P = torch.zeros((S, E), dtype=F64, device=lg.device)
    h = torch.zeros_like(lg)
    used = torch.zeros(T, dtype=torch.bool, device=lg.device)
    losses = []
    Q = sum(b > a for a, b in zip(starts[:-1], starts[1:]))
    for q, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        if b == a:
            continue
        x = ids[a:b][ok[a:b]]
        counts[q] = torch.bincount(x, minlength=E).int()
        P[q] = p[a:b].sum(0) / (b - a)
        losses.append((counts[q].double() * P[q]).sum() * E / (K * (b - a)))
        h[a:b] = gb * E * counts[q].double() / (K * (b - a) ** 2 * Q)
        used[a:b] = True
    balance = torch.stack(losses).mean() if losses else torch.zeros((), dtype=F64, device=lg.device)
    n = max(int(used.sum()), 1)
    z = (lse[used] ** 2).sum() / n
    zt = torch.where(used, 2 * gz * lse / n, torch.zeros_like(lse))[:, None] if soft \
        else torch.zeros((T, 1), dtype=F64, device=lg.device)
    hp = (p * h).sum(1, keepdim=True)
    gw = gw.double() * ok
    wg, wga = (w * gw).sum(1, keepdim=True), (w * gw.abs()).sum(1, keepdim=True)
    c = wg if soft and not renorm else torch.zeros_like(wg)
    ca = wga if soft and not renorm else torch.zeros_like(wg)
    term = w * (gw - (wg / f if renorm else 0))
    terma = w * (gw.abs() + (wga / f if renorm else 0))
    d = p * (h - hp + zt - c)
    da = p * (h.abs() + hp.abs() + zt.abs() + ca)
    d = rest * d.scatter_add(1, at, term * ok)
    da = da.scatter_add(1, at, terma * ok)
    return dict(weights=w, balance=balance, z=z, counts=counts, probs=P, d=d, da=da, lse=lse,
                used=used)


def _check(lg, ids, gw, starts=None, scoring="softmax", renorm=True, f=1.0, gb=0.7, gz=0.3,
           what=""):
    T, E = lg.shape
    lg = lg.detach().requires_grad_(True)
    dev = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV)
    r = router_losses(lg, ids, scoring=scoring, renormalize=renorm, routed_scaling_factor=f,
                      seq_starts=dev)
    outs = [r.weights, r.balance] + ([r.z] if r.z is not None else [])
    gs = [gw, torch.full((), gb, device=DEV), torch.full((), gz, device=DEV)][:len(outs)]
    d, = torch.autograd.grad(outs, lg, gs)
    clamped = [min(max(v, 0), T) for v in (starts or [0, T])]
    e = _formula(lg.detach(), ids, clamped, scoring, renorm, f, gw, gb,
                 gz if scoring == "softmax" else 0.0)
    l64 = lg.detach().double()
    fin = torch.where(torch.isfinite(l64), l64, torch.zeros_like(l64))
    D = float((fin.amax(1) - fin.amin(1)).max()) if T else 0.0
    R = (D + 40) * U

    def near(name, got, want, tol):
        got = got.detach().double()
        assert got.shape == want.shape, name
        bad = ~((got - want).abs() <= tol)
        assert not bool(bad.any()), (what, name, int(bad.sum()),
                                     float((got - want).abs()[bad].max()))

    assert torch.equal(r.counts, e["counts"]), what
    assert r.weights.dtype == r.balance.dtype == r.probs.dtype == F32 and d.dtype == lg.dtype
    near("weights", r.weights, e["weights"], e["weights"] * (2 * R + 4 * U) + 2.0 ** -140)
    near("probs", r.probs, e["probs"], e["probs"] * (R + 2.0 ** -17) + 2.0 ** -140)
    near("balance", r.balance, e["balance"], e["balance"] * (R + 2.0 ** -17))
    if scoring == "softmax":
        dl = (fin.abs().max() if T else 0.0) + 47.0
        near("z", r.z, e["z"], 2 * e["lse"][e["used"]].abs().mean() * dl * U + e["z"] * 2.0 ** -17
             + 2.0 ** -40 if bool(e["used"].any()) else torch.zeros((), dtype=F64, device=DEV))
    else:
        assert r.z is None
    tol = e["da"] * (2 * R + 16 * U) + 2.0 ** -140
    near("gradient", d, e["d"], tol + (e["d"].abs() + tol) * (2.0 ** -8 if d.dtype == BF else U))
    return r, d


SHAPES = [   # T, E, K
    (1, 1, 1), (1, 8, 2), (2, 3, 3), (5, 8, 8), (63, 16, 4), (64, 17, 16), (65, 32, 1), (7, 33, 5),
    (130, 60, 4), (257, 64, 6), (100, 72, 3), (33, 128, 8), (511, 130, 8), (77, 160, 6),
    (129, 256, 8), (40, 257, 8), (301, 384, 16), (66, 512, 10), (35, 513, 9), (19, 1000, 7),
    (50, 1024, 16), (2049, 64, 8), (5003, 128, 8),
]


@pytest.mark.parametrize("scoring,renorm,f", [("softmax", True, 1.0), ("softmax", False, 1.0),
                                              ("sigmoid", True, 2.5), ("sigmoid", False, 0.5)])
def test_shapes(scoring, renorm, f):
    for T, E, K in SHAPES:
        for dtype in (F32, BF):
            lg, ids, gw = _inputs(T, E, K, seed=T + E, dtype=dtype, drop=0.1 if T % 2 else 0.0)
            _check(lg, ids, gw, None, scoring, renorm, f, what=(T, E, K, dtype))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sequences(scoring):
    """Empty ones, one row long, behind and before the rows that none holds."""
    for T, E, K, starts in [
        (10, 8, 2, [0, 10]), (10, 8, 2, [0, 0, 10, 10]), (10, 8, 2, [0, 0, 0]), (10, 8, 2, [3, 7]),
        (10, 8, 2, [2, 2, 5, 5, 5, 9]), (300, 64, 4, list(range(0, 301))),
        (300, 64, 4, list(range(0, 300, 7))), (777, 256, 8, [0, 1, 300, 300, 555, 700]),
        (2500, 512, 10, [0, 900, 901, 2400]), (1200, 1024, 4, [5, 600, 1100]),
        (10, 8, 2, [0, 4, 40]), (10, 8, 2, [-3, 4, 9]), (0, 8, 2, [0, 0]),
        (4096, 16, 2, [0, 1000, 1001, 4000]), (70, 20, 2, [69, 70]),
    ]:
        lg, ids, gw = _inputs(T, E, K, seed=T)
        _check(lg, ids, gw, starts, scoring, what=(T, E, starts[:8]))


def test_no_rows():
    lg, ids, gw = _inputs(0, 64, 4)
    r, d = _check(lg, ids, gw)
    assert r.balance.item() == 0.0 and r.z.item() == 0.0 and not r.counts.any() and d.shape == (0, 64)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_masked_experts_and_empty_rows(scoring, renorm):
    """-inf and the type's lowest value in places, whole rows of -inf, rows without
    an expert, the same expert twice, far logits."""
    lowest = torch.finfo(F32).min
    for E, K in ((8, 2), (60, 4), (256, 8), (700, 12)):
        lg, ids, gw = _inputs(90, E, K, seed=E)
        lg[:, E // 2] = -float("inf")
        lg[3:9] = -float("inf")
        ids[20:25] = -1
        ids[25, 0] = E
        ids[26, -1] = 2 ** 31 - 1
        ids[27, :] = ids[27, :1]
        ids[28, -1] = -2 ** 31
        _check(lg, ids, gw, [0, 40, 90], scoring, renorm, what=E)
        low = torch.where(lg == -float("inf"), torch.full_like(lg, -80.0), lg)
        low[40:45] = -80 + 0.25 * torch.arange(E, device=DEV) / E
        _check(low, ids, gw, [0, 40, 90], scoring, renorm, what=E)
        low = lg.clone()
        low[:, E // 2] = lowest
        low[3:9] = 1.0
        got = router_losses(low, ids, scoring=scoring, renormalize=renorm)
        low[low == lowest] = -float("inf")
        want = router_losses(low, ids, scoring=scoring, renormalize=renorm)
        assert all(x is None or bool((x == y).all()) for x, y in zip(got, want))


def test_nan_stays_in_its_row():
    for bad in (float("nan"), float("inf")):
        lg, ids, gw = _inputs(40, 64, 4, seed=5)
        lg[7, 30] = bad
        lg.requires_grad_(True)
        starts = torch.tensor([0, 20, 40], dtype=torch.int32, device=DEV)
        r = router_losses(lg, ids, seq_starts=starts)
        d, = torch.autograd.grad([r.weights], lg, [gw])
        rows = torch.arange(40, device=DEV) != 7
        assert r.weights[7].isnan().all() and r.weights[rows].isfinite().all()
        assert d[7].isnan().any() and d[rows].isfinite().all()
        assert r.balance.isnan() and r.z.isnan()
        assert r.probs[0].isnan().any() and r.probs[1].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides(dtype):
    """Rows at other strides and addresses, one row repeated, a slice of columns."""
    for E in (8, 64, 100, 256):
        big, ids, gw = _inputs(50, 2 * E + 3, 3, seed=E, dtype=dtype)
        ids = ids % E
        for view in (big[:, :E], big[:, 1:E + 1], big[:, E:2 * E], big[::2, 2:E + 2]):
            n = view.shape[0]
            _check(view, ids[:n].contiguous(), gw[:n].contiguous(), what=(E, view.stride()))
    one, ids, gw = _inputs(1, 64, 3, dtype=dtype)
    _check(one.expand(30, 64), ids.expand(30, 3).contiguous(), gw.expand(30, 3).contiguous())


def test_weights_are_the_routers():
    """What ``route`` gives for its own selection, up to the exponential's rounding."""
    for E, K, kw in ((64, 6, dict()), (512, 10, dict()), (8, 2, dict(renormalize=False)),
                     (256, 8, dict(scoring="sigmoid", routed_scaling_factor=2.5))):
        lg, _, _ = _inputs(333, E, K, seed=E)
        extra = dict(n_group=8, topk_group=4) if E == 256 else {}
        w, ids = route(lg, top_k=K, **kw, **extra)
        r = router_losses(lg, ids, **kw)
        assert float(((r.weights - w).abs() / w).max()) <= 2.0 ** -18
        assert int(r.counts.sum()) == 333 * K


def test_single_gradients():
    """Each output's gradient alone is its part of the whole."""
    lg, ids, gw = _inputs(70, 60, 4, seed=2)
    one = torch.ones((), device=DEV)
    lg.requires_grad_(True)
    r = router_losses(lg, ids)
    parts = [torch.autograd.grad(o, lg, g, retain_graph=True)[0]
             for o, g in ((r.weights, gw), (r.balance, one), (r.z, one))]
    whole, = torch.autograd.grad([r.weights, r.balance, r.z], lg, [gw, one, one])
    scale = sum(p.abs() for p in parts)
    assert bool(((sum(parts) - whole).abs() <= 16 * U * scale + 2.0 ** -140).all())
    assert not r.counts.requires_grad and not r.probs.requires_grad
    with torch.no_grad():
        assert not router_losses(lg, ids).balance.requires_grad


def test_once_differentiable():
    """A gradient of the gradient is refused, not wrong; leaves and their kin are
    checked for changes in place."""
    lg, ids, gw = _inputs(20, 16, 2, seed=6)
    lg.requires_grad_(True)
    d, = torch.autograd.grad(router_losses(lg, ids).weights, lg, gw, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), lg)
    plain, = torch.autograd.grad(router_losses(lg, ids).weights, lg, gw)
    assert torch.equal(d.detach(), plain)
    r = router_losses(lg, ids)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(r.weights, lg, gw)


def test_through_the_products():
    """From hidden states, as a tuning step runs it: the router product's gradient is
    the logits' times its operands."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((300, 96), generator=g)).to(DEV).requires_grad_(True)
    w = (torch.randn((40, 96), generator=g) * 0.1).to(DEV).requires_grad_(True)
    logits = x @ w.t()
    ids = route(logits.detach(), top_k=4)[1]
    r = router_losses(logits, ids)
    loss = (r.weights ** 2).sum() + 0.5 * r.balance + 0.1 * r.z
    d, dw, dx = torch.autograd.grad(loss, [logits, w, x])
    e = _formula(logits.detach(), ids, [0, 300], "softmax", True, 1.0, 2 * r.weights.detach(), 0.5,
                 0.1)
    tol = e["da"] * 2.0 ** -17
    assert bool(((d.double() - e["d"]).abs() <= tol + e["d"].abs() * U).all())
    xd, wd = x.detach().double(), w.detach().double()
    full = tol + e["d"].abs() * 300 * 2.0 ** -23
    assert bool(((dw.double() - e["d"].t() @ xd).abs() <= full.t() @ xd.abs() + 1e-12).all())
    assert bool(((dx.double() - e["d"] @ wd).abs() <= full @ wd.abs() + 1e-12).all())


@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False),
                                            ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(scoring, renorm):
    """Along random directions v of unit length: (F(l + h v) - F(l - h v)) / 2h is off
    by h^2 / 6 times a third derivative and by F's rounding over h.  F = sum of
    weights' dots (|gw| <= 1), balance and z here has |F| <= F0 and third
    derivatives along v below 30 F0 (softmax and sigmoid have them below 6 per
    factor, z's square included); F's parts are off by 2^-16 F0."""
    lg, ids, gw = _inputs(24, 16, 3, seed=9)
    gw = gw.clamp(-1, 1)
    lg.requires_grad_(True)

    def F(x):
        r = router_losses(x, ids, scoring=scoring, renormalize=renorm)
        out = (r.weights.double() * gw.double()).sum() + r.balance.double()
        return out if r.z is None else out + r.z.double()

    r = router_losses(lg, ids, scoring=scoring, renormalize=renorm)
    outs = [r.weights, r.balance] + ([] if r.z is None else [r.z])
    one = torch.ones((), device=DEV)
    d, = torch.autograd.grad(outs, lg, [gw] + [one] * (len(outs) - 1))
    F0 = float((r.weights.sum() + r.balance + (0 if r.z is None else r.z)).detach())
    h = 2.0 ** -4
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for _ in range(8):
            v = torch.randn(lg.shape, generator=g).to(DEV)
            v = v / v.norm()
            diff = float((F(lg + h * v) - F(lg - h * v)) / (2 * h))
            assert abs(diff - float((d.double() * v.double()).sum())) <= \
                F0 * (5 * h * h + 2.0 ** -16 / h)


def test_same_bits_and_other_streams():
    lg, ids, gw = _inputs(3000, 256, 8, seed=3)
    lg.requires_grad_(True)
    starts = torch.tensor([0, 700, 2900], dtype=torch.int32, device=DEV)

    def step(stream=None):
        r = router_losses(lg, ids, seq_starts=starts, stream=stream)
        d, = torch.autograd.grad([r.weights, r.balance, r.z], lg,
                                 [gw, torch.ones((), device=DEV), torch.ones((), device=DEV)])
        return (*r, d)

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        here, there = step(), step(side)
        torch.cuda.synchronize()
        for x, y, z in zip(first, here, there):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_graph():
    """Captured forward and backward, replayed between eager steps, with new inputs."""
    lg, ids, gw = _inputs(600, 128, 8, seed=4)
    one = torch.ones((), device=DEV)

    def step(x):
        x = x.detach().requires_grad_(True)
        r = router_losses(x, ids)
        d, = torch.autograd.grad([r.weights, r.balance, r.z], x, [gw, one, one])
        return r.weights, r.balance, r.z, r.counts, d

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(lg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(lg)
    for seed in range(4):
        new = _inputs(600, 128, 8, seed=10 + seed)
        lg.copy_(new[0])
        ids.copy_(new[1])
        want = [t.detach().clone() for t in step(lg)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def _definition(lg, ids, starts, scoring, renorm, f, gw, gb, gz):
    """The definition in 64 bits (what vanishes there is zero), and the gradient by
    autograd; ids are all experts.  Beside it the magnitudes of the gradient's terms."""
    l = lg.detach().double().requires_grad_(True)
    ids = ids.long()
    (T, E), K, soft = l.shape, ids.shape[1], scoring == "softmax"
    over = lambda v, n: v / torch.where(n > 0, n, torch.ones_like(n))  # noqa: E731
    s = torch.softmax(l, 1) if soft else torch.sigmoid(l)
    p, u = over(s, s.sum(1, keepdim=True)), s.gather(1, ids)
    if renorm:   # (softmax: of the selected logits, as a ratio leaves 1e-18 beside them)
        u = torch.softmax(l.gather(1, ids), 1) if soft else over(u, u.sum(1, keepdim=True))
    m = l.detach().amax(1, keepdim=True)   # (torch.logsumexp's own gradient is exp(l - lse),
    w, lse = f * u, (m + torch.log(torch.exp(l - m).sum(1, keepdim=True)))[:, 0]   # far off: 1)
    S = len(starts) - 1
    counts = torch.zeros((S, E), dtype=torch.int32, device=l.device)
    P = torch.zeros((S, E), dtype=F64, device=l.device)
    h, zt = torch.zeros((T, E), dtype=F64, device=l.device), torch.zeros((T, 1), dtype=F64,
                                                                        device=l.device)
    spans = [(q, a, b) for q, (a, b) in enumerate(zip(starts[:-1], starts[1:])) if b > a]
    n = sum(b - a for _, a, b in spans)
    losses, squares = [], []
    for q, a, b in spans:
        counts[q] = torch.bincount(ids[a:b].reshape(-1), minlength=E).int()
        mean = p[a:b].mean(0)
        P[q] = mean.detach()
        losses.append((counts[q].double() * mean).sum() * E / (K * (b - a)))
        squares.append((lse[a:b] ** 2).sum())
        h[a:b] = abs(gb) * E * counts[q].double() / (K * (b - a) ** 2 * len(spans))
        zt[a:b] = 2 * abs(gz) * lse[a:b, None].detach().abs() / n
    balance, z = torch.stack(losses).mean(), torch.stack(squares).sum() / n
    total = (w * gw.double()).sum() + gb * balance + (gz * z if soft else 0.0)
    d, = torch.autograd.grad(total, l)
    p, w = p.detach(), w.detach()
    wg = (w * gw.double().abs()).sum(1, keepdim=True)
    da = p * (h + (p * h).sum(1, keepdim=True) + (zt + (0 if renorm else wg) if soft else 0))
    da = da.scatter_add(1, ids, w * (gw.double().abs() + (wg / f if renorm else 0)))
    return dict(weights=w, balance=balance.detach(), z=z.detach(), counts=counts, probs=P, d=d,
                da=da, total=total.detach())


MODES = [("softmax", True, 1.0), ("softmax", False, 1.0), ("sigmoid", True, 2.5),
         ("sigmoid", False, 0.5)]


@pytest.mark.parametrize("scoring,renorm,f", MODES)
@pytest.mark.parametrize("dtype", [F32, BF])
def test_far_logits(scoring, renorm, f, dtype):
    """Rows wholly or in part at far finite values, the type's lowest and highest among
    them, in sequences and behind the last one.  Near a far maximum an exponential's
    argument is the exact difference times log2 e, off by 1.22 |l - m| u, where e^(l - m)
    is above 2^-126 (|l - m| < 88: R as for a spread of 88); below it vanishes.  A row
    whose sigmoids all vanish in 64 bits is one without probabilities."""
    top = torch.finfo(dtype).max
    far = [-1e9, -1e10, -1e30, -top, 1e9, 1e10, 1e30, top, -300.0, 300.0, -5000.25, 5000.25]
    R = (88 + 40) * U
    for E, K in ((8, 2), (60, 4), (256, 8), (700, 12)):
        g = torch.Generator().manual_seed(E)
        rows = []
        for v in far:
            r = torch.randn((4, E), generator=g) * 1.5
            r[0] = v                                          # all of a row
            r[1, ::2] = v                                     # half of it
            r[2] = (r[2].double() + v).clamp(-top, top)       # beside v, as far as the type goes
            r[3, E // 2] = v                                  # one
            rows.append(r)
        rows = torch.cat(rows).to(dtype)
        lg = torch.cat([rows, torch.randn((12, E), generator=g).to(dtype), rows]).to(DEV)
        T, used = lg.shape[0], rows.shape[0] + 12
        ids = torch.sort(lg.float(), dim=1, descending=True, stable=True).indices[:, :K]
        ids = ids.to(torch.int32).contiguous()
        gw = torch.randn((T, K), generator=g).to(DEV)
        starts, gb, gz = [0, 0, 23, used], 0.7, 0.3
        lg.requires_grad_(True)
        r = router_losses(lg, ids, scoring=scoring, renormalize=renorm, routed_scaling_factor=f,
                          seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
        outs = [r.weights, r.balance] + ([r.z] if r.z is not None else [])
        d, = torch.autograd.grad(outs, lg, [gw] + [torch.full((), v, device=DEV) for v in (gb, gz)]
                                 [:len(outs) - 1])
        e = _definition(lg, ids, starts, scoring, renorm, f, gw, gb, gz)

        def near(name, got, want, tol):
            bad = ~((got.detach().double() - want).abs() <= tol)
            assert not bool(bad.any()), (E, name, bad.nonzero()[:4].tolist(),
                                         got[bad][:4].tolist(), want[bad][:4].tolist())

        assert torch.equal(r.counts, e["counts"])
        near("weights", r.weights, e["weights"], e["weights"] * (2 * R + 4 * U) + f * 2.0 ** -120)
        near("probs", r.probs, e["probs"], e["probs"] * (R + 2.0 ** -17) + 2.0 ** -120)
        near("balance", r.balance, e["balance"], e["balance"] * (R + 2.0 ** -17))
        if r.z is not None:   # 1e30 squared and more leaves fp32
            assert float(e["z"]) > 1e60 and bool(r.z == float("inf"))
        tol = e["da"] * (2 * R + 16 * U) + 2.0 ** -110
        near("gradient", d, e["d"], tol + (e["d"].abs() + tol) * (2.0 ** -8 if dtype == BF else U))
        # rows behind the last sequence: the weights' gradient alone, whatever the rows are
        alone, = torch.autograd.grad(router_losses(
            lg, ids, scoring=scoring, renormalize=renorm, routed_scaling_factor=f).weights, lg, gw)
        assert torch.equal(d[used:], alone[used:])
        if scoring == "softmax":   # as the router that serves has them, up to E u of its sum
            w, at = route(lg.detach().float(), top_k=K, renormalize=renorm)
            assert torch.equal(at.sort(1).values, ids.sort(1).values)
            have, want = r.weights.sort(1).values, w.sort(1).values
            assert bool(((have - want).abs() <= want * 2.0 ** -14 + 2.0 ** -120).all())


@pytest.mark.parametrize("v", [-1e10, 1e10, 1e18])
def test_far_logits_z(v):
    """z and its gradient where the squares stay in range."""
    lg = torch.full((70, 24), v, device=DEV).requires_grad_(True)
    ids = torch.arange(140, device=DEV, dtype=torch.int32).view(70, 2) % 24
    r = router_losses(lg, ids)
    d, = torch.autograd.grad([r.z], lg, [torch.ones((), device=DEV)])
    want = lg.detach().double().logsumexp(1)[0]
    # lse is off by (|m| + 47) u, its square by twice that; 70 terms are added
    assert abs(float(r.z.detach()) - float(want) ** 2) <= float(want) ** 2 * 80 * U * 4
    assert bool(((d.double() - 2 * want / 70 / 24).abs() <= abs(float(want)) / 840 * 64 * U).all())


def test_weights_into_the_expert_layer():
    """A selection's weights into the framework's experts: refused while they require a
    gradient, taken detached or under no_grad."""
    from xtu_moe_amd import formats as F
    from xtu_moe_amd.layer import ExpertWeights, moe_forward
    g = torch.Generator().manual_seed(8)
    E, K, H, I = 8, 2, 256, 128
    w13, w2 = torch.randn((E, 2 * I, H), generator=g) * 0.05, torch.randn((E, H, I), generator=g) * 0.05
    W = ExpertWeights.from_dense(F.FMT_MXFP4, *F.quantize_mxfp4(w13), *F.quantize_mxfp4(w2),
                                 device=torch.device(DEV))
    for T in (3, 40):
        x = torch.randn((T, H), generator=g).to(BF).to(DEV)
        lg = torch.randn((T, E), generator=g).to(DEV).requires_grad_(True)
        w, ids = route(lg.detach(), top_k=K)
        r = router_losses(lg, ids)
        with pytest.raises(ValueError, match="no backward"):
            moe_forward(x, ids, r.weights, W)
        with torch.no_grad():
            out = moe_forward(x, ids, r.weights, W, out_dtype=F32)
        assert torch.equal(out, moe_forward(x, ids, r.weights.detach(), W, out_dtype=F32))
        (0.01 * r.balance + 0.001 * r.z).backward()
        assert lg.grad.isfinite().all() and bool(lg.grad.any())


def test_gradients_tangents_refused():
    """A tangent that comes in with an output's gradient would be lost as well."""
    from torch.autograd import forward_ad
    lg, ids, gw = _inputs(20, 16, 2, seed=6)
    lg.requires_grad_(True)
    r = router_losses(lg, ids)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(gw, torch.ones_like(gw))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(r.weights, lg, dual, retain_graph=True)
    d, = torch.autograd.grad(r.weights, lg, gw)
    assert d.isfinite().all()


@pytest.mark.parametrize("scoring,renorm,f,term", [
    m + (t,) for m in MODES for t in ("weights", "balance", "z", "all")
    if t != "z" or m[0] == "softmax"])
def test_gradient_against_autograd(scoring, renorm, f, term):
    """Element by element against autograd of the definition in 64 bits, each loss alone
    too: within R's bounds of that loss's own terms, a thousandth of the gradient at most,
    so that a missing term or a wrong sign or factor shows."""
    pick = lambda name, v: v if term in (name, "all") else 0.0  # noqa: E731
    for T, E, K in ((9, 8, 3), (130, 60, 4), (257, 64, 6), (33, 128, 8), (700, 256, 8), (50, 1024, 16)):
        for dtype in (F32, BF):
            lg, ids, gw = _inputs(T, E, K, seed=T + E, dtype=dtype)
            gw = gw if term in ("weights", "all") else gw * 0
            gb, gz = pick("balance", 0.7), pick("z", 0.3)
            starts = [0, T // 3, T // 3, T - T // 5]
            lg.requires_grad_(True)
            r = router_losses(lg, ids, scoring=scoring, renormalize=renorm, routed_scaling_factor=f,
                              seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
            outs = [r.weights, r.balance] + ([r.z] if r.z is not None else [])
            d, = torch.autograd.grad(outs, lg, [gw] + [torch.full((), v, device=DEV)
                                                       for v in (gb, gz)][:len(outs) - 1])
            e = _definition(lg, ids, starts, scoring, renorm, f, gw, gb, gz)
            l64 = lg.detach().double()
            R = (float((l64.amax(1) - l64.amin(1)).max()) + 40) * U
            tol = e["da"] * (2 * R + 16 * U) + 2.0 ** -140
            assert float(tol.norm()) <= float(e["d"].norm()) / 1000, (T, E)
            tol = tol + (e["d"].abs() + tol) * (2.0 ** -8 if dtype == BF else U)
            bad = ~((d.double() - e["d"]).abs() <= tol)
            assert not bool(bad.any()), (T, E, dtype, int(bad.sum()))


@pytest.mark.parametrize("scoring,renorm,f", MODES)
def test_gradient_against_differences_of_the_definition(scoring, renorm, f):
    """Along directions v of unit length against (F(l + h v) - F(l - h v)) / 2h of the
    definition's F in 64 bits: off by h^2 / 6 times a third derivative (at most 30 F0, as
    above) and by 2^-50 F0 / h, beside the kernel's own error; all of that a hundredth of
    what is compared."""
    lg, ids, gw = _inputs(24, 16, 3, seed=9)
    starts, gb, gz, h = [0, 10, 24], 0.7, 0.3, 2.0 ** -13
    lg.requires_grad_(True)
    r = router_losses(lg, ids, scoring=scoring, renormalize=renorm, routed_scaling_factor=f,
                      seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    outs = [r.weights, r.balance] + ([r.z] if r.z is not None else [])
    d, = torch.autograd.grad(outs, lg, [gw] + [torch.full((), v, device=DEV) for v in (gb, gz)]
                             [:len(outs) - 1])
    F = lambda l: _definition(l, ids, starts, scoring, renorm, f, gw, gb, gz)  # noqa: E731
    e, l64 = F(lg), lg.detach().double()
    F0 = float((e["weights"] * gw.double().abs()).sum() + gb * e["balance"] + gz * e["z"])
    own = e["da"] * (2 * (float((l64.amax(1) - l64.amin(1)).max()) + 40) + 16) * U + e["d"].abs() * U
    g = torch.Generator().manual_seed(1)
    largest = 0.0
    for _ in range(8):
        v = torch.randn(lg.shape, generator=g).double().to(DEV)
        v = v / v.norm()
        diff = float((F(l64 + h * v)["total"] - F(l64 - h * v)["total"]) / (2 * h))
        tol = F0 * (5 * h * h + 2.0 ** -50 / h) + float((own * v.abs()).sum())
        assert abs(diff - float((d.double() * v).sum())) <= tol
        largest = max(largest, abs(diff) / tol)
    assert largest > 100   # (no gradient, or one of the other sign, would show)


def test_gradient_penalty_refused():
    """A loss on the gradient, through outputs whose own gradients are constants: refused,
    where a constant in its place would leave that loss out."""
    lg, ids, gw = _inputs(20, 16, 2, seed=6)
    lg.requires_grad_(True)
    one = torch.ones((), device=DEV)
    for pick, g in (("weights", gw), ("balance", one), ("z", one)):
        out = getattr(router_losses(lg, ids), pick)
        d, = torch.autograd.grad(out, lg, g, create_graph=True)
        assert d.requires_grad
        plain, = torch.autograd.grad(getattr(router_losses(lg, ids), pick), lg, g)
        assert torch.equal(d.detach(), plain)
        with pytest.raises(RuntimeError, match="once differentiable"):
            (out.sum() + d.square().sum()).backward()
        assert lg.grad is None


@pytest.mark.parametrize("renorm", [True, False])
def test_infinity_with_sigmoid(renorm):
    """sigmoid(inf) is 1: the row stays finite, and has no slope there."""
    lg, ids, gw = _inputs(40, 64, 4, seed=5)
    lg[7, 30], ids[7, 0] = float("inf"), 30
    ids[7, 1:] = torch.tensor([1, 2, 3], device=DEV)
    lg[8], lg[9, ::2] = float("inf"), float("inf")
    starts = [0, 20, 40]
    lg.requires_grad_(True)
    r = router_losses(lg, ids, scoring="sigmoid", renormalize=renorm,
                      seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    d, = torch.autograd.grad([r.weights, r.balance], lg, [gw, torch.full((), 0.7, device=DEV)])
    # (100 stands for inf: sigmoid(100) is 1 and its slope 0 within 2^-140)
    near = lg.detach().clone()
    near[near == float("inf")] = 100.0
    e = _formula(near, ids, starts, "sigmoid", renorm, 1.0, gw, 0.7, 0.0)
    R = (12 + 40) * U
    assert bool(((r.weights.detach().double() - e["weights"]).abs() <= e["weights"] * (2 * R + 4 * U)).all())
    assert bool(((r.probs.double() - e["probs"]).abs() <= e["probs"] * (R + 2.0 ** -17)).all())
    assert bool(((d.double() - e["d"]).abs() <= e["da"] * (2 * R + 17 * U) + 2.0 ** -120).all())
    assert bool((d[8] == 0).all()) and d[7, 30] == 0


@pytest.mark.parametrize("E", [8, 300])
def test_long_sums(E):
    """Millions of equal rows (one, repeated), whose rounding errors all have one sign: a
    lane adds at most 256 of them in fp32, 64 more joins behind that, the rest is in fp64.
    So P, balance and z are off by R + 320 u (z: twice lse's error more)."""
    T = 1 << 27 if E == 8 else 1 << 24
    g = torch.Generator().manual_seed(E)
    row = torch.randn((1, E), generator=g).to(DEV)
    ids = torch.zeros((T, 1), dtype=torch.int32, device=DEV)
    r = router_losses(row.expand(T, E), ids)
    p = torch.softmax(row.double(), 1)
    tol = (8 + 40 + 320) * U
    assert float(((r.probs.double() - p).abs() / p).max()) <= tol
    assert r.counts[0].tolist() == [T] + [0] * (E - 1)
    assert abs(float(r.balance) / float(p[0, 0] * E) - 1) <= tol
    lse = torch.logsumexp(row.double(), 1)
    assert abs(float(r.z) / float(lse ** 2) - 1) <= 2 * (8 + 6 + 40) * U / float(lse) + 320 * U


@pytest.mark.parametrize("scoring,f", [("softmax", 1.0), ("sigmoid", 2.5)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_selection_far_below_the_maximum(scoring, f, dtype):
    """The best experts dropped, or never selected: renormalised weights keep the ratios of
    those that are, up to where their scores leave fp32 beside the row's largest: off by
    2^-126 over their sum, zero when all of them vanish."""
    for E, K in ((8, 3), (60, 4), (256, 8), (700, 12)):
        g = torch.Generator().manual_seed(E)
        T = 150
        lg = torch.randn((T, E), generator=g).clamp(-4, 4)
        ids = torch.stack([torch.randperm(E // 2, generator=g)[:K] for _ in range(T)]).int().to(DEV)
        down = torch.tensor([30.0, 60.0, 150.0, 600.0, 1e30])[torch.arange(T) % 5, None]
        lg[:, :E // 2] -= down
        lg = lg.to(dtype).to(DEV)
        gw = torch.randn((T, K), generator=g).to(DEV)
        lg.requires_grad_(True)
        r = router_losses(lg, ids, scoring=scoring, routed_scaling_factor=f)
        d, = torch.autograd.grad(r.weights, lg, gw)
        e = _definition(lg, ids, [0, T], scoring, True, f, gw, 0.0, 0.0)
        kept = (down < 100)[:, 0].to(DEV)
        R = (72 + 40) * U   # (4 + 60 + 4 and the type's rounding apart at most)
        beside = 2.0 ** -126 / math.exp(-72)
        tol = e["weights"] * (2 * R + 4 * U + beside) + f * beside
        assert bool(((r.weights.detach().double() - e["weights"]).abs() <= tol)[kept].all()), E
        assert not bool(r.weights[~kept].any()) and not bool(d[~kept].any())
        tol = e["da"] * (2 * R + 16 * U + 2 * beside) + f * 4 * beside * gw.abs().max()
        tol = tol + (e["d"].abs() + tol) * (2.0 ** -8 if dtype == BF else U)
        assert bool(((d.double() - e["d"]).abs() <= tol)[kept].all()), E
