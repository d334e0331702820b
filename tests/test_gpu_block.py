"""The MoE block from hidden states against float64.

Tolerances, derived before the first run.  Selected ids are those of the
float64 scores, in order, but that scores within the error of the fp32 logits
of each other may swap.  Logits: |l^ - l| <= (H + 2) 2^-23
sum |x w|, called dl; a softmax or sigmoid weight is then off by at most a
factor exp(2 dl) (1 + 2^-18).  An expert: gate and up sums as the logits; the
SwiGLU's slope is at most 1.2; its row is rounded to bf16 (2^-8 of the value);
the down sums add (I + 2) 2^-23 sum |a w2|, the weighted sum 2^-20 of its terms,
the output's own rounding 2^-8 (bf16) or 2^-24.
"""
import functools

import pytest
import torch

from xtu_moe_amd import formats as F
from xtu_moe_amd.block import MoeBlock
from xtu_moe_amd.layer import ExpertWeights

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
FMTS = {"bf16": F.FMT_BF16, "fp8": F.FMT_FP8, "mxfp4": F.FMT_MXFP4, "nvfp4": F.FMT_NVFP4}


@functools.lru_cache(maxsize=4)
def _layer(fmt, E, NS, H, I):
    """(ExpertWeights, [(w13, w2) float64 of every expert as a function])."""
    g = torch.Generator(device=DEV).manual_seed(E + H + I)
    n, f = E + NS, FMTS[fmt]
    w13 = torch.empty((n, 2 * I, H), device=DEV).normal_(0, 0.05, generator=g)
    w2 = torch.empty((n, H, I), device=DEV).normal_(0, 0.05, generator=g)
    w13[:, I:] *= 2.0
    q13, s13, g13 = F.quantize_w13(f, w13)
    q2, s2, g2 = F.quantize(f, w2)
    W = ExpertWeights.from_dense(f, q13, s13, q2, s2, g13, g2, n_shared=NS)
    at = lambda t, e: None if t is None else t[e:e + 1]  # noqa: E731

    def dense(e):
        g13e = at(g13, e)
        if f == F.FMT_NVFP4 and g13e is not None and g13e.dim() == 2:
            one = torch.ones(1, device=DEV)
            d13 = F.dequantize(f, at(q13, e), at(s13, e), one).double()[0]
            d13[:I] *= g13e[0, 0].double()
            d13[I:] *= g13e[0, 1].double()
        else:
            d13 = F.dequantize(f, at(q13, e), at(s13, e), g13e).double()[0]
        return d13, F.dequantize(f, at(q2, e), at(s2, e), at(g2, e)).double()[0]

    return W, dense


def _router(E, H, sigmoid, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    gate = torch.empty((E, H), device=DEV).normal_(0, 1.5 / H ** 0.5, generator=g).to(BF)
    kw = dict(scoring="softmax")
    if sigmoid:
        kw = dict(scoring="sigmoid", routed_scaling_factor=2.5,
                  bias=torch.empty(E, device=DEV).normal_(0, 0.1, generator=g))
    return gate, kw


def _select64(x, gate, K, kw, ids):
    """Weights of the chosen ids in float64, after a check that they are the
    choice; and the relative error allowed to them."""
    lg = x.double() @ gate.double().t()
    dl = (x.shape[1] + 2) * 2.0 ** -23 * (x.double().abs() @ gate.double().abs().t()).amax()
    slack = 2.0 ** -20 * (1 + lg.abs().amax())   # what fp32 logits are off in practice, at most
    ids, scoring_groups = ids.long(), kw.get("n_group", 1)
    if kw["scoring"] == "softmax":
        want = lg.sort(dim=1, descending=True, stable=True)
        scores, p = lg, torch.softmax(lg, 1)
    else:
        p = torch.sigmoid(lg)
        scores = p + kw["bias"].double() if kw.get("bias") is not None else p
        G = kw.get("n_group", 1)
        by = scores.view(len(x), G, -1)
        top2 = by.sort(dim=2, descending=True).values[..., :2].sum(2)
        order = top2.sort(dim=1, descending=True)
        keep = kw.get("topk_group", 1)
        # groups within the error of the last one kept may stand in for it
        ok = top2 >= order.values[:, keep - 1:keep] - slack
        scores = scores.masked_fill(~ok.repeat_interleave(by.shape[2], 1), -1e30)
        want = scores.sort(dim=1, descending=True, stable=True)
    # in order, each once; only scores within the error of each other may swap
    assert all(len(set(r)) == K for r in ids.tolist())
    got = scores.gather(1, ids)
    same = torch.equal(ids, want.indices[:, :K])
    near = (got - want.values[:, :K]).abs() <= slack
    if not same and scoring_groups > 1:   # a stand-in group's scores may come in between
        near |= got >= want.values[:, K - 1:K] - slack
    assert same or bool(near.all())
    w = p.gather(1, ids)
    if kw.get("renormalize", True):
        w = w / w.sum(1, keepdim=True)
    if kw["scoring"] == "sigmoid":
        w = w * kw.get("routed_scaling_factor", 1.0)
    return w, float(torch.expm1(2 * dl)) + 2.0 ** -18


def _check(blk, dense, x, res, shared_gate=None, kw=None):
    out, wts, ids = res
    W, H, I, K = blk.W, blk.W.H, blk.W.I, blk.top_k
    lim, al, be = blk.limit, blk.alpha, blk.beta
    xd = x.double()
    w, rw = _select64(x, blk.gate_weight, K, kw, ids)
    assert wts.dtype == F32 and ids.dtype == torch.int32
    assert bool(((wts.double() - w).abs() <= rw * w + 2.0 ** -30).all())
    y, e = torch.zeros_like(xd), torch.zeros_like(xd)
    for ex in sorted(set(ids.reshape(-1).tolist())) + list(range(W.E, W.n_experts)):
        d13, d2 = dense(ex)
        if ex < W.E:
            tok, k = (ids == ex).nonzero(as_tuple=True)
            we, ew = w[tok, k][:, None], rw
        else:
            tok = torch.arange(len(x), device=DEV)
            we, ew = torch.ones((len(x), 1), dtype=torch.float64, device=DEV), 0.0
            if shared_gate is not None:
                v = shared_gate[ex - W.E].double()
                we = torch.sigmoid(xd @ v)[:, None]
                ew = float((H + 2) * 2.0 ** -23 * (xd.abs() @ v.abs()).amax()) + 2.0 ** -18
        r = xd[tok]
        z, ez = r @ d13.t(), (H + 3) * 2.0 ** -23 * (r.abs() @ d13.abs().t())
        gt, u, eg, eu = z[:, :I], z[:, I:], ez[:, :I], ez[:, I:]
        if lim > 0:
            gt, u = gt.clamp(max=lim), u.clamp(-lim, lim)
        gate = gt * torch.sigmoid(al * gt)
        a = gate * (u + be)
        ea = (u.abs() + abs(be) + eu) * 1.2 * max(1.0, abs(al)) * eg + gate.abs() * eu
        ea = ea + (a.abs() + ea) * (2.0 ** -8 + 2.0 ** -18)
        yy = a @ d2.t()
        ey = ea @ d2.abs().t() + (I + 3) * 2.0 ** -23 * (a.abs() @ d2.abs().t())
        y.index_add_(0, tok, yy * we)
        e.index_add_(0, tok, we.abs() * (ey + (yy.abs() + ey) * (ew + 2.0 ** -20)))
    e = e + (y.abs() + e) * (2.0 ** -8 if out.dtype == BF else 2.0 ** -23) + 2.0 ** -40
    bad = (out.double() - y).abs() > e
    assert not bool(bad.any()), \
        f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"
    # the bounds are sums of worst cases; what random signs leave is far less
    assert float((out.double() - y).norm() / y.norm()) < 2.0 ** -7


def _x(T, H, seed):
    g = torch.Generator(device=DEV).manual_seed(1000 + seed)
    return torch.empty((T, H), device=DEV).normal_(0, 1, generator=g).to(BF)


LAYERS = [   # E, NS, K, H, I, sigmoid groups (0: softmax), shared gate
    (8, 0, 2, 256, 128, 0, False), (5, 1, 5, 256, 128, 0, True), (64, 2, 6, 512, 256, 1, True),
    (128, 0, 8, 1024, 384, 0, False), (60, 4, 4, 768, 640, 0, True), (160, 1, 6, 512, 128, 8, False),
    (256, 1, 8, 2560, 512, 8, False), (512, 1, 10, 2048, 512, 0, True), (16, 1, 16, 256, 1792, 4, True),
    (1, 1, 1, 256, 128, 0, False), (32, 0, 3, 7168, 256, 4, False), (8, 1, 2, 512, 2048, 0, False),
]


def _block(fmt, layer, **more):
    E, NS, K, H, I, groups, gated = layer
    W, dense = _layer(fmt, E, NS, H, I)
    gate, kw = _router(E, H, groups > 0, 7)
    if groups > 1:
        kw.update(n_group=groups, topk_group=max(1, groups // 2))
        while K > kw["topk_group"] * (E // groups):
            kw["topk_group"] += 1
    sg = _x(NS, H, 77) * 0.05 if gated and NS else None
    blk = MoeBlock(gate, W, top_k=K, shared_gate=sg, **kw, **more)
    return blk, dense, sg, dict(kw, **{k: v for k, v in more.items() if k == "renormalize"})


@pytest.mark.parametrize("layer", LAYERS)
@pytest.mark.parametrize("fmt", sorted(FMTS))
def test_layers(fmt, layer):
    blk, dense, sg, kw = _block(fmt, layer)
    for T in (1, 2, 3, 5, 8, 11, 16, 17, 40):
        x = _x(T, layer[3], T)
        _check(blk, dense, x, blk(x, return_routing=True, out_dtype=F32 if T % 2 else BF), sg, kw)


@pytest.mark.parametrize("fmt", sorted(FMTS))
def test_swiglu_parameters(fmt):
    blk, dense, sg, kw = _block(fmt, LAYERS[2], swiglu_limit=0.5, swiglu_alpha=1.7, swiglu_beta=1.0)
    for T in (2, 9, 33):
        x = _x(T, 512, T)
        _check(blk, dense, x, blk(x, return_routing=True), sg, kw)


@pytest.mark.parametrize("layer", [LAYERS[3], LAYERS[6], LAYERS[8]])
def test_weights_not_renormalised(layer):
    blk, dense, sg, kw = _block("mxfp4", layer, renormalize=False)
    for T in (1, 7, 20):
        x = _x(T, layer[3], T)
        _check(blk, dense, x, blk(x, return_routing=True), sg, kw)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_equal_scores_go_to_the_lowest_index(sigmoid):
    """Router rows that repeat give equal logits; the lowest indices win, in
    order."""
    W, dense = _layer("bf16", 64, 2, 512, 256)
    gate = _x(4, 512, 5).repeat(16, 1) * 0.05
    kw = dict(scoring="sigmoid" if sigmoid else "softmax")
    blk = MoeBlock(gate, W, top_k=6, **kw)
    for T in (1, 4, 16, 30):
        x = _x(T, 512, T)
        lg = x.double() @ gate[:4].double().t()
        best = lg.argmax(1)
        want = best[:, None] + 4 * torch.arange(6, device=DEV)
        out, wts, ids = blk(x, return_routing=True)
        assert torch.equal(ids.long(), want)
        assert bool((wts - 1 / 6).abs().max() < 1e-6)


@pytest.mark.parametrize("fmt", sorted(FMTS))
@pytest.mark.parametrize("layer", [LAYERS[0], LAYERS[2], LAYERS[7]])
def test_few_tokens_keep_unrounded_rows(fmt, layer):
    """Up to eight tokens of these layers keep activation rows in two bf16
    parts (2^-18 of a value): with fp32 output nothing of 2^-9 is left.  The
    fp32 sums of at most 4096 terms leave some 2^-23 sqrt(4096) = 2^-17 of
    them; rows rounded to bf16 alone leave 2^-9.2 of the norm, at most 2^-8.8
    (2^-8 / sqrt(3) where every mantissa is 1), and that is the bound where two
    parts do not fit: both parts of T (K + NS) rows of I + 8 values in a
    compute unit's 160 KB of LDS (LAYERS[7] with T = 8: 2 * 88 * 520 * 2 =
    183 040 bytes)."""
    blk, dense, sg, kw = _block(fmt, layer)
    W, K = blk.W, blk.top_k
    for T in (1, 3, 8):
        x = _x(T, layer[3], 40 + T)
        out, wts, ids = blk(x, return_routing=True, out_dtype=F32)
        xd, y = x.double(), torch.zeros((T, W.H), dtype=torch.float64, device=DEV)
        for t in range(T):
            pairs = [(int(ids[t, k]), wts[t, k].double()) for k in range(K)]
            pairs += [(W.E + s, 1.0 if sg is None else torch.sigmoid(xd[t] @ sg[s].double()))
                      for s in range(W.n_shared)]
            for e, w in pairs:
                d13, d2 = dense(e)
                z = d13 @ xd[t]
                y[t] += w * (d2 @ (torch.nn.functional.silu(z[:W.I]) * z[W.I:]))
        fits = 2 * T * (K + W.n_shared) * (W.I + 8) * 2 < 160 * 1024
        assert float((out.double() - y).norm() / y.norm()) < 2.0 ** (-13 if fits else -8.8)


def test_no_tokens_and_given_output():
    blk, dense, sg, kw = _block("fp8", LAYERS[5])
    out, wts, ids = blk(_x(0, 512, 0), return_routing=True)
    assert out.shape == (0, 512) and wts.shape == (0, 6) and ids.shape == (0, 6)
    for T in (3, 24):
        x = _x(T, 512, T)
        o = torch.full((T, 512), 9.0, device=DEV)
        got = blk(x, out=o)
        assert got.data_ptr() == o.data_ptr()
        assert torch.equal(o, blk(x, out_dtype=F32))


def test_calls_refused():
    blk, dense, sg, kw = _block("bf16", LAYERS[0])
    x = _x(4, 256, 0)
    for bad in (x.float(), x[:, :128], x.t().contiguous().t(), x[0], x.cpu()):
        with pytest.raises(ValueError):
            blk(bad)
    with pytest.raises(ValueError, match="output type"):
        blk(x, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="out must be"):
        blk(x, out=torch.empty((4, 512), dtype=BF, device=DEV)[:, ::2])
    with pytest.raises(ValueError, match="overlaps"):
        blk(x, out=x)


@pytest.mark.parametrize("layer", [LAYERS[2], LAYERS[7]])
def test_nan_stays_in_its_token(layer):
    blk, dense, sg, kw = _block("mxfp4", layer)
    H = layer[3]
    for T in (2, 8, 20):
        x = _x(T, H, T)
        ref = blk(x, return_routing=True)
        x2 = x.clone()
        x2[0, 3] = float("nan")
        out, wts, ids = blk(x2, return_routing=True)
        assert torch.equal(ids[1:], ref[2][1:]) and torch.equal(wts[1:], ref[1][1:])
        # (the order of a token's fp32 sums goes by the batch's active experts,
        # so its outputs are held to their bounds, not to the other batch's bits)
        _check(blk, dense, x[1:], (out[1:], wts[1:], ids[1:]), sg, kw)
        assert bool(((ids >= 0) & (ids < layer[0])).all())


@pytest.mark.parametrize("fmt", sorted(FMTS))
def test_same_call_same_bits(fmt):
    for layer, T in ((LAYERS[6], 1), (LAYERS[7], 6), (LAYERS[2], 16), (LAYERS[11], 4)):
        blk, *_ = _block(fmt, layer)
        x = _x(T, layer[3], T)
        first = blk(x, return_routing=True)
        for _ in range(10):
            for a, b in zip(first, blk(x, return_routing=True)):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Blocks on two streams whose launches overlap on the device."""
    blks = [_block(f, l)[0] for f, l in (("mxfp4", LAYERS[6]), ("fp8", LAYERS[7]))]
    xs = [_x(4, b.W.H, 4) for b in blks]
    refs = [b(x) for b, x in zip(blks, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for k in range(20):
        for i in (0, 1):
            outs.append((i, blks[i](xs[i], stream=streams[(i + k) % 2])))
    torch.cuda.synchronize()
    for i, o in outs:
        assert torch.equal(o, refs[i])


@pytest.mark.parametrize("T", [3, 40])
def test_graphs_captured_from_one_stream_replayed_at_once(T):
    blks = [_block(f, l)[0] for f, l in (("mxfp4", LAYERS[6]), ("nvfp4", LAYERS[7]))]
    xs = [_x(T, b.W.H, 4) for b in blks]
    outs, graphs = [], []
    for b, x in zip(blks, xs):
        b(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b(x, return_routing=True))
        graphs.append(g)
    side = torch.cuda.Stream()
    for k in range(8):
        for x in xs:
            x.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for b, x, o in zip(blks, xs, outs):
            for a, r in zip(o, b(x, return_routing=True)):
                assert torch.equal(a, r)


@pytest.mark.parametrize("bias_dtype", [F32, BF])
def test_storage_replaced_between_calls(bias_dtype):
    """The router, the shared gates and the bias are read where they lie at the
    call: other storage under them, or other values in place, and every batch
    size answers with those."""
    E, NS, K, H, I = 64, 2, 6, 512, 256
    W, dense = _layer("mxfp4", E, NS, H, I)

    def fresh(seed):
        gate, kw = _router(E, H, True, seed)
        return gate, _x(NS, H, seed) * 0.05, kw["bias"].to(bias_dtype)

    def block(gate, shared, bias):
        return MoeBlock(gate, W, top_k=K, shared_gate=shared, scoring="sigmoid", bias=bias)

    params = [torch.nn.Parameter(t, requires_grad=False) for t in fresh(30)]
    blk = block(*params)
    xs = [_x(T, H, T) for T in (1, 5, 16, 17, 40)]
    before = [blk(x, return_routing=True) for x in xs]
    for k in range(3):
        new = fresh(31 + k)
        if k < 2:
            for p, t in zip(params, new):
                p.data = t.clone()
        else:
            for p, t in zip(params, new):
                p.copy_(t)
        want = block(*new)
        for x, old in zip(xs, before):
            got, ref = blk(x, return_routing=True), want(x, return_routing=True)
            for a, b in zip(got, ref):
                assert torch.equal(a, b)
            assert not torch.equal(got[0], old[0])


def test_storage_that_does_not_fit_refused():
    E, NS, K, H, I = 64, 2, 6, 512, 256
    W, dense = _layer("mxfp4", E, NS, H, I)
    gate, kw = _router(E, H, True, 30)
    shared = _x(NS, H, 30) * 0.05
    params = [torch.nn.Parameter(t, requires_grad=False) for t in (gate, shared, kw["bias"])]
    blk = MoeBlock(params[0], W, top_k=K, shared_gate=params[1], scoring="sigmoid", bias=params[2])
    x = _x(3, H, 3)
    want = blk(x)
    off = torch.empty(E * H + 1, dtype=BF, device=DEV)[1:].view(E, H)
    for p, bad, match in (
            (params[0], gate[:32].clone(), "gate_weight"), (params[0], gate.float(), "gate_weight"),
            (params[0], gate.t().contiguous().t(), "gate_weight"), (params[0], gate.cpu(), "is on"),
            (params[0], off, "16 bytes"), (params[1], shared[:1].clone(), "shared_gate"),
            (params[1], shared.cpu(), "is on"), (params[2], kw["bias"][:60].clone(), "bias"),
            (params[2], kw["bias"].cpu(), "is on")):
        good, p.data = p.data, bad
        for xx in (x, _x(40, H, 4)):
            with pytest.raises(ValueError, match=match):
                blk(xx)
        p.data = good
    assert torch.equal(blk(x), want)
