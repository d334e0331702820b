"""The dense product with 4-bit weights against float64.

Tolerances, derived before the first run, are the dense product's: with
z = g sum_k x_k w_k + b from fp32 sums of exact products, |z^ - z| <= (K + 4) 2^-23 S,
S = sum |x_k w_k| + |b| (each addition rounds or truncates by at most one unit of
2^-23 relative to a partial sum of at most S; the second-level or group scale's
multiplication is one more).  The activations have slope at most 1.2 and are
evaluated to 2^-19 relative plus 2^-20 absolute; swiglu's two factors bound each
other's error by their own sizes.  row_scale and residual add one rounding each
(2^-24), and the output one more: 2^-24 (fp32) or 2^-8 (bf16) of the value.
"""
import pytest
import torch

from test_gpu_linear import _act64
from test_linear4 import GROUPS, forms
from xtu_moe_amd import _lib, formats as F
from xtu_moe_amd.linear import ACTIVATIONS
from xtu_moe_amd.linear4 import ARGS, Weight4, linear4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _rand(shape, seed, std=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def _weight(fmt, group, N, K, gated=False, seed=0):
    """(Weight4, the matrix in 64 bits); every code occurs, scales near 0.02."""
    g = torch.Generator().manual_seed(1000 + seed)
    rows = N * (2 if gated else 1)
    codes = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8)
    nib = torch.stack([codes & 15, codes >> 4], -1).view(rows, K).long()
    gs = None
    if fmt == F.FMT_INT4:
        s = torch.rand((rows, K // group), generator=g) * 0.02 + 0.002
        w = (nib - 8).double() * s.double().repeat_interleave(group, 1)
    else:
        w = torch.tensor(F.E2M1_VALUES, dtype=torch.float64)[nib]
        if fmt == F.FMT_MXFP4:
            s = torch.randint(116, 123, (rows, K // 32), generator=g, dtype=torch.uint8)
            sv = torch.exp2(s.double() - 127)
        else:   # subnormal, zero and negative scales too
            s = torch.randint(0, 0x7f, (rows, K // 16), generator=g, dtype=torch.uint8)
            s |= (torch.rand(s.shape, generator=g) < 0.1).to(torch.uint8) << 7
            sv = s.view(torch.float8_e4m3fn).double()
            gs = torch.tensor([3e-4, 5e-4][:2 if gated else 1])
            sv = sv * gs.double().repeat_interleave(N)[:, None]
        w = w * sv.repeat_interleave(group, 1)
    W = Weight4.from_dense(fmt, codes.to(DEV), s.to(DEV), gs, gated=gated)
    return W, w.to(DEV)


def _check(out, x, w, act="none", bias=None, row_scale=None, residual=None, limit=0.0, alpha=1.0,
           beta=0.0, what=""):
    x = x.double()
    K = x.shape[1]
    z, S = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    err = (K + 4) * 2.0 ** -23 * S
    if act == "swiglu":
        N = w.shape[0] // 2
        g, u, eg, eu = z[:, :N], z[:, N:], err[:, :N], err[:, N:]
        y = _act64(act, g, u, limit, alpha, beta)
        gg = g.clamp(max=limit) if limit > 0 else g
        gate = gg * torch.sigmoid(alpha * gg)
        slope = 1.2 * max(1.0, abs(alpha))
        e = (u.abs() + abs(beta) + eu) * slope * eg + gate.abs() * eu
    else:
        y = _act64(act, z, None, limit, alpha, beta)
        e = 1.2 * err
    e = e + y.abs() * 2.0 ** -19 + 2.0 ** -20
    if row_scale is not None:
        s = row_scale.double().reshape(-1, 1)
        y, e = y * s, e * s.abs() + (y * s).abs() * 2.0 ** -23
    if residual is not None:
        e = e + (y.abs() + residual.double().abs()) * 2.0 ** -23
        y = y + residual.double()
    e = e + (y.abs() + e) * (2.0 ** -8 if out.dtype == BF else 2.0 ** -23)
    assert out.shape == y.shape
    bad = ~((out.double() - y).abs() <= e)
    assert not bool(bad.any()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


SIZES = [   # M, N, K / 128
    (1, 1, 1), (1, 8, 2), (1, 513, 16), (2, 17, 3), (3, 100, 9), (4, 512, 16), (5, 256, 1),
    (7, 1171, 10), (8, 64, 40), (15, 33, 7), (16, 700, 56), (16, 48, 130), (17, 130, 5),
    (31, 64, 16), (33, 20, 24), (47, 1000, 16), (64, 129, 8), (65, 256, 12), (100, 72, 33),
    (128, 300, 4), (129, 65, 17), (300, 520, 8),
]


@pytest.mark.parametrize("fmt,group", GROUPS)
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(fmt, group, gated):
    for i, (M, N, kb) in enumerate(SIZES):
        for K in (128 * kb, 128 * kb - group) if kb > 1 else (128, group):
            x = _rand((M, K), i)
            W, w = _weight(fmt, group, N, K, gated, seed=i)
            for odt in (BF, F32):
                out = linear4(x, W, activation="swiglu" if gated else "none", out_dtype=odt)
                _check(out, x, w, "swiglu" if gated else "none", what=(M, N, K, odt))


@pytest.mark.parametrize("fmt,group", GROUPS)
@pytest.mark.parametrize("gated", [False, True])
def test_every_form(fmt, group, gated):
    """Each kernel, whole and with K split, with the whole epilogue; and x at odd
    addresses, copied first."""
    for i, (form, M, N, K) in enumerate(forms(fmt, group, gated)):
        big = _rand((M, K + 8), i)
        W, w = _weight(fmt, group, N, K, gated, seed=70 + i)
        b = _rand((w.shape[0],), 2, 0.5, F32)
        r = _rand((M, N), 4, 1.0, BF if i % 2 else F32)
        for act in ("swiglu",) if gated else ("none", "gelu"):
            x = big[:, :K]
            out = linear4(x, W, bias=b, activation=act, residual=r, out_dtype=F32)
            _check(out, x, w, act, b, residual=r, what=(form, M, N, K, act))
            x = big[:, 1:K + 1]
            _check(linear4(x, W, activation=act), x, w, act, what=(form, M, N, K, "odd"))


@pytest.mark.parametrize("fmt,group", GROUPS)
@pytest.mark.parametrize("gated", [False, True])
def test_entry_without_a_workspace(fmt, group, gated):
    """No copy of x and no K split: other kernels, the same results up to rounding."""
    stream = torch.cuda.current_stream().cuda_stream
    for M, N, K, first in ((1, 40, 256, 1), (16, 2000, 8192, 0), (64, 260, 8192, 0), (50, 300, 640, 1),
                           (200, 205, 1280, 1), (130, 260, 4096, 0), (65, 64, 128, 3)):
        big = _rand((M, K + 8), M)
        x = big[:, first:first + K]
        W, w = _weight(fmt, group, N, K, gated, seed=M)
        for vec in (True, False):
            hold = torch.full((M, N + 4), 7.0, dtype=F32, device=DEV)
            out = hold[:, :N] if vec else hold[:, 1:N + 1]
            args = ARGS.pack(x.data_ptr(), W.data.data_ptr(), 0 if W.gs is None else W.gs.data_ptr(),
                             0, 0, 0, out.data_ptr(), 0, x.stride(0), 0, out.stride(0), 0, 0, M, N, K,
                             6 if gated else 3, fmt, group, 0, 0, 0, 0.0, 1.0, 0.0)
            assert _lib.load().xtu_linear4(args, stream) == 0
            _check(out, x, w, "swiglu" if gated else "gelu", what=(M, N, K, first))
            assert int((hold == 7.0).sum()) >= 4 * M


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("M", [1, 6, 16, 40, 140])
def test_epilogue(act, M):
    gated = act == "swiglu"
    for i, (fmt, group) in enumerate(GROUPS):
        N, K = (203, 384) if i % 2 else (204, 640)
        rows = 2 * N if gated else N
        x = _rand((M, K), i)
        W, w = _weight(fmt, group, N, K, gated, seed=50 + i)
        b = _rand((rows,), 2, 0.5, F32 if M % 2 else BF)
        s = torch.sigmoid(_rand((M, 1), 3, 1.0, F32))
        r = _rand((M, N), 4, 1.0, BF if M % 2 else F32)
        kw = dict(swiglu_limit=0.75, swiglu_alpha=1.7, swiglu_beta=1.0) if gated else {}
        ck = dict(limit=0.75, alpha=1.7, beta=1.0) if gated else {}
        for odt in (BF, F32):
            out = linear4(x, W, bias=b, activation=act, row_scale=s, residual=r, out_dtype=odt, **kw)
            _check(out, x, w, act, b, s, r, what=(fmt, odt), **ck)
        out = linear4(x, W, activation=act, row_scale=s[:, 0], **kw)
        _check(out, x, w, act, None, s, **ck)
        out = linear4(x, W, bias=b, activation=act, **kw)
        _check(out, x, w, act, b, **ck)


@pytest.mark.parametrize("fmt,group", GROUPS)
def test_strides_alignment_and_in_place(fmt, group):
    K = 384
    for M, N in ((1, 40), (5, 40), (16, 33), (50, 64), (130, 37)):
        W, w = _weight(fmt, group, N, K, seed=M)
        big = _rand((2 * M + 2, K + 16), 7)
        for view in (big[:M, :K], big[:M, 1:K + 1], big[1:M + 1, 8:K + 8], big[::2][:M, 2:K + 2],
                     big[:1, :K].expand(M, K)):
            _check(linear4(view, W, out_dtype=F32), view, w, what=(M, view.stride()))
        x = big[:M, :K]
        for cols in (N, N + 3, N + 8):
            hold = torch.full((M + 2, cols), 7.0, dtype=BF, device=DEV)
            out = hold[1:M + 1, cols - N:]
            assert linear4(x, W, out=out) is out
            _check(out, x, w)
            hold[1:M + 1, cols - N:] = 7.0   # nothing else is written
            assert bool((hold == 7.0).all())
            y = _rand((M, cols), 8, 1.0, F32)[:, :N]
            before = y.clone()
            linear4(x, W, residual=y, out=y)
            _check(y, x, w, residual=before)
            wide = _rand((M, cols), 9)[:, :N]
            _check(linear4(x, W, residual=wide, out_dtype=F32), x, w, residual=wide)


@pytest.mark.parametrize("fmt,group", GROUPS)
def test_values_past_the_rows_are_not_read(fmt, group):
    """NaN beside the rows and in K's padding stays out."""
    for K in (group, 128 + group, 640 - group if group < 128 else 640):
        for M in (1, 3, 16, 20, 70):
            big = torch.full((M + 1, K + 24), float("nan"), dtype=BF, device=DEV)
            big[:M, 8:K + 8] = _rand((M, K), K)
            W, w = _weight(fmt, group, 20, K, seed=K)
            out = linear4(big[:M, 8:K + 8], W, out_dtype=F32)
            _check(out, big[:M, 8:K + 8], w, what=(M, K))


@pytest.mark.parametrize("fmt,group", GROUPS)
def test_nan_and_infinity_stay_in_their_row(fmt, group):
    for M in (4, 16, 60):
        for act in ("none", "relu", "gelu", "swiglu"):
            W, w = _weight(fmt, group, 40, 256, act == "swiglu", seed=3)
            x = _rand((M, 256), 5)
            x[2, 100] = float("nan")
            out = linear4(x, W, activation=act, swiglu_limit=1.0, out_dtype=F32)
            rows = torch.arange(M, device=DEV) != 2
            assert out[2].isnan().all() and out[rows].isfinite().all(), (act, M)
    x = _rand((3, 256), 6)
    x[1, 7] = float("inf")
    W, w = _weight(fmt, group, 40, 256, seed=4)
    out = linear4(x, W, out_dtype=F32)
    want = torch.where(w[:, 7] == 0, float("nan"), w[:, 7].sign() * float("inf"))
    assert torch.equal(out[1].isnan(), want.isnan())
    assert bool((out[1] == want)[~want.isnan()].all()) and out[[0, 2]].isfinite().all()


def test_scales_over_their_range():
    """e8m0 from 0 to 252, e4m3 from its smallest to 448, INT4's -8 and far scales."""
    x = _rand((3, 64), 1, 0.5)
    codes = torch.full((16, 32), 0x77, dtype=torch.uint8)   # 6
    for b in (0, 1, 20, 127, 200, 250):
        W = Weight4.from_dense("mxfp4", codes.to(DEV), torch.full((16, 2), b, dtype=torch.uint8,
                                                                  device=DEV))
        w = torch.full((16, 64), 6 * 2.0 ** (b - 127), dtype=torch.float64, device=DEV)
        out = linear4(x * 0.01, W, out_dtype=F32)
        y = (x * 0.01).double() @ w.t()
        S = (x * 0.01).double().abs() @ w.t()
        assert bool(((out.double() - y).abs() <= 68 * 2.0 ** -23 * S + 2.0 ** -140).all()), b
    for b in (0x01, 0x08, 0x7e, 0x81):
        W = Weight4.from_dense("nvfp4", codes.to(DEV),
                               torch.full((16, 4), b, dtype=torch.uint8, device=DEV), 1e-3)
        sv = torch.tensor([b], dtype=torch.uint8).view(torch.float8_e4m3fn).double().item()
        w = torch.full((16, 64), 6 * sv * torch.tensor(1e-3).double().item(), dtype=torch.float64,
                       device=DEV)
        _check(linear4(x, W, out_dtype=F32), x, w)
    lowest = torch.zeros((16, 32), dtype=torch.uint8)       # code 0: -8
    for s in (1e-30, 1.0, 1e30):
        W = Weight4.from_dense("int4", lowest.to(DEV), torch.full((16, 1), s, device=DEV))
        sv = torch.tensor(s).double().item()
        out = linear4(x, W, out_dtype=F32)
        y = x.double().sum(1, keepdim=True) * (-8 * sv)
        S = x.double().abs().sum(1, keepdim=True) * 8 * sv
        assert bool(((out.double() - y).abs() <= 68 * 2.0 ** -23 * S).all()), s


def test_no_rows():
    W, _ = _weight(F.FMT_MXFP4, 32, 40, 64)
    assert linear4(_rand((0, 64), 1), W).shape == (0, 40)


def test_same_bits_other_stream_and_graph():
    """Eager calls, calls on another stream at the same time, and replays between
    eager calls, on new inputs each."""
    cases = []
    for i, (M, N, K, fmt, group, act) in enumerate([
            (1, 512, 2048, 2, 32, "swiglu"), (16, 1000, 7168, 3, 16, "none"),
            (7, 200, 1184, 4, 32, "gelu"), (50, 512, 4096, 2, 32, "none"),
            (200, 320, 2048, 4, 128, "swiglu")]):
        W, w = _weight(fmt, group, N, K, act == "swiglu", seed=i)
        cases.append((_rand((M, K), i), W, w, act))
    run = lambda stream=None: [linear4(x, W, activation=act, out_dtype=F32, stream=stream)  # noqa: E731
                               for x, W, _, act in cases]
    first = run()
    for o, (x, W, w, act) in zip(first, cases):
        _check(o, x, w, act)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        here, there = run(), run(side)
        torch.cuda.synchronize()
        for a, b, c in zip(first, here, there):
            assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for seed in range(4):
        for i, (x, _, _, _) in enumerate(cases):
            x.copy_(_rand(tuple(x.shape), 100 + 10 * seed + i))
        want = [o.clone() for o in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_beside_the_bf16_product():
    """A shared expert in 4 bits added to a routed sum, as a layer runs it: gate/up,
    down with its gate as row scale, in place."""
    from xtu_moe_amd.linear import linear
    H, I = 512, 256
    for M in (1, 9, 70):
        W13, w13 = _weight(F.FMT_NVFP4, 16, I, H, True, seed=1)
        W2, w2 = _weight(F.FMT_NVFP4, 16, H, I, seed=2)
        x, v = _rand((M, H), 3), _rand((1, H), 4, 0.05)
        y = _rand((M, H), 5, 1.0, F32)
        routed = y.clone()
        act = linear4(x, W13, activation="swiglu")
        _check(act, x, w13, "swiglu")
        g = linear(x, v, activation="sigmoid", out_dtype=F32)
        linear4(act, W2, row_scale=g, residual=y, out=y)
        _check(y, act, w2, row_scale=g, residual=routed)
