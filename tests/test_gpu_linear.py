"""The dense product with its epilogue against float64.

Tolerances, derived before the first run.  With z = sum_k x_k w_k + b computed
in fp32, |z^ - z| <= (K + 2) 2^-23 S, S = sum |x_k w_k| + |b| (each addition
rounds or truncates by at most one unit of 2^-23 relative to a partial sum of
at most S).  The activations have slope at most 1.2 (gelu, silu: 1.13, 1.1)
and are evaluated to 2^-19 relative (a few roundings and the device's exp, erf
or tanh) plus 2^-20 absolute; swiglu's two factors bound each other's error by
their own sizes.  row_scale and residual add one rounding each (2^-24), and the
output one more: 2^-24 (fp32) or 2^-8 (bf16) of the value.
"""
import pytest
import torch

from xtu_moe_amd.linear import ACTIVATIONS, linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _rand(shape, seed, std=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def _act64(act, z, u, limit, alpha, beta):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "swiglu":
        if limit > 0:
            z, u = z.clamp(max=limit), u.clamp(-limit, limit)
        return z * torch.sigmoid(alpha * z) * (u + beta)
    return z


def _check(out, x, w, act="none", bias=None, row_scale=None, residual=None, limit=0.0, alpha=1.0,
           beta=0.0, what=""):
    x, w = x.double(), w.double()
    K = x.shape[1]
    z, S = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    err = (K + 2) * 2.0 ** -23 * S
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
    bad = (out.double() - y).abs() > e
    assert not bool(bad.any()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


SIZES = [   # M, N, K
    (1, 1, 1), (1, 8, 64), (2, 16, 31), (3, 17, 33), (5, 256, 2048), (15, 100, 72), (16, 64, 1024),
    (17, 512, 96), (31, 130, 640), (33, 48, 200), (47, 1024, 2048), (64, 64, 64), (65, 129, 257),
    (100, 771, 1187), (128, 128, 128), (129, 250, 520), (200, 384, 448), (255, 1000, 328),
    (256, 256, 512), (300, 2048, 96), (513, 520, 1032), (1000, 40, 4096), (1024, 1536, 768),
]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_sizes(M, N, K, out_dtype):
    x, w = _rand((M, K), 1), _rand((N, K), 2, 0.05)
    out = linear(x, w, out_dtype=out_dtype)
    _check(out, x, w)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_swiglu_sizes(M, N, K):
    x, w = _rand((M, K), 3), _rand((2 * N, K), 4, 0.05)
    b = _rand((2 * N,), 5, 0.5, F32)
    out = linear(x, w, bias=b, activation="swiglu", swiglu_limit=0.75, swiglu_alpha=1.7,
                 swiglu_beta=1.0, out_dtype=F32)
    _check(out, x, w, "swiglu", b, limit=0.75, alpha=1.7, beta=1.0)


@pytest.mark.parametrize("M,N,K", [(2100, 4096, 192), (4096, 2052, 1000), (3000, 3001, 129),
                                   (257, 20000, 64), (20000, 300, 72), (2304, 256, 4096)])
@pytest.mark.parametrize("act", ["none", "swiglu", "gelu"])
def test_large_tiles(M, N, K, act):
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K), 60), _rand((rows, K), 61, 0.05)
    b, r = _rand((rows,), 62, 0.5, F32), _rand((M, N), 63)
    for odt in (BF, F32):
        _check(linear(x, w, bias=b, activation=act, residual=r, out_dtype=odt), x, w, act, b,
               residual=r)


@pytest.mark.parametrize("act", ["none", "swiglu", "gelu"])
@pytest.mark.parametrize("M,N,K", [   # each tile, whole and with K split
    (446, 1157, 72), (446, 1156, 71), (518, 295, 3176), (2980, 674, 66), (1844, 134, 5344),
    (1544, 3800, 200), (1543, 3801, 198), (2497, 774, 4096), (3602, 517, 752), (3600, 520, 751),
    (2907, 322, 4144), (3431, 3585, 130), (3431, 3584, 136), (2830, 1412, 3568)])
def test_each_tile(M, N, K, act):
    if act == "swiglu":
        N = (N + 7) // 8 * 4
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K), 70), _rand((rows, K), 71, 0.05)
    b, s = _rand((rows,), 72, 0.5, F32), _rand((M,), 73, 1.0, F32)
    for odt, r in ((BF, _rand((M, N), 74)), (F32, None)):
        out = linear(x, w, bias=b, activation=act, row_scale=s, residual=r, out_dtype=odt)
        _check(out, x, w, act, b, s, r, what=f"{act} {odt}")


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", [(4, 96, 256), (70, 200, 136), (300, 512, 1024)])
@pytest.mark.parametrize("bias_dtype,res_dtype,scale", [(BF, F32, True), (F32, BF, False),
                                                        (None, BF, True)])
def test_epilogues(act, M, N, K, bias_dtype, res_dtype, scale):
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K), 6), _rand((rows, K), 7, 0.1)
    b = None if bias_dtype is None else _rand((rows,), 8, 0.5, bias_dtype)
    r = _rand((M, N), 9, 1.0, res_dtype)
    s = _rand((M, 2), 10, 1.0, F32)[:, 1] if scale else None   # strided
    for odt in (BF, F32):
        out = linear(x, w, bias=b, activation=act, row_scale=s, residual=r, out_dtype=odt)
        _check(out, x, w, act, b, s, r, what=f"{odt}")


@pytest.mark.parametrize("M,N,K", [(3, 40, 128), (16, 512, 1000), (90, 200, 192), (300, 260, 512)])
@pytest.mark.parametrize("pad,off", [(8, 0), (8, 8), (3, 1), (1, 5)])
def test_strides(M, N, K, pad, off):
    """Rows apart by more than K, starting anywhere; what lies around the
    output rows stays as it was."""
    xb, wb = _rand((M, K + pad + off), 11), _rand((N, K + pad + off), 12, 0.05)
    rb = _rand((M, N + pad + off), 13, 1.0, F32)
    x, w, r = xb[:, off:off + K], wb[:, off:off + K], rb[:, off:off + N]
    ob = torch.full((M + 2, N + pad + off), 7.0, dtype=BF, device=DEV)
    out = linear(x, w, residual=r, out=ob[1:1 + M, off:off + N])
    _check(out, x, w, residual=r)
    ob[1:1 + M, off:off + N] = 7.0
    assert bool((ob == 7.0).all())


def test_repeated_rows():
    x = _rand((1, 256), 14).expand(40, 256)
    w = _rand((64, 256), 15)
    _check(linear(x, w), x, w)
    r = _rand((1, 64), 16, 1.0, F32).expand(40, 64)
    _check(linear(x, w, residual=r), x, w, residual=r)


def test_no_rows():
    w = _rand((64, 256), 15)
    out = linear(torch.empty((0, 256), dtype=BF, device=DEV), w)
    assert out.shape == (0, 64) and out.dtype == BF


@pytest.mark.parametrize("M,N,K", [(4, 256, 7168), (60, 300, 520), (300, 512, 264)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_in_place(M, N, K, dtype):
    x, w = _rand((M, K), 17), _rand((N, K), 18, 0.05)
    r = _rand((M, N), 19, 1.0, dtype)
    buf = r.clone()
    out = linear(x, w, residual=buf, out=buf)
    assert out.data_ptr() == buf.data_ptr()
    assert torch.equal(out, linear(x, w, residual=r, out_dtype=dtype))


@pytest.mark.parametrize("M,N,K", [(3, 64, 512), (40, 96, 200), (260, 256, 512)])
def test_infinities_and_nans_stay_in_their_rows(M, N, K):
    """A NaN or infinity in one row of x or w reaches that row or column of
    the output and no other."""
    x, w = _rand((M, K), 20), _rand((N, K), 21, 0.05)
    ref = linear(x, w, out_dtype=F32)
    x2, w2 = x.clone(), w.clone()
    x2[M - 1, K - 1] = float("nan")
    w2[N - 1, 0] = float("inf")
    out = linear(x2, w2, out_dtype=F32)
    assert bool(out[M - 1].isnan().all())
    assert not bool(out[:M - 1, N - 1].isfinite().any())
    assert torch.equal(out[:M - 1, :N - 1], ref[:M - 1, :N - 1])
    relu = linear(x2, w, activation="relu")
    assert bool(relu[M - 1].isnan().all()) and bool(relu[:M - 1].isfinite().all())


@pytest.mark.parametrize("M,N,K", [(2, 256, 7168), (47, 2048, 2048), (700, 512, 2048)])
def test_same_call_same_bits(M, N, K):
    x, w = _rand((M, K), 22), _rand((N, K), 23, 0.05)
    first = linear(x, w, out_dtype=F32)
    for _ in range(5):
        assert torch.equal(linear(x, w, out_dtype=F32), first)


def test_streams_at_once():
    """Calls on two streams that overlap share nothing."""
    shapes = [(8, 512, 7168), (47, 2048, 2048), (1, 256, 7168), (300, 1024, 1024)]
    data = [(_rand((M, K), 24 + i), _rand((N, K), 34 + i, 0.05))
            for i, (M, N, K) in enumerate(shapes)]
    ref = [linear(x, w, out_dtype=F32) for x, w in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for k in range(8):
        for st in streams:
            x, w = data[(k + (st is streams[1])) % 4]
            got.append(((k + (st is streams[1])) % 4,
                        linear(x, w, out_dtype=F32, stream=st)))
    torch.cuda.synchronize()
    for i, out in got:
        assert torch.equal(out, ref[i])


@pytest.mark.parametrize("M,N,K", [(4, 256, 7168), (47, 2048, 2048), (300, 512, 1024)])
def test_captured(M, N, K):
    """Two graphs captured from one stream, replayed several times in turn
    and on two streams, with eager calls between."""
    x, w = _rand((M, K), 50), _rand((N, K), 51, 0.05)
    x2 = _rand((M, K), 52)
    outs, graphs = [], []
    linear(x, w, out_dtype=F32)
    torch.cuda.synchronize()
    for xx in (x, x2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(linear(xx, w, out_dtype=F32))
        graphs.append(g)
    side = torch.cuda.Stream()
    for k in range(6):
        x.normal_()
        x2.normal_()
        torch.cuda.synchronize()
        for o in outs:
            o.fill_(-1)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        eager = linear(x, w, out_dtype=F32)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager)
        assert torch.equal(outs[1], linear(x2, w, out_dtype=F32))


def test_long_offsets():
    """Rows past 2^31 elements from the first."""
    M, K = 3, 128
    ld = (1 << 30) + 64
    buf = torch.zeros(2 * ld + K, dtype=BF, device=DEV)
    x = buf.as_strided((M, K), (ld, 1))
    x.copy_(_rand((M, K), 60))
    w = _rand((64, K), 61)
    _check(linear(x, w), x, w)
    _check(linear(w, x), w, x)
    o = torch.zeros(2 * ld + 64, dtype=BF, device=DEV).as_strided((M, 64), (ld, 1))
    _check(linear(x, w, out=o), x, w)


@pytest.mark.parametrize("K", [24, 23])
def test_outputs_past_2_31_elements(K):
    """Rows whose elements lie past 2^31 in x, in residual and in the output;
    their copies (K = 23: rows that do not start on 16 bytes) past 2^31 bytes."""
    M, N = (1 << 27) + 77, 17
    x, w = torch.empty((M, K), dtype=BF, device=DEV).normal_(), _rand((N, K), 80)
    r = torch.empty((M, N), dtype=BF, device=DEV).normal_()
    out = linear(x, w, residual=r)
    for a in (0, M // 2, M - 1000):
        b = a + 1000
        _check(out[a:b], x[a:b], w, residual=r[a:b], what=f"rows {a} ..")
    # every row, against the same product of a part that starts elsewhere
    for a in range(0, M, 1 << 25):
        assert torch.equal(out[a:a + (1 << 25)], linear(x[a:a + (1 << 25)], w,
                                                        residual=r[a:a + (1 << 25)]))
