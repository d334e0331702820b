"""NaN stays NaN through every activation, clamped or not, of the dense product
and of the MoE block, and stays where it belongs."""
import pytest
import torch

from test_gpu_linear import _rand
from test_gpu_linear_forms import _raw
from test_linear_plan import FORMS, plan
from xtu_moe_amd import formats as F
from xtu_moe_amd.block import MoeBlock
from xtu_moe_amd.layer import ExpertWeights, moe_forward
from xtu_moe_amd.linear import ACTIVATIONS, linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
NAN = float("nan")
SIZES = [(3, 64, 512), (16, 41, 200), (200, 96, 136), FORMS[0, True][1][0], FORMS[0, True][1][1]]


@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, act, limit):
    """Of a row of x: its whole row of the output; of a row of w: its column."""
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K), 110), _rand((rows, K), 111, 0.05)
    kw = dict(activation=act, swiglu_limit=limit, out_dtype=F32)
    ref = linear(x, w, **kw)
    x2 = x.clone()
    x2[M - 1, K // 2] = NAN
    out = linear(x2, w, **kw)
    assert bool(out[M - 1].isnan().all()) and torch.equal(out[:M - 1], ref[:M - 1])
    for row in {N - 1, rows - 1}:   # swiglu: of the gate, then of the up product
        w2 = w.clone()
        w2[row, 0] = NAN
        out = linear(x, w2, **kw)
        assert bool(out[:, N - 1].isnan().all()) and torch.equal(out[:, :N - 1], ref[:, :N - 1])
        b = torch.zeros(rows, device=DEV)
        b[row] = NAN
        out = linear(x, w, bias=b, **kw)
        assert bool(out[:, N - 1].isnan().all()) and torch.equal(out[:, :N - 1], ref[:, :N - 1])


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
def test_product_of_operands_that_no_tile_takes(act):
    M, N, K = 65, 33, 65
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K + 1), 112)[:, 1:], _rand((rows, K + 1), 113, 0.05)[:, 1:]
    ref = _raw(x, w, act)
    x[3, 7] = NAN
    out = _raw(x, w, act)
    assert bool(out[3].isnan().all()) and torch.equal(out[4:], ref[4:])


@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("fmt,plane", [("bf16", "gate"), ("bf16", "up"), ("fp8", "gate"),
                                       ("fp8", "up"), ("nvfp4", "gate"), ("nvfp4", "up")])
def test_block(fmt, plane, limit):
    """Of one expert's weights or scales: the tokens that use the expert, all
    of their outputs, and no other token."""
    E, K, H, I = 8, 2, 256, 256
    f = F.fmt_of(fmt)
    g = torch.Generator(device=DEV).manual_seed(4)
    w13 = torch.empty((E, 2 * I, H), device=DEV).normal_(0, 0.1, generator=g)
    w2 = torch.empty((E, H, I), device=DEV).normal_(0, 0.1, generator=g)
    q13, s13, g13 = F.quantize_w13(f, w13)
    q2, s2, g2 = F.quantize(f, w2)
    gate = torch.empty((E, H), device=DEV).normal_(0, 0.1, generator=g).to(BF)

    def block():
        # (planes that need no packing are taken as they are: the clean block's own)
        own = [None if t is None else t.clone() for t in (q13, s13, q2, s2, g13, g2)]
        return MoeBlock(gate, ExpertWeights.from_dense(f, *own), top_k=K, swiglu_limit=limit)

    clean, bad, up = block(), 5, int(plane == "up")
    if fmt == "bf16":
        q13[bad, I * up + 9, 100] = NAN
    elif fmt == "fp8":
        s13[bad, 2 * up, 1] = NAN        # block rows: two of the gate, two of the up half
    else:
        g13 = g13[:, None].expand(-1, 2).clone() if g13.dim() == 1 else g13
        g13[bad, up] = NAN
    poisoned = block()
    for T in (1, 2, 8, 16):
        x = torch.empty((T, H), device=DEV).normal_(0, 1, generator=g).to(BF)
        x[0] = (gate[bad].float() * 10).to(BF)      # token 0 chooses the expert
        for odt in (BF, F32):
            ref, rw, ri = clean(x, return_routing=True, out_dtype=odt)
            out, wts, ids = poisoned(x, return_routing=True, out_dtype=odt)
            assert torch.equal(ids, ri) and torch.equal(wts, rw)
            hit = (ids == bad).any(1)
            assert bool(hit[0]) and bool((T < 8) | (~hit).any())
            assert bool(out[hit].isnan().all())
            assert torch.equal(out[~hit], ref[~hit]) and bool(ref.isfinite().all())


@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp4", "nvfp4"])
def test_block_token(fmt, limit):
    """Of one token: its whole row, for few tokens and for more."""
    E, K, H, I = 8, 2, 256, 256
    f = F.fmt_of(fmt)
    g = torch.Generator(device=DEV).manual_seed(5)
    w13 = torch.empty((E, 2 * I, H), device=DEV).normal_(0, 0.1, generator=g)
    w2 = torch.empty((E, H, I), device=DEV).normal_(0, 0.1, generator=g)
    q13, s13, g13 = F.quantize_w13(f, w13)
    q2, s2, g2 = F.quantize(f, w2)
    gate = torch.empty((E, H), device=DEV).normal_(0, 0.1, generator=g).to(BF)
    blk = MoeBlock(gate, ExpertWeights.from_dense(f, q13, s13, q2, s2, g13, g2), top_k=K,
                   swiglu_limit=limit)
    for T in (1, 2, 8, 16, 24):
        x = torch.empty((T, H), device=DEV).normal_(0, 1, generator=g).to(BF)
        x[T - 1, 3] = NAN
        out, wts, ids = blk(x, return_routing=True)
        assert bool(out[T - 1].isnan().all()) and bool(out[:T - 1].isfinite().all())
        assert bool(((ids >= 0) & (ids < E)).all())


@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("T", [1, 3, 24, 96, 700])
def test_layer(fmt, limit, T):
    """The expert layer over given routing: a token of NaN has its whole row.
    (MXFP4 prefills write activations as fp6 and fp4 pieces, which hold no NaN.)"""
    if fmt == "mxfp4" and T > 96:
        return
    E, K, H, I = 8, 2, 512, 256
    f = F.fmt_of(fmt)
    g = torch.Generator(device=DEV).manual_seed(6)
    w13 = torch.empty((E, 2 * I, H), device=DEV).normal_(0, 0.1, generator=g)
    w2 = torch.empty((E, H, I), device=DEV).normal_(0, 0.1, generator=g)
    q13, s13, g13 = F.quantize_w13(f, w13)
    q2, s2, g2 = F.quantize(f, w2)
    W = ExpertWeights.from_dense(f, q13, s13, q2, s2, g13, g2)
    x = torch.empty((T, H), device=DEV).normal_(0, 1, generator=g).to(BF)
    ids = torch.stack([torch.randperm(E, generator=g, device=DEV)[:K] for _ in range(T)])
    ids, wts = ids.to(torch.int32), torch.full((T, K), 0.5, device=DEV)
    ref = moe_forward(x, ids, wts, W, swiglu_limit=limit).clone()
    x[T // 2, 7] = NAN
    out = moe_forward(x, ids, wts, W, swiglu_limit=limit)
    keep = torch.arange(T, device=DEV) != T // 2
    assert torch.equal(out[keep], ref[keep]) and bool(out[T // 2].isnan().all())
