"""Every form of the dense product's tile kernel (tile, whole or K split, plain
or swiglu, vector or single-column epilogue), and the kernel for operands that
the tiles do not take, with each term of the epilogue; bounds as derived in
test_gpu_linear."""
import pytest
import torch

from test_gpu_linear import _check, _rand
from test_linear_plan import FORMS, plan
from xtu_moe_amd import _lib
from xtu_moe_amd.linear import ACTIVATIONS, ARGS, linear, raw_stream

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32

CASES = [(tile, split, act, M, N, K)
         for (tile, split), sides in sorted(FORMS.items())
         for gated, sizes in enumerate(sides) for M, N, K in sizes
         for act in (("swiglu",) if gated else ("none", "gelu_tanh"))]


@pytest.mark.parametrize("tile,split,act,M,N,K", CASES)
def test_forms(tile, split, act, M, N, K):
    got = plan(M, N, K, act)
    assert got[0] == tile and (got[1] > 1) == split
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K), 90), _rand((rows, K), 91, 0.05)
    s = _rand((M,), 92, 1.0, F32)
    for odt, bias, r in ((BF, F32, _rand((M, N), 93)), (F32, BF, _rand((M, N), 94, 1.0, F32)),
                         (F32, None, None)):
        b = None if bias is None else _rand((rows,), 95, 0.5, bias)
        sc = s if r is not None else None
        out = linear(x, w, bias=b, activation=act, row_scale=sc, residual=r, out_dtype=odt,
                     swiglu_limit=1.5)
        _check(out, x, w, act, b, sc, r, limit=1.5, what=f"{odt}")


def _raw(x, w, act="none", bias=None, row_scale=None, residual=None, out_dtype=F32, workspace=0):
    """xtu_linear with a workspace of so many bytes."""
    (M, K), rows = x.shape, w.shape[0]
    N = rows // 2 if act == "swiglu" else rows
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    bf = lambda t: t is not None and t.dtype == BF  # noqa: E731
    out = torch.full((M + 1, N), 7.0, dtype=out_dtype, device=DEV)
    ws = torch.full((workspace + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    rc = _lib.load().xtu_linear(
        ARGS.pack(p(x), p(w), p(bias), p(row_scale), p(residual), p(out),
                  p(ws) if workspace else 0, x.stride(0), w.stride(0),
                  0 if residual is None else residual.stride(0), N,
                  0 if row_scale is None else row_scale.stride(0), workspace, M, N, K,
                  ACTIVATIONS[act], bf(bias), bf(residual), out_dtype == BF, 1.5, 1.0, 0.0),
        raw_stream(torch.cuda.current_device()))
    _lib.check("xtu_linear", rc)
    assert bool((out[M] == 7.0).all()) and bool((ws[workspace:] == 0x5a).all())
    return out[:M]


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", [(17, 1, 1), (65, 33, 65), (100, 96, 63), (190, 131, 250)])
def test_operands_that_no_tile_takes(act, M, N, K):
    """Without a workspace to copy them to: x and w start on odd 2-byte
    addresses."""
    rows = 2 * N if act == "swiglu" else N
    x, w = _rand((M, K + 3), 96)[:, 1:1 + K], _rand((rows, K + 1), 97, 0.1)[:, 1:]
    b, s = _rand((rows,), 98, 0.5, BF), _rand((M, 2), 99, 1.0, F32)[:, 1]
    for odt, r in ((BF, _rand((M, N), 100, 1.0, F32)), (F32, _rand((M, N), 101))):
        _check(_raw(x, w, act, b, s, r, odt), x, w, act, b, s, r, limit=1.5)
        _check(_raw(x, w, act, None, None, None, odt), x, w, act, limit=1.5)


@pytest.mark.parametrize("act", ["none", "swiglu", "silu"])
def test_workspaces_of_every_size(act):
    """Less than the whole workspace: no K split, or no copy; never a byte
    behind it."""
    M, N, K = 70, 41, 1417
    rows = 2 * N if act == "swiglu" else N
    assert plan(M, N, K, act)[1] > 1
    for k, aligned in ((K, 0), (K - 1, 1)):
        x, w = _rand((M, k), 102), _rand((rows, k), 103, 0.05)
        whole = _lib.load().xtu_linear_workspace_bytes(M, N, k, ACTIVATIONS[act], aligned)
        assert whole > 0
        pack = 0 if aligned else (M + rows) * (-(-k // 8)) * 16
        for size in sorted({0, 16, max(pack - 16, 0), pack, pack + 16, whole - 16, whole}):
            _check(_raw(x, w, act, workspace=size), x, w, act, limit=1.5, what=f"{size} bytes")
