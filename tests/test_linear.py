"""The dense product's refusals: everything that the kernels could not take
is turned away on the host, before a launch."""
import os

import pytest
import torch

from xtu_moe_amd import _lib
from xtu_moe_amd.linear import ACTIVATIONS, ARGS, linear

BF = torch.bfloat16


def _xw(M=3, N=4, K=8):
    return torch.zeros((M, K), dtype=BF), torch.zeros((N, K), dtype=BF)


def _refused(match, *args, **kw):
    with pytest.raises(ValueError, match=match):
        linear(*args, **kw)


def test_operands_refused():
    x, w = _xw()
    _refused("2-D", x[0], w)
    _refused("2-D", x.float(), w)
    _refused("2-D", x, w.half())
    _refused("columns", x, w[:, :7])
    _refused("contiguous", torch.zeros((8, 3), dtype=BF).t(), w)
    _refused("contiguous", x, torch.zeros((8, 4), dtype=BF).t())
    _refused("at least one row", x, w[:0])
    _refused("at least one row", x[:, :0], w[:, :0])
    _refused("CUDA", x, w)


def test_activations_refused():
    x, w = _xw()
    _refused("unknown activation", x, w, activation="tanh")
    _refused("even number", x, w[:3], activation="swiglu")
    for name in ACTIVATIONS:   # the others get as far as the device check
        _refused("CUDA", x, w, activation=name)


def test_epilogue_operands_refused():
    x, w = _xw()
    f32 = torch.float32
    _refused("bias", x, w, bias=torch.zeros(3))
    _refused("bias", x, w, bias=torch.zeros(4, dtype=torch.float16))
    _refused("bias", x, w, bias=torch.zeros(8)[::2])
    _refused("bias", x, w, bias=torch.zeros(2), activation="swiglu")   # 2N values
    _refused("row_scale", x, w, row_scale=torch.zeros(4))
    _refused("row_scale", x, w, row_scale=torch.zeros(3, dtype=BF))
    _refused("residual", x, w, residual=torch.zeros((2, 4), dtype=f32))
    _refused("columns", x, w, residual=torch.zeros((3, 3), dtype=f32))
    _refused("residual", x, w, residual=torch.zeros((3, 4), dtype=torch.float64))
    _refused("residual", x, w, residual=torch.zeros((4, 3), dtype=f32).t())


def test_outputs_refused():
    x, w = _xw()
    _refused("output type", x, w, out_dtype=torch.float16)
    _refused("output type", x, w, out=torch.zeros((3, 4), dtype=BF), out_dtype=torch.float32)
    _refused("does not hold", x, w, out=torch.zeros((2, 4), dtype=BF))
    _refused("does not hold", x, w, out=torch.zeros((1, 4), dtype=BF).expand(3, 4))
    _refused("columns", x, w, out=torch.zeros((3, 5), dtype=BF))
    both = torch.zeros((3, 16), dtype=BF)
    _refused("overlaps x", both[:, :8], w, out=both[:, 4:8])
    _refused("overlaps residual", x, w, residual=both[:, 0:4], out=both[:, 2:6])
    buf = torch.zeros((4, 4), dtype=BF)
    _refused("overlaps residual", x, w, residual=buf[:3], out=buf[1:])
    _refused("CUDA", x, w, residual=buf[:3], out=buf[:3])   # in place: allowed


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_entry_refuses_on_the_host():
    call = _lib.load().xtu_linear

    def rc(x=16, ldx=8, w=16, ldw=8, M=1, N=1, K=1, act=0, out=16, ldo=8, ldr=0, sst=0, ws=0):
        return call(ARGS.pack(x, w, 0, 0, 0, out, ws, ldx, ldw, ldr, ldo, sst, 0, M, N, K, act, 0,
                              0, 1, 0.0, 1.0, 0.0), None)

    assert call(None, None) == 1
    assert rc(M=0) == 0                       # nothing to do, nothing launched
    for bad in (dict(x=0), dict(w=0), dict(out=0), dict(M=-1), dict(N=0), dict(K=0),
                dict(act=7), dict(act=-1), dict(ldx=-1), dict(ldw=-1), dict(ldr=-1),
                dict(sst=-1), dict(ws=8), dict(M=2, N=9), dict(N=1 << 29), dict(K=1 << 29),
                dict(M=1 << 30, N=1 << 20, ldo=1 << 20)):
        assert rc(**bad) == 1, bad


def test_sizes_past_the_kernels_indices_refused():
    """The kernels count rows in 32 bits, up to a tile past the last one."""
    x, w = _xw(1, 4, 8)
    for rows in ((1 << 31) - 511, (1 << 31) - 1, 1 << 31, 1 << 33):
        _refused("rows", x.expand(rows, 8), w)
    _refused("CUDA", x.expand((1 << 31) - 512, 8), w)
    for act in ("none", "swiglu"):   # N columns: 2N rows of w for swiglu
        _refused("columns", x, w[:1].expand((2 if act == "swiglu" else 1) * (1 << 28) + 2, 8),
                 activation=act)
        _refused("CUDA", x, w[:1].expand((2 if act == "swiglu" else 1) * (1 << 28), 8),
                 activation=act)
    long = torch.empty((1, (1 << 28) + 1), dtype=BF)   # (never touched)
    _refused("columns", long, long)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_entry_refuses_row_counts_on_the_host():
    lib = _lib.load()
    for M in ((1 << 31) - 511, (1 << 31) - 1):
        assert lib.xtu_linear(ARGS.pack(16, 16, 0, 0, 0, 16, 0, 8, 8, 0, 8, 0, 0, M, 1, 1, 0, 0, 0,
                                        1, 0.0, 1.0, 0.0), None) == 1
        assert lib.xtu_linear_workspace_bytes(M, 1, 1, 0, 0) == 0
    assert lib.xtu_linear_workspace_bytes((1 << 31) - 512, 1, 1, 0, 0) > 0
