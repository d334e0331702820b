"""The router's training step: what is refused on the host, before a launch."""
import os

import pytest
import torch

from xtu_moe_amd import _lib
from xtu_moe_amd.router import ARGS, router_losses

I32 = torch.int32


def _refused(match, *args, **kw):
    with pytest.raises(ValueError, match=match):
        router_losses(*args, **kw)


def test_arguments_refused():
    lg, ids = torch.zeros((3, 8)), torch.zeros((3, 2), dtype=I32)
    _refused("scoring", lg, ids, scoring="tanh")
    _refused("scaling factor", lg, ids, routed_scaling_factor=2.5)
    for f in (0.0, -1.0, float("inf"), float("nan")):
        _refused("positive", lg, ids, scoring="sigmoid", routed_scaling_factor=f)
    _refused("2-D", lg[0], ids)
    _refused("2-D", lg.half(), ids)
    _refused("2-D", lg.double(), ids)
    _refused("contiguous", torch.zeros((8, 3)).t(), ids)
    _refused("1024", torch.zeros((3, 1025)), ids)
    _refused("1024", torch.zeros((3, 0)), ids)
    _refused("ids", lg, ids.long())
    _refused("ids", lg, ids[:2])
    _refused("ids", lg, torch.zeros((3, 4), dtype=I32)[:, ::2])
    _refused("16", lg, torch.zeros((3, 17), dtype=I32))
    _refused("16", lg, torch.zeros((3, 0), dtype=I32))
    _refused("seq_starts", lg, ids, seq_starts=torch.zeros(1, dtype=I32))
    _refused("seq_starts", lg, ids, seq_starts=torch.zeros(3))
    _refused("seq_starts", lg, ids, seq_starts=torch.zeros((2, 2), dtype=I32))
    _refused("seq_starts", lg, ids, seq_starts=torch.zeros(6, dtype=I32)[::2])
    _refused("CUDA", lg, ids)
    _refused("rows", lg[:1].expand((1 << 30) + 1, 8), ids)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_entries_refuse_on_the_host():
    lib = _lib.load()

    def pack(logits=16, ids=16, starts=0, weights=16, stat=16, counts=16, probs=16, balance=16,
             z=16, norm=16, ws=16, ld=8, nws=1 << 40, T=4, E=8, K=2, S=1, mode=0, renorm=1, bf16=0,
             scale=1.0):
        return ARGS.pack(logits, ids, starts, weights, stat, counts, probs, balance, z, norm, ws,
                         ld, nws, T, E, K, S, mode, renorm, bf16, scale)

    assert lib.xtu_router_losses(None, None) == 1
    assert lib.xtu_router_grad(None, 0, 0, 0, 16, None) == 1
    both = (dict(logits=0), dict(ids=0), dict(weights=0), dict(stat=0), dict(counts=0),
            dict(norm=0), dict(ld=-1), dict(T=-1), dict(T=(1 << 30) + 1), dict(E=0), dict(E=1025),
            dict(K=0), dict(K=17), dict(S=0), dict(S=2), dict(mode=2), dict(scale=0.0),
            dict(scale=float("nan")), dict(scale=float("inf")), dict(logits=2), dict(ids=2),
            dict(S=1 << 24, starts=16, E=1024))
    for bad in both:
        assert lib.xtu_router_losses(pack(**bad), None) == 1, bad
        assert lib.xtu_router_grad(pack(**bad), 0, 0, 0, 16, None) == 1, bad
    for bad in (dict(probs=0), dict(balance=0), dict(z=0), dict(mode=1), dict(ws=0), dict(ws=8),
                dict(nws=lib.xtu_router_workspace_bytes(4, 8, 1) - 1)):
        assert lib.xtu_router_losses(pack(**bad), None) == 1, bad
    assert lib.xtu_router_grad(pack(), 0, 0, 0, 0, None) == 1
    assert lib.xtu_router_grad(pack(), 0, 0, 0, 8, None) == 1
    assert lib.xtu_router_grad(pack(mode=1), 0, 0, 16, 16, None) == 1   # z is softmax's
    assert lib.xtu_router_grad(pack(T=0, logits=0, ids=0), 0, 0, 0, 0, None) == 0   # nothing to do
    for bad in ((-1, 8, 1), ((1 << 30) + 1, 8, 1), (4, 0, 1), (4, 1025, 1), (4, 8, 0)):
        assert lib.xtu_router_workspace_bytes(*bad) == 0
    assert lib.xtu_router_workspace_bytes(0, 8, 1) > 0   # no rows: the sums of none


def test_tangents_refused():
    """No forward-mode derivative: a result without one would lose it silently."""
    from torch.autograd import forward_ad
    lg, ids = torch.zeros((3, 8)), torch.zeros((3, 2), dtype=I32)
    with forward_ad.dual_level():
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                _refused("forward-mode", forward_ad.make_dual(lg, torch.ones_like(lg)), ids)
                _refused("CUDA", lg, ids)


def test_limits_refused():
    """What the entry does not take is a ValueError, not a library error."""
    lg, ids = torch.zeros((3, 1024)), torch.zeros((3, 2), dtype=I32)
    for E, most in ((1024, (1 << 18) - 1), (17, (1 << 23) - 1), (16, (1 << 24) - 1)):
        starts = torch.zeros(most + 2, dtype=I32)
        _refused("sixteens", lg[:, :E], ids, seq_starts=starts)
        _refused("CUDA", lg[:, :E], ids, seq_starts=starts[1:])
    for f in (1e39, 2.0 ** 128, 1e-39, 5e-324):
        _refused("positive", lg, ids, scoring="sigmoid", routed_scaling_factor=f)
    for f in (2.0 ** -126, torch.finfo(torch.float32).max):
        _refused("CUDA", lg, ids, scoring="sigmoid", routed_scaling_factor=f)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_limits_are_the_entrys():
    lib = _lib.load()
    for E, most in ((1024, (1 << 18) - 1), (17, (1 << 23) - 1), (16, (1 << 24) - 1)):
        assert lib.xtu_router_workspace_bytes(4, E, most) > 0
        assert lib.xtu_router_workspace_bytes(4, E, most + 1) == 0
