"""The expert layer has no backward: routing weights that require a gradient are
refused by every entry that takes them, on the host, before anything runs."""
import types

import pytest
import torch
from torch.autograd import forward_ad

from xtu_moe_amd import cpu_split, layer, ring
from xtu_moe_amd.cpu_experts import CpuExperts
from xtu_moe_amd.cpu_split import PoolSplitLayer
from xtu_moe_amd.host_layer import HostResidentLayer

T, K, H = 3, 2, 32
X, IDS = torch.zeros((T, H), dtype=torch.bfloat16), torch.zeros((T, K), dtype=torch.int32)
W = types.SimpleNamespace(fmt=2, H=H, I=H, E=4, n_shared=0)


def _bare(cls):
    return object.__new__(cls)


ENTRIES = {
    "moe_forward": lambda w: layer.moe_forward(X, IDS, w, W),
    "combine": lambda w: layer.combine(None, None, w, None),
    "split": lambda w: cpu_split.pin_split(IDS, w, IDS, 4),
    "split layer": lambda w: _bare(PoolSplitLayer).forward(X, IDS, w),
    "host engine": lambda w: _bare(CpuExperts).forward(X, IDS, w),
    "host decode": lambda w: _bare(CpuExperts).cpu_decode(0, T, K, X, IDS, w, X),
    "host layer": lambda w: _bare(HostResidentLayer).forward(X, IDS, w),
    "ring": lambda w: ring.gpu_moe_layer_from_engine_tiled(None, X, IDS, w, H, H, 4, K, device="cpu"),
}


@pytest.mark.parametrize("name", list(ENTRIES))
def test_weights_that_require_a_gradient(name):
    logits = torch.zeros((T, K), requires_grad=True)
    for w in (logits, torch.softmax(logits, 1), torch.nn.Parameter(torch.ones((T, K)))):
        with pytest.raises(ValueError, match="no backward"):
            ENTRIES[name](w)


@pytest.mark.parametrize("name", list(ENTRIES))
def test_weights_with_a_tangent(name):
    """A forward-mode tangent, under no_grad too (which does not stop it)."""
    with forward_ad.dual_level():
        w = forward_ad.make_dual(torch.ones((T, K)), torch.ones((T, K)))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="forward-mode"):
                ENTRIES[name](w)


@pytest.mark.parametrize("name", list(ENTRIES))
def test_others_pass(name):
    """Under no_grad, in inference mode and without a gradient the check says nothing:
    what is raised is of what comes behind it."""
    w = torch.ones((T, K), requires_grad=True)
    for mode, t in ((torch.no_grad, w), (torch.inference_mode, w), (torch.enable_grad, w.detach())):
        with mode():
            try:
                ENTRIES[name](t)
            except Exception as e:   # noqa: BLE001
                assert "backward" not in str(e)
