"""The MoE block's refusals, before any launch."""
import pytest
import torch

from xtu_moe_amd import formats as F
from xtu_moe_amd.block import MoeBlock
from xtu_moe_amd.layer import ExpertWeights

BF = torch.bfloat16


def _weights(E=4, NS=1, H=256, I=128):
    n = E + NS
    return ExpertWeights.from_dense(F.FMT_BF16, torch.zeros((n, 2 * I, H), dtype=BF), None,
                                    torch.zeros((n, H, I), dtype=BF), None, n_shared=NS)


def test_weights_must_be_resident():
    with pytest.raises(ValueError, match="device-resident"):
        MoeBlock(torch.zeros((4, 256), dtype=BF), _weights(), top_k=2)


@pytest.mark.parametrize("kw,match", [
    (dict(top_k=0), "top_k"), (dict(top_k=5), "top_k"), (dict(top_k=17), "top_k"),
    (dict(top_k=2, scoring="tanh"), "scoring"),
    (dict(top_k=2, bias=torch.zeros(4)), "sigmoid"),
    (dict(top_k=2, scoring="sigmoid", bias=torch.zeros(5)), "bias"),
    (dict(top_k=2, scoring="sigmoid", n_group=3), "groups"),
    (dict(top_k=2, scoring="sigmoid", n_group=4, topk_group=1), "groups"),
    (dict(top_k=2, scoring="sigmoid", n_group=2, topk_group=3), "groups"),
    (dict(top_k=2, gate=torch.zeros((5, 256), dtype=BF)), "gate_weight"),
    (dict(top_k=2, gate=torch.zeros((4, 256))), "gate_weight"),
    (dict(top_k=2, gate=torch.zeros((4, 512), dtype=BF)[:, ::2]), "gate_weight"),
    (dict(top_k=2, gate=None), "gate_weight"),
    (dict(top_k=2, shared_gate=torch.zeros((2, 256), dtype=BF)), "shared_gate"),
    (dict(top_k=2, shared_gate=torch.zeros((1, 256))), "shared_gate"),
])
def test_arguments_refused(kw, match):
    kw = dict(kw)
    gate = kw.pop("gate", torch.zeros((4, 256), dtype=BF))
    with pytest.raises(ValueError, match=match):
        MoeBlock.check(gate, _weights(), **kw)


def test_shared_gate_needs_shared_experts():
    with pytest.raises(ValueError, match="shared"):
        MoeBlock.check(torch.zeros((4, 256), dtype=BF), _weights(NS=0), top_k=2,
                       shared_gate=torch.zeros((0, 256), dtype=BF))


@pytest.mark.parametrize("kw", [
    dict(n_group=2, topk_group=1), dict(n_group=2, topk_group=2), dict(topk_group=2),
    dict(routed_scaling_factor=2.5), dict(routed_scaling_factor=0.0), dict(bias=torch.zeros(4)),
])
def test_softmax_takes_no_groups_bias_or_scale(kw):
    gate = torch.zeros((4, 256), dtype=BF)
    with pytest.raises(ValueError, match="go with sigmoid"):
        MoeBlock.check(gate, _weights(), top_k=2, scoring="softmax", **kw)
    with pytest.raises(ValueError, match="go with sigmoid"):
        MoeBlock(gate, _weights(), top_k=2, scoring="softmax", **kw)
    MoeBlock.check(gate, _weights(), top_k=2, scoring="softmax", n_group=1, topk_group=1,
                   routed_scaling_factor=1.0)
    if kw.get("topk_group", 1) <= kw.get("n_group", 1):
        MoeBlock.check(gate, _weights(), top_k=1, scoring="sigmoid", **kw)
