"""What the hook makes of a gate's bias: a term of the logits, or the selection's
own, which must not count in both places.  (What the operators make of the two is
tested on the GPU.)"""
import types

import pytest
import torch

from xtu_moe_amd.mixed_experts import XiaotuExpertsBF16

E, H, BF = 8, 256, torch.bfloat16


def _layer(bias=None, scoring="sigmoid", **attrs):
    gate = types.SimpleNamespace(weight=torch.zeros((E, H), dtype=BF))
    if bias is not None:
        gate.bias = bias
    return types.SimpleNamespace(gate=gate, top_k=2, scoring_func=scoring, **attrs)


def _hook(layer):
    hook = XiaotuExpertsBF16()
    hook._read_layer_attrs(layer)
    hook._weights = types.SimpleNamespace(E=E, H=H)
    return hook


def _terms(hook):
    """(bias of the logits, bias of the selection) of a call without logits."""
    w, logit = hook._gate(torch.zeros((2, H), dtype=BF))
    assert w is not None
    return logit, hook._selection_args(torch.device("cpu")).get("bias")


def _param(seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.nn.Parameter(torch.randn(E, generator=g).to(dtype))


ALIASES = {
    "none given": lambda b: {},
    "the same": lambda b: dict(e_score_correction_bias=b),
    "data": lambda b: dict(e_score_correction_bias=b.data),
    "detached": lambda b: dict(e_score_correction_bias=b.detach()),
    "another view": lambda b: dict(e_score_correction_bias=b.detach().view(2, 4).reshape(E)),
    "parameter of data": lambda b: dict(e_score_correction_bias=torch.nn.Parameter(b.data)),
    "clone": lambda b: dict(e_score_correction_bias=b.detach().clone()),
    "fp32 copy": lambda b: dict(e_score_correction_bias=b.detach().double().float()),
    "bf16 copy": lambda b: dict(e_score_correction_bias=b.detach().to(BF)),
}


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("how", sorted(ALIASES))
def test_sigmoid_gate_bias_counts_once(how, dtype):
    b = _param(1, dtype)
    layer = _layer(b, **ALIASES[how](b))
    logit, sel = _terms(_hook(layer))
    assert logit is None
    want = b if how != "bf16 copy" else b.to(BF)
    assert torch.equal(sel, want.detach().float())


@pytest.mark.parametrize("how", sorted(ALIASES))
def test_sigmoid_gate_bias_passed_to_the_call(how):
    """apply(e_score_correction_bias=...): the selection's, whatever tensor
    holds it; the gate's bias stays what it was at loading."""
    b = _param(2)
    hook = _hook(_layer(b))
    given = ALIASES[how](b).get("e_score_correction_bias")
    hook._take_selection_bias(given)
    logit, sel = _terms(hook)
    assert logit is None
    assert torch.equal(sel, (b if given is None else given).detach().float())
    other = _param(3).detach()
    hook._take_selection_bias(other)
    logit, sel = _terms(hook)
    assert logit is None and torch.equal(sel, other)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_replaced_after_loading(scoring):
    b = _param(4)
    layer = _layer(b, scoring)
    hook = _hook(layer)
    for new in (_param(5), _param(6).data):
        layer.gate.bias = new
        logit, sel = _terms(hook)
        if scoring == "softmax":
            assert torch.equal(logit, new.detach()) and sel is None
        else:
            assert logit is None and torch.equal(sel, new.detach())
    b2 = _param(7)
    layer.gate.bias = b2
    b2.data = _param(8).data
    logit, sel = _terms(hook)
    assert torch.equal((logit if scoring == "softmax" else sel), _param(8).detach())
    hook._read_layer_attrs(layer)        # loaded again
    assert torch.equal((_terms(hook)[0] if scoring == "softmax" else _terms(hook)[1]),
                       _param(8).detach())


def test_two_biases():
    """A selection bias of its own beside a gate's bias: the latter is the
    logits', also when either is replaced."""
    b, c = _param(9), _param(10)
    for layer in (_layer(b, e_score_correction_bias=c), _layer(b)):
        if not hasattr(layer, "e_score_correction_bias"):
            layer.gate.e_score_correction_bias = c
        hook = _hook(layer)
        logit, sel = _terms(hook)
        assert torch.equal(logit, b.detach()) and torch.equal(sel, c.detach())
        layer.gate.bias = _param(11)
        hook._take_selection_bias(_param(12).detach())
        logit, sel = _terms(hook)
        assert torch.equal(logit, _param(11).detach()) and torch.equal(sel, _param(12).detach())


def test_bias_that_came_after_loading_refused():
    """Nothing says what it is: with sigmoid scoring the call is refused."""
    for attrs in ({}, dict(e_score_correction_bias=_param(13))):
        layer = _layer(None, **attrs)
        hook = _hook(layer)
        assert _terms(hook)[0] is None
        layer.gate.bias = _param(14)
        with pytest.raises(ValueError, match="gate's bias"):
            _terms(hook)
        hook._take_selection_bias(layer.gate.bias.data)      # says what it is
        logit, sel = _terms(hook)
        assert logit is None and torch.equal(sel, _param(14).detach())
    soft = _layer(None, "softmax")
    hook = _hook(soft)
    soft.gate.bias = _param(14)
    assert torch.equal(_terms(hook)[0], _param(14).detach())


def test_bias_set_on_the_hook():
    hook = _hook(_layer(_param(15)))
    hook.e_score_correction_bias = _param(16).detach()
    logit, sel = _terms(hook)
    assert logit is None and torch.equal(sel, _param(16).detach())


def test_biases_of_zeros_say_nothing():
    """Two tensors of zeros may be a bias and its copy or two biases that are
    filled later: refused with sigmoid scoring, unless they share storage."""
    b = torch.nn.Parameter(torch.zeros(E))
    with pytest.raises(ValueError, match="gate's bias"):
        _terms(_hook(_layer(b, e_score_correction_bias=torch.zeros(E))))
    for c in (b, b.data):
        assert _terms(_hook(_layer(b, e_score_correction_bias=c)))[0] is None
    assert _terms(_hook(_layer(b)))[0] is None
