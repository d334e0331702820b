"""The quant-method hook given hidden states alone: the router's product from
the layer's gate rows, and a MoE layer built of the block and dense products.

The hook's outputs are held to the block's and the products' own float64
bounds (test_gpu_block, test_gpu_linear), each from its actual inputs."""
import types

import pytest
import torch

import test_gpu_linear as TL
from helpers import make_dense_layer
from test_gpu_block import _block, _check as check_block, _layer, _router, _x
from xtu_moe_amd import formats as F
from xtu_moe_amd import host_layer as HL
from xtu_moe_amd.block import MoeBlock
from xtu_moe_amd.layer import moe_forward, route
from xtu_moe_amd.linear import linear
from xtu_moe_amd.mixed_experts import (XiaotuExpertsBF16, XiaotuExpertsFp8, XiaotuExpertsMxfp4,
                                       XiaotuExpertsNvfp4)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
HOOKS = {"bf16": (XiaotuExpertsBF16, None), "fp8": (XiaotuExpertsFp8, "weight_scale_inv"),
         "mxfp4": (XiaotuExpertsMxfp4, "weight_scale"),
         "nvfp4": (XiaotuExpertsNvfp4, "weight_scale")}


def _hook(fmt, E, H, I, K, sigmoid, seed, **attrs):
    """(hook, gate rows, routing arguments) of a layer with a gate."""
    cls, scale = HOOKS[fmt]
    d = make_dense_layer(getattr(F, "FMT_" + fmt.upper()), E, H, I, seed=seed)
    gate, kw = _router(E, H, sigmoid, seed)
    lay = types.SimpleNamespace(layer_name="model.layers.1.mlp.experts", w13_weight=d["w13"],
                                w2_weight=d["w2"], top_k=K, renormalize=True,
                                scoring_func=kw["scoring"], swiglu_limit=7.0,
                                gate=types.SimpleNamespace(weight=torch.nn.Parameter(gate)))
    if sigmoid:
        kw.update(n_group=4, topk_group=2)
        lay.use_grouped_topk, lay.num_expert_group, lay.topk_group = True, 4, 2
        lay.routed_scaling_factor = 2.5
        lay.gate.e_score_correction_bias = kw["bias"]
    if scale:
        setattr(lay, "w13_" + scale, d["s13"])
        setattr(lay, "w2_" + scale, d["s2"])
    if fmt == "nvfp4":
        lay.w13_weight_scale_2, lay.w2_weight_scale_2 = d["gs13"], d["gs2"]
    for k, v in attrs.items():
        setattr(lay, k, v)
    hook = cls()
    hook.process_weights_after_loading(lay)
    return hook, gate, kw


def _same_bits(a, b):
    torch.cuda.synchronize()
    assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("fmt", sorted(HOOKS))
def test_hook_takes_the_router_product(fmt, sigmoid):
    """The hook's answer is the block's over its weights, for few tokens and
    more, into a given output and without one."""
    hook, gate, kw = _hook(fmt, 32, 512, 256, 4, sigmoid, 5)
    blk = MoeBlock(gate, hook._weights, top_k=4, swiglu_limit=7.0, **kw)
    for T in (1, 3, 16, 40):
        x = _x(T, 512, T)
        want = blk(x)
        _same_bits(hook.apply(x, None, None), want)
        buf = torch.full((T, 512), 9.0, dtype=BF, device=DEV)
        assert hook.apply(x, None, None, output=buf) is buf
        _same_bits(buf, want)
        _same_bits(hook.apply(x.float(), None, None), blk(x, out_dtype=F32))
        y = x.clone()                                    # in place
        assert hook.apply(y, None, None, output=y) is y
        _same_bits(y, want)
    assert hook.apply(_x(0, 512, 0), None, None).shape == (0, 512)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_gate_rewritten_between_calls(sigmoid):
    hook, gate, kw = _hook("mxfp4", 32, 512, 256, 4, sigmoid, 6)
    x = _x(5, 512, 5)
    hook.apply(x, None, None)
    lay = hook._layer_ref
    gate2 = _router(32, 512, sigmoid, 9)[0]
    lay.gate.weight.data = gate2.clone()                 # another tensor
    blk = MoeBlock(gate2, hook._weights, top_k=4, swiglu_limit=7.0, **kw)
    _same_bits(hook.apply(x, None, None), blk(x))
    lay.gate.weight.data.copy_(gate)                     # in place
    blk = MoeBlock(gate, hook._weights, top_k=4, swiglu_limit=7.0, **kw)
    _same_bits(hook.apply(x, None, None), blk(x))


def test_logit_bias_expert_map_and_unaligned_rows():
    """What the block does not take: the product gives logits, and the layer's
    own routing follows."""
    E, H, K = 32, 512, 4
    hook, gate, kw = _hook("fp8", E, H, 256, K, False, 7)
    lay, x = hook._layer_ref, _x(6, H, 6)

    def want(logits, em=None):
        w, i = route(logits, top_k=K)
        if em is not None:
            i = em.to(DEV)[i.long()]
            w, i = torch.where(i < 0, 0.0, w), i.clamp(min=0).to(torch.int32)
        return moe_forward(x, i.contiguous(), w.contiguous(), hook._weights, swiglu_limit=7.0)

    plain = linear(x, gate, out_dtype=F32)
    em = torch.full((E,), -1, dtype=torch.int32)
    em[::2] = torch.arange(E // 2, dtype=torch.int32)
    _same_bits(hook.apply(x, None, None, expert_map=em), want(plain, em))
    lay.gate.bias = torch.linspace(-2, 2, E, device=DEV, dtype=BF)
    _same_bits(hook.apply(x, None, None),
               hook.apply(x, None, None,
                          router_logits=linear(x, gate, bias=lay.gate.bias, out_dtype=F32)))
    del lay.gate.bias
    off = torch.empty(E * H + 1, dtype=BF, device=DEV)[1:].view(E, H)
    off.copy_(gate)
    lay.gate.weight = off
    _same_bits(hook.apply(x, None, None), hook.apply(x, None, None, router_logits=plain))


def test_int8_and_host_resident_layers_route_for_themselves(monkeypatch):
    monkeypatch.setenv("XIAOTU_MOE_INT8_ALIGN", "1")
    hook, gate, kw = _hook("mxfp4", 32, 512, 256, 4, True, 8)
    x = _x(24, 512, 8)
    logits = linear(x, gate, out_dtype=F32)
    _same_bits(hook.apply(x, None, None), hook.apply(x, None, None, router_logits=logits))
    monkeypatch.delenv("XIAOTU_MOE_INT8_ALIGN")
    monkeypatch.setenv(HL.RESIDENT_LAYERS_ENV, "0-0")    # layer 1 stays in host memory
    monkeypatch.setenv(HL.PIN_SLOTS_ENV, "0")
    host, gate, kw = _hook("mxfp4", 32, 512, 256, 4, True, 8)
    assert host._weights is None
    _same_bits(host.apply(x, None, None), host.apply(x, None, None, router_logits=logits))


def test_without_a_gate_refused():
    hook, gate, kw = _hook("bf16", 8, 256, 128, 2, False, 9)
    lay, x = hook._layer_ref, _x(2, 256, 2)
    for w in (gate.float(), gate[:, :128], gate.cpu(), gate[0], None):
        lay.gate.weight = w
        with pytest.raises(ValueError, match="router_logits"):
            hook.apply(x, None, None)
    del lay.gate
    with pytest.raises(ValueError, match="router_logits"):
        hook.apply(x, None, None)


def test_gate_of_another_size_refused():
    hook, gate, kw = _hook("bf16", 8, 256, 128, 2, False, 9)
    lay, x = hook._layer_ref, _x(2, 256, 2)
    em = torch.arange(8, dtype=torch.int32)
    for w, m in ((gate[:6].clone(), None), (torch.cat([gate, gate]), None), (gate, em[:7]),
                 (torch.cat([gate, gate]), em)):
        lay.gate.weight = w
        with pytest.raises(ValueError, match="rows do not fit"):
            hook.apply(x, None, None, expert_map=m)
    lay.gate.weight, lay.gate.bias = gate, torch.zeros(7, device=DEV)
    with pytest.raises(ValueError, match="rows do not fit"):
        hook.apply(x, None, None)


class _Net:
    """Two MoE layers with unquantised shared experts, as a model runs them:
    h += routed(h) + sigmoid(h . v) * down(swiglu(gate/up(h)))."""

    def __init__(self, H, I, Is):
        self.parts = []
        for fmt, spec, seed in (("mxfp4", (64, 0, 6, H, I, 1, False), 1),
                                ("nvfp4", (60, 0, 4, H, I, 0, False), 2)):
            blk, dense, _, kw = _block(fmt, spec, swiglu_limit=7.0)
            self.parts.append((blk, dense, kw, TL._rand((2 * Is, H), seed, 0.04),
                               TL._rand((H, Is), seed + 10, 0.04),
                               TL._rand((1, H), seed + 20, 0.02)))

    def __call__(self, h, check=False):
        for blk, dense, kw, w13, w2, v in self.parts:
            res = blk(h, return_routing=True, out_dtype=F32)
            routed = res[0].clone() if check else res[0]
            scale = linear(h, v, activation="sigmoid", out_dtype=F32)
            act = linear(h, w13, activation="swiglu", swiglu_limit=7.0)
            moe = linear(act, w2, row_scale=scale, residual=res[0], out=res[0])
            if check:
                check_block(blk, dense, h, (routed, res[1], res[2]), None, kw)
                TL._check(scale, h, v, "sigmoid")
                TL._check(act, h, w13, "swiglu", limit=7.0)
                TL._check(moe, act, w2, row_scale=scale, residual=routed)
            h = (h + moe).to(BF)
        return h


@pytest.mark.parametrize("T", [1, 5, 16, 33, 200])
def test_layers_run_together(T):
    net = _Net(512, 256, 384)
    x = _x(T, 512, T)
    first = net(x, check=True)
    _same_bits(net(x), first)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = net(x)
    for k in range(4):
        x.copy_(_x(T, 512, 50 + k))
        g.replay()
        _same_bits(out, net(x))


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("how", ["none given", "data", "copy", "passed", "replaced"])
def test_sigmoid_gate_bias_selects_once(how, T):
    """A sigmoid gate's bias is the selection's: the block with it is the
    answer, however the layer holds it."""
    E, H, K = 32, 512, 4
    cls, scale = HOOKS["mxfp4"]
    d = make_dense_layer(F.FMT_MXFP4, E, H, 256, seed=11)
    gate, kw = _router(E, H, True, 11)
    kw["bias"] *= 10                       # enough to change the choice
    first = kw["bias"].flip(0).contiguous() if how == "replaced" else kw["bias"]
    bias = torch.nn.Parameter(first.clone())
    lay = types.SimpleNamespace(layer_name="model.layers.1.mlp.experts", w13_weight=d["w13"],
                                w2_weight=d["w2"], top_k=K, renormalize=True, swiglu_limit=7.0,
                                scoring_func="sigmoid", routed_scaling_factor=2.5,
                                gate=types.SimpleNamespace(weight=gate, bias=bias))
    lay.w13_weight_scale, lay.w2_weight_scale = d["s13"], d["s2"]
    if how == "data":
        lay.e_score_correction_bias = bias.data
    elif how == "copy":
        lay.e_score_correction_bias = bias.detach().clone()
    hook = cls()
    hook.process_weights_after_loading(lay)
    if how == "replaced":
        lay.gate.bias = torch.nn.Parameter(kw["bias"].clone())
    more = dict(e_score_correction_bias=bias.detach().clone()) if how == "passed" else {}
    x = _x(T, H, 12)
    blk = MoeBlock(gate, hook._weights, top_k=K, swiglu_limit=7.0, **kw)
    out = hook.apply(x, None, None, **more)
    _same_bits(out, blk(x))
    logits = linear(x, gate, out_dtype=F32)
    if T > 16:
        _same_bits(hook.apply(x, None, None, router_logits=logits), out)
    twice = route(logits + kw["bias"], top_k=K, **kw)[1]
    assert not torch.equal(twice, blk(x, return_routing=True)[2])


@pytest.mark.parametrize("em", [False, True])
def test_grouped_softmax_refused(em):
    """Groups, a scaling factor or a selection bias are not part of the softmax
    selection: from hidden states alone the hook says so."""
    E, H = 32, 512
    hook, gate, kw = _hook("fp8", E, H, 256, 4, False, 13, use_grouped_topk=True)
    x = _x(6, H, 13)
    m = torch.arange(E, dtype=torch.int32) if em else None
    want = hook.apply(x, None, None, expert_map=m)   # one group, no factor: plain softmax
    _same_bits(want, MoeBlock(gate, hook._weights, top_k=4, swiglu_limit=7.0)(x)
               if not em else want)
    for name, value in (("num_expert_group", 4), ("topk_group", 2), ("routed_scaling_factor", 2.5),
                        ("e_score_correction_bias", torch.zeros(E, device=DEV))):
        before = getattr(hook, name)
        with pytest.raises(ValueError, match="go with sigmoid"):
            hook.apply(x, None, None, expert_map=m, **{name: value})
        setattr(hook, name, before)
    hook._layer_ref.gate.bias = torch.linspace(-2, 2, E, device=DEV)   # a term of the logits
    hook.apply(x, None, None, expert_map=m)
    hook._read_layer_attrs(hook._layer_ref)
    _same_bits(hook.apply(x, None, None, expert_map=m),
               hook.apply(x, None, None, expert_map=m, router_logits=linear(
                   x, gate, bias=hook._layer_ref.gate.bias, out_dtype=F32)))
