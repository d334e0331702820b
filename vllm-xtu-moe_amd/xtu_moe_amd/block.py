"""The MoE block from hidden states: router product, selection, routed and
shared experts.

    logits = x Wg^T;  (ids, weights) = selection(logits)
    y = sum_k weights_k E_{ids_k}(x) + sum_s g_s S_s(x),   g_s = sigmoid(x . v_s) or 1

The layer entries of this package begin at router logits or at ids, as the
reference's hook does (vllm_xiaotu_moe/mixed_experts.py:1919-2123); the block
begins where a model's MoE layer does, at the hidden states, with the
reference host's router (hybrid_model.py:1877) and shared expert (:1752)
inside.
"""
from __future__ import annotations

import contextlib
import struct

import torch

from . import _lib
from .formats import FMT_BF16, FMT_FP8, FMT_MXFP4, FMT_NVFP4
from .layer import ExpertWeights, _same_device, moe_forward, route, scratch_per_call
from .linear import _current_device, _overlap, linear, on_stream, raw_stream

# xtu_few_args: x, gate, shared_gate, bias, six planes, out, ids, weights,
# workspace; its bytes; fmt, T, H, I, E, n_shared, K, mode, renormalize, n_group,
# topk_group, out_bf16; routed_scaling, limit, alpha, beta
ARGS = struct.Struct("@14PN12i4f")
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 16, 64   # the routers' limits


def _check_rows(name, t, n, H, dev=None):
    """Raises ValueError where t is not bf16 rows [n, H] (on dev, starting on 16
    bytes) that the kernels can read."""
    if t.shape != (n, H) or t.dtype is not torch.bfloat16 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous bf16 [{n}, {H}], got {tuple(t.shape)} {t.dtype}")
    if dev is not None:
        if t.get_device() != dev.index:
            _same_device(dev, **{name: t})
        if t.data_ptr() & 15:
            raise ValueError(f"{name} must start on 16 bytes")


def check_selection(scoring, bias=None, n_group=1, topk_group=1, routed_scaling_factor=1.0,
                    renormalize=True):
    """Raises ValueError for a selection that the routers do not make: they
    would choose among all experts by the softmax, unscaled."""
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"unsupported scoring function {scoring!r}")
    if scoring == "softmax" and (bias is not None or int(n_group) != 1 or int(topk_group) != 1
                                 or float(routed_scaling_factor) != 1.0):
        raise ValueError("a selection bias, groups and a scaling factor go with sigmoid scoring")


class MoeBlock:
    """One layer's MoE block over resident experts.

    gate_weight: bf16 [E, H], the router's rows.  weights: ExpertWeights (E
    routed, then n_shared shared experts).  scoring "softmax" (no groups, bias
    or scaling factor: those are refused) or "sigmoid" (grouped, selection by
    score + bias), with the arguments of ``route``.
    shared_gate: bf16 [n_shared, H]; shared expert s is scaled by
    sigmoid(x . shared_gate[s]) (without it by 1).  swiglu_*: the clamped gated
    SiLU of every expert.  Every call reads the tensors given here as they are
    then, in the storage that they have then (their owner may write them or put
    other storage under them, ``param.data = ...``, between calls); ones that no
    longer fit are refused.
    """

    def __init__(self, gate_weight, weights: ExpertWeights, *, top_k, scoring="softmax",
                 renormalize=True, bias=None, n_group=1, topk_group=1, routed_scaling_factor=1.0,
                 shared_gate=None, swiglu_limit=0.0, swiglu_alpha=1.0, swiglu_beta=0.0):
        W = weights
        self.check(gate_weight, W, top_k=top_k, scoring=scoring, bias=bias, n_group=n_group,
                   topk_group=topk_group, routed_scaling_factor=routed_scaling_factor,
                   shared_gate=shared_gate)
        if not W.w13.is_cuda:
            raise ValueError("the block needs device-resident expert weights")
        if W.fmt not in (FMT_BF16, FMT_FP8, FMT_MXFP4, FMT_NVFP4) or W.n_slots != W.n_experts:
            raise ValueError("the block needs BF16, FP8, MXFP4 or NVFP4 planes of every expert")
        self.W, self.gate_weight, self.shared_gate, self.bias = W, gate_weight, shared_gate, bias
        self._dev = W.device
        self.top_k, self.scoring, self.renormalize = int(top_k), scoring, bool(renormalize)
        self.n_group, self.topk_group = int(n_group), int(topk_group)
        self.routed_scaling_factor = float(routed_scaling_factor)
        self.limit = float(swiglu_limit or 0.0)
        self.alpha, self.beta = float(swiglu_alpha), float(swiglu_beta)
        self._operands()
        # the packed planes stay where they are (held here as they lie)
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self._held = tuple(None if t is None else t.detach()
                           for t in (W.w13, W.s13, W.gs13, W.w2, W.s2, W.gs2))
        self._planes = tuple(ptr(t) for t in self._held)
        self._shape = (W.H, W.I, W.E, W.n_shared, self.top_k, int(scoring == "sigmoid"),
                       self.renormalize, self.n_group, self.topk_group)
        self._floats = (self.routed_scaling_factor, self.limit, self.alpha, self.beta)
        self._few_bytes = {}   # workspace by token count, of the few
        self._entry = _lib.load().xtu_few_block
        # the shared experts as further routed ones: their weight is then the
        # gate's (the same planes)
        self._W_all = None
        if shared_gate is not None:
            self._W_all = ExpertWeights(W.fmt, W.H, W.I, W.n_experts, 0, W.w13, W.s13, W.w2, W.s2,
                                        W.gs13, W.gs2, mutable=W.mutable,
                                        fp8_scales_ok=W.slot_fp8_scales_ok)

    @staticmethod
    def check(gate_weight, W, *, top_k, scoring="softmax", bias=None, n_group=1, topk_group=1,
              routed_scaling_factor=1.0, shared_gate=None):
        """Raises ValueError for a router or shared gate that does not fit W."""
        if gate_weight is None:
            raise ValueError("gate_weight is missing")
        if shared_gate is not None and W.n_shared == 0:
            raise ValueError("shared_gate without shared experts")
        _check_rows("gate_weight", gate_weight, W.E, W.H)
        if shared_gate is not None:
            _check_rows("shared_gate", shared_gate, W.n_shared, W.H)
        check_selection(scoring, bias, n_group, topk_group, routed_scaling_factor)
        if bias is not None and tuple(bias.shape) != (W.E,):
            raise ValueError(f"bias must be [{W.E}], got {tuple(bias.shape)}")
        top_k, n_group, topk_group = int(top_k), int(n_group), int(topk_group)
        if not 1 <= top_k <= min(W.E, MAX_TOP_K):
            raise ValueError(f"top_k {top_k} is not in 1 .. min(E, {MAX_TOP_K})")
        if W.E > MAX_EXPERTS:
            raise ValueError(f"{W.E} routed experts, at most {MAX_EXPERTS}")
        if scoring == "sigmoid" and (not 1 <= n_group <= MAX_GROUPS or W.E % n_group
                                     or not 1 <= topk_group <= n_group
                                     or top_k > topk_group * (W.E // n_group)):
            raise ValueError(f"{n_group} groups with {topk_group} kept do not fit {W.E} experts, "
                             f"top {top_k}")

    def _operands(self):
        """(gate_weight, shared_gate, bias fp32 or None) as they are now, checked
        against the layer: the kernels take their addresses."""
        W, gate, shared, bias = self.W, self.gate_weight, self.shared_gate, self.bias
        _check_rows("gate_weight", gate, W.E, W.H, self._dev)
        if shared is not None:
            _check_rows("shared_gate", shared, W.n_shared, W.H, self._dev)
        if bias is not None:
            if bias.shape != (W.E,):
                raise ValueError(f"bias must be [{W.E}], got {tuple(bias.shape)}")
            if bias.get_device() != self._dev.index:
                _same_device(self._dev, bias=bias)
            if bias.dtype is not torch.float32 or not bias.is_contiguous():
                bias = bias.to(torch.float32).contiguous()
        return gate, shared, bias

    def __call__(self, x, *, out=None, out_dtype=None, return_routing=False, stream=None):
        """x bf16 [T, H] -> [T, H] bf16 (or out_dtype fp32, or into out); with
        return_routing (out, topk_weights fp32 [T, K], topk_ids int32 [T, K])."""
        W = self.W
        if x.dim() != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous() \
                or x.shape[1] != W.H:
            raise ValueError(f"x must be contiguous bf16 [T, {W.H}], got {tuple(x.shape)} {x.dtype}")
        odt = out.dtype if out is not None else out_dtype or torch.bfloat16
        if odt not in (torch.bfloat16, torch.float32) or (out_dtype or odt) != odt:
            raise ValueError(f"output type {odt} (out_dtype {out_dtype}): bf16 or fp32")
        if out is not None and (tuple(out.shape) != tuple(x.shape) or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {tuple(x.shape)}, got {tuple(out.shape)}")
        _same_device(self._dev, x=x, out=out)
        if stream is not None or self._dev.index != _current_device():
            with on_stream(stream, self._dev):
                return self(x, out=out, out_dtype=out_dtype, return_routing=return_routing)
        if out is not None and _overlap(out, x):
            raise ValueError("out overlaps x")
        operands = self._operands()
        if out is None:
            out = torch.empty(x.shape, dtype=odt, device=x.device)
        T = x.shape[0]
        need = self._few_bytes.get(T)
        if need is None:
            need = int(_lib.call("xtu_few_workspace_bytes", W.fmt, T, W.E, self.top_k, W.n_shared,
                                 W.H, W.I)) if T else 0
            if need:
                self._few_bytes[T] = need
        ids = x.new_empty((T, self.top_k), dtype=torch.int32)
        wts = x.new_empty((T, self.top_k), dtype=torch.float32)
        if need:
            self._few(x, out, ids, wts, need, *operands)
        elif T:
            # (eagerly the stream's scratch: calls on it run in order)
            capturing = torch.cuda.is_current_stream_capturing()
            with scratch_per_call() if capturing else contextlib.nullcontext():
                self._composed(x, out, ids, wts, *operands)
        return (out, wts, ids) if return_routing else out

    def _few(self, x, out, ids, wts, need, gate, shared, bias):
        """A few tokens, in two launches."""
        if x.data_ptr() & 15:
            x = x.clone()
        # per call: calls on other streams, and graphs, have their own
        ws = x.new_empty(need, dtype=torch.uint8)
        rc = self._entry(ARGS.pack(x.data_ptr(), gate.data_ptr(),
                                   0 if shared is None else shared.data_ptr(),
                                   0 if bias is None else bias.data_ptr(), *self._planes,
                                   out.data_ptr(), ids.data_ptr(), wts.data_ptr(), ws.data_ptr(),
                                   need, self.W.fmt, x.shape[0], *self._shape,
                                   out.dtype == torch.bfloat16, *self._floats),
                         raw_stream(x.device.index))
        if rc:
            _lib.check("xtu_few_block", rc)

    def _composed(self, x, out, ids, wts, gate, shared, bias):
        """Any number of tokens: the products and the layer one after the other."""
        logits = linear(x, gate, out_dtype=torch.float32)
        kw = dict(scoring=self.scoring, bias=bias, n_group=self.n_group,
                  topk_group=self.topk_group, routed_scaling_factor=self.routed_scaling_factor,
                  renormalize=self.renormalize)
        act = dict(swiglu_limit=self.limit, swiglu_alpha=self.alpha, swiglu_beta=self.beta,
                   out=out)
        if shared is None:
            moe_forward(x, ids, wts, self.W, router=dict(logits=logits, **kw), **act)
            return
        route(logits, top_k=self.top_k, ids_out=ids, wts_out=wts, **kw)
        gates = linear(x, shared, activation="sigmoid", out_dtype=torch.float32)
        sids = torch.arange(self.W.E, self.W.n_experts, dtype=torch.int32, device=x.device)
        moe_forward(x, torch.cat([ids, sids.expand(x.shape[0], -1)], 1),
                    torch.cat([wts, gates], 1), self._W_all, **act)
