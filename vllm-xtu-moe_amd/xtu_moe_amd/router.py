"""The router's training step: losses, per-expert counts and the selected
experts' weights, with their gradient in the logits.

    ids = layer.route(logits, top_k=K)[1]
    r = router_losses(logits, ids)
    (0.01 * r.balance + 0.001 * r.z).backward()

``layer.route`` selects; this gives what a training step differentiates, and the
counts that say how evenly the experts are used (also to pick a pool's).
``weights`` carry a task loss's gradient where the caller combines the experts'
outputs differentiably; ``layer.moe_forward`` has no backward and refuses them
(``r.weights.detach()`` goes in).  The
reference serves only: its router (vllm_xiaotu_moe/hybrid_model.py:1877) has no
losses and no gradient.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from .block import MAX_EXPERTS, MAX_TOP_K
from .layer import _has_tangent, _same_device
from .linear import _current_device, on_stream, raw_stream

# xtu_router_args: logits, ids, starts, weights, stat, counts, probs, balance, z,
# norm, workspace; ld; its bytes; T, E, K, S, mode, renormalize, logits_bf16; scale
ARGS = struct.Struct("@11PlN7if")
MAX_ROWS = 1 << 30
MAX_PARTS = 1 << 24   # sequences times sixteens of experts, below: the second launch's grid
MIN_SCALE, MAX_SCALE = 2.0 ** -126, torch.finfo(torch.float32).max   # what the kernels hold
_WS_BYTES: dict = {}
_ENTRIES = None


class RouterLosses(NamedTuple):
    """weights fp32 [T, K]; balance and z fp32 scalars (z None with sigmoid
    scoring); counts int32 and probs fp32 [S, E], without gradient.  The backward
    reads weights and counts: to change them (an all-reduce), take a clone."""
    weights: torch.Tensor
    balance: torch.Tensor
    z: Optional[torch.Tensor]
    counts: torch.Tensor
    probs: torch.Tensor


def router_losses(logits, ids, *, scoring="softmax", renormalize=True, routed_scaling_factor=1.0,
                  seq_starts=None, stream=None) -> RouterLosses:
    """Losses, counts and weights of a selection; differentiable in logits.

    logits [T, E] fp32 or bf16, rows contiguous at any row stride; ids int32
    [T, K], the selected experts (an id outside 0 .. E - 1 is no expert: weight
    0, not counted).  scoring: "softmax" (p = softmax(logits)) or "sigmoid"
    (scores s = sigmoid(logits), p = s / sum s).  seq_starts int32 [S + 1] on
    the device: sequence q is rows seq_starts[q] .. seq_starts[q + 1]
    (ascending; values are clamped to 0 .. T); rows outside them get weights and
    take part in no loss and no count.  Without it all rows are one sequence.  At
    most 2^30 rows, S ceil(E / 16) < 2^24, and 2^31 - 1 selections of one expert in
    a sequence (counts are int32).

    weights: the selected experts' p (sigmoid: s), divided by their sum with
    renormalize, times routed_scaling_factor (sigmoid only), as ``route`` gives
    them.  balance: mean over non-empty sequences of E / (K n) sum_e counts_e
    P_e with n rows and P their mean p: 1 for even use.  z: mean over the
    sequences' rows of logsumexp(logits)^2.  A row of -inf has p = 0 and no
    gradient; NaN gives NaN, and so does +inf with softmax (sigmoid: its score is
    1).  Rows of far finite logits are as any (sigmoid: one whose largest is below -708,
    whose scores vanish in 64 bits too, is as a row of -inf); z is inf where a square
    leaves fp32.  Renormalised weights lose accuracy where every selected logit lies
    more than 70 below the row's largest, and are 0 from 87 on: their scores leave
    fp32 beside it.  fp32 arithmetic, sums over rows in fp32 up to
    a lane's 256 rows and in fp64 from there; the same call gives the same bits.  Once differentiable, backwards only.
    Capturable into a HIP graph.
    """
    T, E, K, S = _check(logits, ids, scoring, routed_scaling_factor, seq_starts)
    dev = logits.device
    if stream is not None or dev.index != _current_device():
        with on_stream(stream, dev):
            return router_losses(logits, ids, scoring=scoring, renormalize=renormalize,
                                 routed_scaling_factor=routed_scaling_factor,
                                 seq_starts=seq_starts)
    shape = (T, E, K, S, int(scoring == "sigmoid"), bool(renormalize),
             logits.dtype == torch.bfloat16, float(routed_scaling_factor))
    if torch.is_grad_enabled() and logits.requires_grad:
        return RouterLosses(*_Losses.apply(logits, ids, seq_starts, shape))
    return RouterLosses(*_forward(logits, ids, seq_starts, shape)[:5])


def _check(logits, ids, scoring, scale, seq_starts):
    """(T, E, K, S); raises ValueError for what the kernels do not take."""
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"unsupported scoring function {scoring!r}")
    if scoring == "softmax" and float(scale) != 1.0:
        raise ValueError("a scaling factor goes with sigmoid scoring")
    if not MIN_SCALE <= float(scale) <= MAX_SCALE:
        raise ValueError(f"routed_scaling_factor {scale} is not a positive fp32 number")
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits must be a 2-D fp32 or bf16 tensor, got {tuple(logits.shape)} "
                         f"{logits.dtype}")
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS or T > MAX_ROWS:
        raise ValueError(f"logits of {T} rows of {E} experts: 1 .. {MAX_EXPERTS} experts, at most "
                         f"{MAX_ROWS} rows")
    if _has_tangent(logits):
        raise ValueError("router_losses has no forward-mode derivative: logits carry a tangent")
    if logits.stride(1) != 1 and E > 1:
        raise ValueError(f"logits' rows must be contiguous (column stride {logits.stride(1)})")
    if ids.dim() != 2 or ids.dtype != torch.int32 or ids.shape[0] != T or not ids.is_contiguous():
        raise ValueError(f"ids must be contiguous int32 [{T}, K], got {tuple(ids.shape)} {ids.dtype}")
    K = ids.shape[1]
    if not 1 <= K <= MAX_TOP_K:
        raise ValueError(f"ids of {K} experts a row, 1 .. {MAX_TOP_K}")
    S = 1
    if seq_starts is not None:
        if seq_starts.dim() != 1 or seq_starts.dtype != torch.int32 \
                or not seq_starts.is_contiguous() or seq_starts.numel() < 2:
            raise ValueError(f"seq_starts must be contiguous int32 [S + 1], got "
                             f"{tuple(seq_starts.shape)} {seq_starts.dtype}")
        S = seq_starts.numel() - 1
        if S * -(-E // 16) >= MAX_PARTS:
            raise ValueError(f"{S} sequences of {E} experts: fewer than {MAX_PARTS} divided by the "
                             "sixteens of experts")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    _same_device(logits.device, ids=ids, seq_starts=seq_starts)
    return T, E, K, S


def _pack(logits, ids, starts, weights, stat, counts, probs, balance, z, norm, ws, nws, shape):
    T, E, K, S, mode, renorm, bf16, scale = shape
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    return ARGS.pack(logits.data_ptr(), ids.data_ptr(), ptr(starts), weights.data_ptr(),
                     stat.data_ptr(), counts.data_ptr(), ptr(probs), ptr(balance), ptr(z),
                     norm.data_ptr(), ptr(ws), logits.stride(0), nws, T, E, K, S, mode, renorm,
                     bf16, scale)


def _entries():
    global _ENTRIES
    if _ENTRIES is None:
        lib = _lib.load()
        _ENTRIES = lib.xtu_router_losses, lib.xtu_router_grad
    return _ENTRIES


def _forward(logits, ids, starts, shape):
    """(weights, balance, z, counts, probs, stat, norm)."""
    T, E, K, S, mode = shape[:5]
    new, f32 = logits.new_empty, torch.float32
    weights, stat = new((T, K), dtype=f32), new((T, 2), dtype=f32)
    norm, probs = new(2, dtype=f32), new((S, E), dtype=f32)
    balance, z = new((), dtype=f32), None if mode else new((), dtype=f32)
    counts = new((S, E), dtype=torch.int32)
    nws = _WS_BYTES.get((T, E, S))
    if nws is None:
        nws = int(_lib.call("xtu_router_workspace_bytes", T, E, S))
        if len(_WS_BYTES) >= 4096:   # a server's batch sizes
            _WS_BYTES.clear()
        _WS_BYTES[T, E, S] = nws
    # per call: calls on other streams, and graphs, have their own
    ws = new(nws, dtype=torch.uint8)
    rc = _entries()[0](_pack(logits, ids, starts, weights, stat, counts, probs, balance, z, norm,
                             ws, nws, shape), raw_stream(logits.device.index))
    if rc:
        _lib.check("xtu_router_losses", rc)
    return weights, balance, z, counts, probs, stat, norm


def _grad(ctx, g_weights, g_balance, g_z):
    logits, ids, starts, weights, counts = ctx.saved_tensors
    if _has_tangent(logits, g_weights, g_balance, g_z):
        raise RuntimeError("router_losses' gradient has no forward-mode derivative")
    out = logits.new_empty(logits.shape)
    grads = [None if g is None else g.contiguous() for g in (g_weights, g_balance, g_z)]
    rc = _entries()[1](_pack(logits, ids, starts, weights, ctx.stat, counts, None, None, None,
                             ctx.norm, None, 0, ctx.shape),
                       *[0 if g is None else g.data_ptr() for g in grads], out.data_ptr(),
                       raw_stream(logits.device.index))
    if rc:
        _lib.check("xtu_router_grad", rc)
    return out


class _Once(torch.autograd.Function):
    """The gradient as a node of its own, where a graph of it is asked for: a derivative
    of it is refused whatever it is asked through (it depends on the logits also where
    the outputs' gradients are constants)."""
    @staticmethod
    def forward(ctx, losses, logits, g_weights, g_balance, g_z):
        return _grad(losses, g_weights, g_balance, g_z)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("router_losses is once differentiable: its gradient has none")


class _Losses(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, starts, shape):
        weights, balance, z, counts, probs, ctx.stat, ctx.norm = _forward(logits, ids, starts,
                                                                          shape)
        ctx.save_for_backward(logits, ids, starts, weights, counts)
        ctx.shape = shape
        ctx.mark_non_differentiable(counts, probs)
        ctx.set_materialize_grads(False)
        return weights, balance, z, counts, probs

    @staticmethod
    def backward(ctx, g_weights, g_balance, g_z, _counts, _probs):
        if g_weights is None and g_balance is None and g_z is None:
            return None, None, None, None
        if torch.is_grad_enabled():   # create_graph
            d = _Once.apply(ctx, ctx.saved_tensors[0], g_weights, g_balance, g_z)
        else:
            d = _grad(ctx, g_weights, g_balance, g_z)
        return d, None, None, None
