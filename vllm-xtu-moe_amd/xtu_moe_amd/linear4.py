"""The dense product with 4-bit weights and group scales.

    y = residual + row_scale * act(x @ w.T + bias),  w in MXFP4, NVFP4 or INT4

``linear.linear`` for the matrices that a quantised checkpoint keeps in its
experts' formats: a shared expert beside the routed ones, a dense layer, a
projection.  The weights are packed once (``Weight4.from_dense``); the arguments
and the epilogue are ``linear``'s.  The reference leaves these products to its
host (vllm_xiaotu_moe/hybrid_model.py:1752 ``_shared_out``), and INT4 to its CPU
engine (xiaotu_moe/csrc/moe/moe_v2_packed4_base.inc:4-16).
"""
from __future__ import annotations

import struct
from dataclasses import dataclass, replace
from typing import Optional

import torch

from . import _lib
from .formats import (FMT_INT4, FMT_MXFP4, FMT_NAMES, FMT_NVFP4, fmt_of, linear4_group,
                      linear4_record, pack_linear4)
from .layer import _has_tangent, _same_device
from .linear import (_OPERAND, _TYPES, ACTIVATIONS, MAX_COLS, MAX_ROWS, _current_device, _overlap,
                     _rows, on_stream, raw_stream)

# xtu_linear4_args: x, w, gs, bias, row_scale, residual, out, workspace; ldx, ldr,
# ldo, scale_stride, workspace_bytes; M, N, K, act, fmt, group, three bf16 flags;
# limit, alpha, beta
ARGS = struct.Struct("@8P4lN9i3f")
MAX_E8M0 = 252   # 6 * 2^(252 - 127) is the largest weight that bf16 holds
_WS_BYTES: dict = {}
_ENTRY = None


@dataclass(frozen=True, eq=False)
class Weight4:
    """One matrix [N, K] (gated: gate rows [N, K], then up rows [N, K]) in the
    kernels' layout: ``data`` u8 records, ``gs`` fp32 [1] or [2] (NVFP4; else
    None).  Made by ``from_dense``; its fields do not change."""
    fmt: int
    N: int
    K: int
    group: int
    gated: bool
    data: torch.Tensor
    gs: Optional[torch.Tensor]

    def __post_init__(self):
        halves = 2 if self.gated else 1
        need = (halves * -(-self.N // 16), -(-self.K // 128), linear4_record(self.fmt, self.group))
        d, gs = self.data, self.gs
        if d.dtype != torch.uint8 or tuple(d.shape) != need or not d.is_contiguous() \
                or d.data_ptr() % 16:
            raise ValueError(f"records must be contiguous u8 {need} on 16 bytes, got "
                             f"{tuple(d.shape)} {d.dtype}")
        if (gs is not None) != (self.fmt == FMT_NVFP4) or gs is not None and (
                gs.dtype != torch.float32 or gs.shape != (halves,) or gs.device != d.device
                or not gs.is_contiguous() or gs.requires_grad):
            raise ValueError(f"second-level scales must be fp32 [{halves}] beside NVFP4 records, "
                             "without a gradient")

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self):
        return self.data.numel()

    def to(self, device):
        """The same matrix on another device."""
        return replace(self, data=self.data.to(device),
                       gs=None if self.gs is None else self.gs.to(device))

    @classmethod
    def from_dense(cls, fmt, codes, scales, global_scale=None, *, gated=False, device=None):
        """Packs a checkpoint's tensors.

        fmt: "mxfp4", "nvfp4" or "int4" (or its number in ``formats``).  codes
        u8 [rows, K / 2], low nibble = even k.  scales, as bytes or as torch's
        type of them: MXFP4 e8m0 [rows, K / 32] (at most 252: larger ones leave
        bf16's range; 255 is NaN); NVFP4 e4m3 (no NaN) [rows, K / 16]; INT4 finite
        fp32, fp16 or bf16 [rows, K / 32, 64 or 128], for value code - 8.
        global_scale: NVFP4's second-level scale, a finite number or a tensor of one
        (gated: one or two, gate and up).  gated: rows are [gate; up], for
        activation "swiglu".  Reads the scales back once to check them.  The
        result is a constant: parameters are packed as they are now, detached.
        """
        fmt = fmt_of(fmt)
        if fmt not in (FMT_MXFP4, FMT_NVFP4, FMT_INT4):
            raise ValueError(f"4-bit weights are mxfp4, nvfp4 or int4, not {FMT_NAMES[fmt]}")
        if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.numel() == 0:
            raise ValueError(f"codes must be u8 [rows, K / 2], got {tuple(codes.shape)} {codes.dtype}")
        rows, K = codes.shape[0], codes.shape[1] * 2
        halves = 2 if gated else 1
        if rows % halves:
            raise ValueError(f"gated weights of {rows} rows: gate and up rows in equal number")
        if rows // halves > MAX_COLS or K > MAX_COLS:
            raise ValueError(f"weights of {rows} rows of {K} values, at most {MAX_COLS} of each")
        if scales.dim() != 2 or scales.shape[0] != rows:
            raise ValueError(f"scales must be [{rows}, K / group], got {tuple(scales.shape)}")
        scales = scales.detach()
        group = linear4_group(fmt, scales, K)
        if fmt == FMT_INT4:
            if scales.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise ValueError(f"INT4 scales must be fp32, fp16 or bf16, got {scales.dtype}")
            if not bool((scales.abs().float() < 2.0 ** 123).all()):
                raise ValueError("INT4 scales must be finite (below 2^123)")
        else:
            own = torch.float8_e4m3fn if fmt == FMT_NVFP4 else torch.float8_e8m0fnu
            if scales.dtype not in (torch.uint8, own):
                raise ValueError(f"{FMT_NAMES[fmt]} scales must be bytes, got {scales.dtype}")
            b = scales = scales.contiguous().view(torch.uint8)
            if fmt == FMT_MXFP4 and bool((b > MAX_E8M0).any()):
                raise ValueError(f"e8m0 scales above {MAX_E8M0} leave bf16's range")
            if fmt == FMT_NVFP4 and bool(((b & 0x7f) == 0x7f).any()):
                raise ValueError("e4m3 scales must not be NaN")
        dev = torch.device(device) if device is not None else codes.device
        gs = None
        if fmt == FMT_NVFP4:
            if global_scale is None:
                raise ValueError("NVFP4 weights need their second-level scale")
            gs = torch.as_tensor(global_scale, dtype=torch.float32).detach().reshape(-1).to(dev)
            if gs.numel() not in (1, halves):
                raise ValueError(f"second-level scales: {gs.numel()}, expected 1"
                                 + (" or 2 (gate, up)" if gated else ""))
            if not bool(gs.isfinite().all()):
                raise ValueError("second-level scales must be finite")
            gs = gs.expand(halves).clone(memory_format=torch.contiguous_format)   # its own
        elif global_scale is not None:
            raise ValueError(f"{FMT_NAMES[fmt]} weights have no second-level scale")
        split = lambda t: t.to(dev).contiguous().view(halves, rows // halves, -1)  # noqa: E731
        data = pack_linear4(fmt, split(codes), split(scales), group)
        return cls(fmt, rows // halves, K, group, bool(gated), data, gs)


def _entry():
    global _ENTRY
    if _ENTRY is None:
        _ENTRY = _lib.load().xtu_linear4
    return _ENTRY


def linear4(x, w: Weight4, *, bias=None, activation="none", row_scale=None, residual=None,
            out=None, out_dtype=None, swiglu_limit=0.0, swiglu_alpha=1.0, swiglu_beta=0.0,
            stream=None):
    """residual + row_scale * act(x @ w.T + bias); returns [M, N].

    x [M, K] bf16, rows contiguous at any row stride and alignment; M may be 0.
    w: a Weight4, gated with activation "swiglu" and only then.  The other
    arguments are ``linear``'s: activation "none", "relu", "silu", "gelu",
    "gelu_tanh", "sigmoid" or "swiglu"; bias [N] (swiglu [2N]: gate, up) and
    residual [M, N] bf16 or fp32; row_scale fp32 [M] or [M, 1]; out bf16 (default)
    or fp32 per out_dtype, or the given tensor, which may be ``residual`` itself
    and otherwise overlaps no input.  Weights enter the fp32 sums exactly;
    the epilogue is fp32, rounded once.  Capturable into a HIP graph.  No
    backward: inputs that require a gradient, or carry a forward-mode tangent,
    are refused.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
    if not isinstance(w, Weight4):
        raise ValueError(f"w must be a Weight4, got {type(w).__name__}")
    if w.gated != (act == 6):
        raise ValueError("gated weights go with activation 'swiglu', and only they")
    N, K = w.N, w.K
    ldx = _rows("x", x, _OPERAND, K)
    M = x.shape[0]
    if M > MAX_ROWS:
        raise ValueError(f"x has {M} rows, at most {MAX_ROWS}")
    dev = x.device
    same = w.data.device == dev
    rows = 2 * N if w.gated else N
    grad = x.requires_grad
    bp = sp = rp = sst = ldr = 0
    b16 = r16 = False
    if bias is not None:
        if bias.shape != (rows,) or bias.dtype not in _TYPES or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous bf16 or fp32 [{rows}], got "
                             f"{tuple(bias.shape)} {bias.dtype}")
        bp, b16 = bias.data_ptr(), bias.dtype == torch.bfloat16
        same, grad = same and bias.device == dev, grad or bias.requires_grad
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.shape not in ((M,), (M, 1)):
            raise ValueError(f"row_scale must be fp32 [{M}] or [{M}, 1], got "
                             f"{tuple(row_scale.shape)} {row_scale.dtype}")
        sp, sst = row_scale.data_ptr(), row_scale.stride(0)
        same, grad = same and row_scale.device == dev, grad or row_scale.requires_grad
    if residual is not None:
        ldr = _rows("residual", residual, _TYPES, N)
        if residual.shape[0] != M:
            raise ValueError(f"residual has {residual.shape[0]} rows, expected {M}")
        rp, r16 = residual.data_ptr(), residual.dtype == torch.bfloat16
        same, grad = same and residual.device == dev, grad or residual.requires_grad
    odt = out.dtype if out is not None else out_dtype or torch.bfloat16
    if odt not in _TYPES or (out_dtype or odt) != odt:
        raise ValueError(f"output type {odt} (out_dtype {out_dtype}): bf16 or fp32")
    ldo = N
    if out is not None:
        ldo = _rows("out", out, _TYPES, N)
        if out.shape[0] != M or (M > 1 and ldo < N):
            raise ValueError(f"out {tuple(out.shape)} with row stride {ldo} does not hold "
                             f"[{M}, {N}]")
        for name, t in (("x", x), ("w", w.data), ("w's scale", w.gs), ("bias", bias),
                        ("row_scale", row_scale), ("residual", residual)):
            if t is None or not _overlap(out, t):
                continue
            if name == "residual" and t.data_ptr() == out.data_ptr() and t.dtype == out.dtype \
                    and (ldr == ldo or M == 1):
                continue   # in place: every element is read before it is written
            raise ValueError(f"out overlaps {name}")
        same, grad = same and out.device == dev, grad or out.requires_grad
    if grad and torch.is_grad_enabled():
        raise ValueError("linear4 has no backward: an input requires a gradient")
    if _has_tangent(x, bias, row_scale, residual, out):
        raise ValueError("linear4 has no forward-mode derivative: an input carries a tangent")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if not same:
        _same_device(dev, w=w.data, bias=bias, row_scale=row_scale, residual=residual, out=out)
    if stream is not None or dev.index != _current_device():
        with on_stream(stream, dev):   # outputs belong to the stream that writes them
            return linear4(x, w, bias=bias, activation=activation, row_scale=row_scale,
                           residual=residual, out=out, out_dtype=out_dtype,
                           swiglu_limit=swiglu_limit, swiglu_alpha=swiglu_alpha,
                           swiglu_beta=swiglu_beta)
    if out is None:
        out = x.new_empty((M, N), dtype=odt)
    if M == 0:
        return out
    xp = x.data_ptr()
    aligned = not (xp & 15 or (M > 1 and ldx & 7))
    key = (M, N, K, act == 6, w.fmt, w.group, aligned)
    nws = _WS_BYTES.get(key)
    if nws is None:
        nws = int(_lib.call("xtu_linear4_workspace_bytes", M, N, K, act, w.fmt, w.group,
                            int(aligned)))
        if len(_WS_BYTES) >= 4096:   # a server's prompt lengths
            _WS_BYTES.clear()
        _WS_BYTES[key] = nws
    # allocated per call: calls on other streams, and graphs, have their own
    ws = x.new_empty(nws, dtype=torch.uint8) if nws else None
    rc = _entry()(ARGS.pack(xp, w.data.data_ptr(), 0 if w.gs is None else w.gs.data_ptr(),
                            bp, sp, rp, out.data_ptr(), ws.data_ptr() if nws else 0, ldx, ldr, ldo,
                            sst, nws, M, N, K, act, w.fmt, w.group, b16, r16,
                            odt == torch.bfloat16, swiglu_limit or 0.0, swiglu_alpha, swiglu_beta),
                  raw_stream(dev.index))
    if rc:
        _lib.check("xtu_linear4", rc)
    return out
