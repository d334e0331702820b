"""The dense product with a fused epilogue, for what surrounds the experts.

    y = residual + row_scale * act(x @ w.T + bias)

The reference leaves these products to its host (vllm_xiaotu_moe/
hybrid_model.py:1752 ``_shared_out`` for the shared expert, :1877 for the
router); here they are one launch of the HIP library each: the router product
(``out_dtype=torch.float32``), an unquantised shared expert's gate/up
(``activation="swiglu"``) and down (``row_scale`` = its gate, ``residual`` =
the routed experts' sum), or any projection.
"""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from .layer import _p, _same_device, _stream

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "sigmoid": 5,
               "swiglu": 6}
# workspace bytes per (M, N, K, swiglu, aligned)
_WS_BYTES: dict = {}
_TYPES = (torch.bfloat16, torch.float32)


def _extent(t):
    """[first, last) byte addresses that t's elements lie in."""
    if t.numel() == 0:
        return 0, 0
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _overlap(a, b) -> bool:
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 < b1 and b0 < a1


def _rows(name, t, dtypes, cols=None):
    """A matrix whose rows are contiguous; returns its row stride."""
    if t.dim() != 2 or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a 2-D {' or '.join(str(d) for d in dtypes)} tensor, got "
                         f"{tuple(t.shape)} {t.dtype}")
    if cols is not None and t.shape[1] != cols:
        raise ValueError(f"{name} has {t.shape[1]} columns, expected {cols}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous (column stride {t.stride(1)})")
    return t.stride(0)


@contextlib.contextmanager
def on_stream(stream, dev):
    """Device `dev` current, and `stream` (a torch stream, a raw handle or
    None) the stream that work and allocations go to."""
    with torch.cuda.device(dev):
        if stream is None:
            yield
            return
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(_stream(stream), device=dev)
        with torch.cuda.stream(stream):
            yield


def linear(x, w, *, bias=None, activation="none", row_scale=None, residual=None, out=None,
           out_dtype=None, swiglu_limit=0.0, swiglu_alpha=1.0, swiglu_beta=0.0, stream=None):
    """residual + row_scale * act(x @ w.T + bias); returns [M, N].

    x [M, K] and w [N, K] bf16, rows contiguous at any row stride; M may be 0.
    activation: "none", "relu", "silu", "gelu" (erf), "gelu_tanh", "sigmoid",
    or "swiglu" (w and bias hold 2N rows, gate rows then up rows; the clamped
    gated SiLU of the experts with swiglu_*).  bias [N] (swiglu [2N]) and
    residual [M, N] bf16 or fp32; row_scale fp32 [M] or [M, 1], multiplied
    after the activation.  out: bf16 (default) or fp32 per out_dtype, or the
    given tensor, which may be ``residual`` itself and otherwise overlaps no
    input.  fp32 sums and epilogue, rounded once.  Capturable into a HIP graph.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
    ldx = _rows("x", x, (torch.bfloat16,))
    M, K = x.shape
    ldw = _rows("w", w, (torch.bfloat16,), K)
    rows = w.shape[0]
    if rows == 0 or K == 0 or (act == 6 and rows % 2):
        raise ValueError(f"w of shape {tuple(w.shape)} does not fit activation {activation!r} "
                         "(at least one row and column; an even number of rows for swiglu)")
    N = rows // 2 if act == 6 else rows
    if bias is not None and (tuple(bias.shape) != (rows,) or bias.dtype not in _TYPES
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous bf16 or fp32 [{rows}], got "
                         f"{tuple(bias.shape)} {bias.dtype}")
    sst = 0
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or tuple(row_scale.shape) not in ((M,), (M, 1)):
            raise ValueError(f"row_scale must be fp32 [{M}] or [{M}, 1], got "
                             f"{tuple(row_scale.shape)} {row_scale.dtype}")
        sst = row_scale.stride(0)
    ldr = 0
    if residual is not None:
        ldr = _rows("residual", residual, _TYPES, N)
        if residual.shape[0] != M:
            raise ValueError(f"residual has {residual.shape[0]} rows, expected {M}")
    odt = out.dtype if out is not None else out_dtype or torch.bfloat16
    if odt not in _TYPES or (out_dtype or odt) != odt:
        raise ValueError(f"output type {odt} (out_dtype {out_dtype}): bf16 or fp32")
    ldo = N
    if out is not None:
        ldo = _rows("out", out, _TYPES, N)
        if out.shape[0] != M or (M > 1 and ldo < N):
            raise ValueError(f"out {tuple(out.shape)} with row stride {ldo} does not hold "
                             f"[{M}, {N}]")
        for name, t in (("x", x), ("w", w), ("bias", bias), ("row_scale", row_scale),
                        ("residual", residual)):
            if t is None or not _overlap(out, t):
                continue
            if name == "residual" and t.data_ptr() == out.data_ptr() and t.dtype == out.dtype \
                    and (ldr == ldo or M == 1):
                continue   # in place: every element is read before it is written
            raise ValueError(f"out overlaps {name}")
    dev = x.device
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    _same_device(dev, w=w, bias=bias, row_scale=row_scale, residual=residual, out=out)
    if stream is not None or dev.index != torch.cuda.current_device():
        with on_stream(stream, dev):   # outputs belong to the stream that writes them
            return linear(x, w, bias=bias, activation=activation, row_scale=row_scale,
                          residual=residual, out=out, out_dtype=out_dtype,
                          swiglu_limit=swiglu_limit, swiglu_alpha=swiglu_alpha,
                          swiglu_beta=swiglu_beta)
    if out is None:
        out = torch.empty((M, N), dtype=odt, device=dev)
    if M == 0:
        return out
    xp, wp = x.data_ptr(), w.data_ptr()
    aligned = not ((ldx if M > 1 else 0) | ldw | K) & 7 and not (xp | wp) & 15
    key = (M, N, K, act == 6, aligned)
    nws = _WS_BYTES.get(key)
    if nws is None:
        nws = _WS_BYTES[key] = int(_lib.call("xtu_linear_workspace_bytes", M, N, K, act,
                                             int(aligned)))
    # allocated per call: calls on other streams, and graphs, have their own
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.call("xtu_linear", xp, ldx, wp, ldw, M, N, K, act, _p(bias),
              int(bias is not None and bias.dtype == torch.bfloat16), _p(row_scale), sst,
              _p(residual), int(residual is not None and residual.dtype == torch.bfloat16), ldr,
              out.data_ptr(), int(odt == torch.bfloat16), ldo, float(swiglu_limit or 0.0),
              float(swiglu_alpha), float(swiglu_beta), _p(ws), nws, _stream())
    return out
