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
import struct

import torch

from . import _lib
from .layer import _same_device, _stream

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "sigmoid": 5,
               "swiglu": 6}
# xtu_linear_args: x, w, bias, row_scale, residual, out, workspace; ldx, ldw, ldr,
# ldo, scale_stride, workspace_bytes; M, N, K, act, three bf16 flags; limit, alpha, beta
ARGS = struct.Struct("@7P5lN7i3f")
# workspace bytes per (M, N, K, swiglu, aligned)
_WS_BYTES: dict = {}
# what the kernels' 32-bit indices reach (xtu_linear refuses the same)
MAX_ROWS, MAX_COLS = (1 << 31) - 512, 1 << 28
_TYPES = (torch.bfloat16, torch.float32)
_OPERAND = (torch.bfloat16,)
_ENTRY = None


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
    shape, strides = t.shape, t.stride()
    if len(shape) != 2 or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a 2-D {' or '.join(str(d) for d in dtypes)} tensor, got "
                         f"{tuple(shape)} {t.dtype}")
    if cols is not None and shape[1] != cols:
        raise ValueError(f"{name} has {shape[1]} columns, expected {cols}")
    if strides[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}'s rows must be contiguous (column stride {strides[1]})")
    return strides[0]


def _entry():
    global _ENTRY
    if _ENTRY is None:
        _ENTRY = _lib.load().xtu_linear
    return _ENTRY


def raw_stream(index: int) -> int:
    """Handle of the current stream of device `index`."""
    return torch._C._cuda_getCurrentRawStream(index)


def _current_device() -> int:
    return torch._C._cuda_getDevice()


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

    x [M, K] and w [N, K] bf16, rows contiguous at any row stride; M may be 0
    (at most 2^31 - 512 rows, 2^28 columns of x and of the output).
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
    ldx = _rows("x", x, _OPERAND)
    M, K = x.shape
    ldw = _rows("w", w, _OPERAND, K)
    rows = w.shape[0]
    if rows == 0 or K == 0 or (act == 6 and rows % 2):
        raise ValueError(f"w of shape {tuple(w.shape)} does not fit activation {activation!r} "
                         "(at least one row and column; an even number of rows for swiglu)")
    N = rows // 2 if act == 6 else rows
    if M > MAX_ROWS:
        raise ValueError(f"x has {M} rows, at most {MAX_ROWS}")
    if N > MAX_COLS or K > MAX_COLS:
        raise ValueError(f"{N} output columns of {K} values, at most {MAX_COLS} columns of each")
    dev = x.device
    same = w.device == dev
    bp = sp = rp = sst = ldr = 0
    b16 = r16 = False
    if bias is not None:
        if bias.shape != (rows,) or bias.dtype not in _TYPES or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous bf16 or fp32 [{rows}], got "
                             f"{tuple(bias.shape)} {bias.dtype}")
        bp, b16 = bias.data_ptr(), bias.dtype == torch.bfloat16
        same = same and bias.device == dev
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.shape not in ((M,), (M, 1)):
            raise ValueError(f"row_scale must be fp32 [{M}] or [{M}, 1], got "
                             f"{tuple(row_scale.shape)} {row_scale.dtype}")
        sp, sst = row_scale.data_ptr(), row_scale.stride(0)
        same = same and row_scale.device == dev
    if residual is not None:
        ldr = _rows("residual", residual, _TYPES, N)
        if residual.shape[0] != M:
            raise ValueError(f"residual has {residual.shape[0]} rows, expected {M}")
        rp, r16 = residual.data_ptr(), residual.dtype == torch.bfloat16
        same = same and residual.device == dev
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
        same = same and out.device == dev
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if not same:
        _same_device(dev, w=w, bias=bias, row_scale=row_scale, residual=residual, out=out)
    if stream is not None or dev.index != _current_device():
        with on_stream(stream, dev):   # outputs belong to the stream that writes them
            return linear(x, w, bias=bias, activation=activation, row_scale=row_scale,
                          residual=residual, out=out, out_dtype=out_dtype,
                          swiglu_limit=swiglu_limit, swiglu_alpha=swiglu_alpha,
                          swiglu_beta=swiglu_beta)
    if out is None:
        out = x.new_empty((M, N), dtype=odt)
    if M == 0:
        return out
    xp, wp = x.data_ptr(), w.data_ptr()
    aligned = not ((ldx if M > 1 else 0) | ldw | K) & 7 and not (xp | wp) & 15
    nws = _WS_BYTES.get((M, N, K, act == 6, aligned))
    if nws is None:
        nws = int(_lib.call("xtu_linear_workspace_bytes", M, N, K, act, int(aligned)))
        if len(_WS_BYTES) >= 4096:   # a server's prompt lengths
            _WS_BYTES.clear()
        _WS_BYTES[M, N, K, act == 6, aligned] = nws
    # allocated per call: calls on other streams, and graphs, have their own
    ws = x.new_empty(nws, dtype=torch.uint8) if nws else None
    rc = _entry()(ARGS.pack(xp, wp, bp, sp, rp, out.data_ptr(), ws.data_ptr() if nws else 0, ldx,
                            ldw, ldr, ldo, sst, nws, M, N, K, act, b16, r16,
                            odt == torch.bfloat16, swiglu_limit or 0.0, swiglu_alpha, swiglu_beta),
                  raw_stream(dev.index))
    if rc:
        _lib.check("xtu_linear", rc)
    return out
