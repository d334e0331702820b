"""Timed cases of two operators beside the expert layer: the dense product
with its epilogue (``linear.linear``) and the MoE block from hidden states for
a few tokens (``block.MoeBlock``).

linear: y = residual + row_scale * act(x w^T + bias), bf16 operands; "swiglu"
takes w as [gate rows; up rows].  It is the router product (fp32 logits), an
unquantised shared expert's gate/up and down, and a plain projection.

block: router product, selection, routed and shared experts of a decode batch
of 1 to 16 tokens, in four weight formats.

The plain forms (``own`` false) are elementary torch operations in 32 bits;
router logits in 64, since the selection compares neighbouring scores.
"""
from __future__ import annotations

import os
import sys

import torch

own = False

DEV = "cuda"
STD = 0.02               # standard deviation of the weights
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "swiglu")
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# e2m1 codes of N(0, 1) draws in units of the group scale, as 256 equally
# likely ones: shares of |v| for a group maximum near 4.5 steps
CODE_SHARE = (30, 55, 47, 37, 51, 25, 9, 2)

SHAPES = {
    "ds": dict(E=256, shared=1, H=7168, I=2048, K=8, grouped=True, gated=False, limit=0.0),
    "qwen": dict(E=512, shared=1, H=2048, I=512, K=10, grouped=False, gated=True, limit=7.0),
    "e128": dict(E=128, shared=0, H=2048, I=768, K=8, grouped=False, gated=False, limit=0.0),
    "tiny": dict(E=8, shared=0, H=1024, I=2048, K=2, grouped=False, gated=False, limit=0.0),
}


def _linear(name, M, N, K, act="none", bias=False, scale=False, residual="none", out="bf16"):
    c = dict(op="linear", M=M, N=N, K=K, act=act, bias=bias, scale=scale, residual=residual,
             out=out)
    if name:
        c["name"] = name
    return c


def _block(name, shape, fmt, T):
    c = dict(op="block", shape=shape, fmt=fmt, T=T)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user's decode step: a small shared expert's gate/up (latency)
        _linear("shared-gate-up-m1", 1, 512, 2048, act="swiglu"),
        # router logits of a drafted run of tokens over 256 experts
        _linear("router-m4", 4, 256, 7168, out="f32"),
        # a ragged decode batch: the large shared expert's down, added to the routed sum
        _linear("shared-down-m47", 47, 7168, 2048, scale=True, residual="f32"),
        # odd sizes throughout: no row starts on 16 bytes
        _linear("odd-m1013", 1013, 771, 1187, act="gelu", bias=True, residual="bf16"),
        # router logits of a prompt over 512 experts
        _linear("router-m4096", 4096, 512, 2048, bias=True, out="f32"),
        # a prompt through the large shared expert's down, gated, added in bf16
        _linear("shared-down-m2048", 2048, 7168, 2048, scale=True, residual="bf16"),
        # a long prompt through the large shared expert's gate/up
        _linear("shared-gate-up-m8192", 8192, 2048, 7168, act="swiglu"),
        # one user's decode step over many small experts, gated shared expert
        _block("qwen-nvfp4-t1", "qwen", "nvfp4", 1),
        # two users of the large model
        _block("ds-mxfp4-t2", "ds", "mxfp4", 2),
        # its decode with drafted tokens
        _block("ds-mxfp4-t8", "ds", "mxfp4", 8),
        # an FP8 checkpoint, a few users
        _block("e128-fp8-t5", "e128", "fp8", 5),
        # unquantised experts, few of them
        _block("tiny-bf16-t3", "tiny", "bf16", 3),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    if rng.random() < 0.55:
        act = rng.choice(ACTS)
        M = _log(rng, 1, 8192)
        N = _log(rng, 8, 7168)
        K = _log(rng, 64, 7168)
        if rng.random() < 0.6:   # most widths are multiples of 64
            N, K = max(64, N // 64 * 64), K // 64 * 64
        if act == "swiglu":
            N = max(1, N // 2)
        while M * N * K * (2 if act == "swiglu" else 1) > 8192 * 2048 * 7168 * 2:
            M //= 2
        return _linear(None, M, N, K, act=act, bias=rng.random() < 0.5, scale=rng.random() < 0.4,
                       residual=rng.choice(("none", "bf16", "f32")),
                       out=rng.choice(("bf16", "bf16", "f32")))
    shape, fmt, hi = rng.choice([
        ("ds", "mxfp4", 8), ("ds", "fp8", 3), ("ds", "nvfp4", 6), ("qwen", "mxfp4", 16),
        ("qwen", "nvfp4", 16), ("e128", "fp8", 16), ("e128", "bf16", 16), ("tiny", "bf16", 16),
        ("tiny", "mxfp4", 16),
    ])
    return _block(None, shape, fmt, rng.randint(1, hi))


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(gen, shape, std, dtype=torch.bfloat16):
    return torch.empty(shape, device=DEV).normal_(0, std, generator=gen).to(dtype)


def _linear_inputs(case, seed):
    g = _generator(seed)
    M, N, K = case["M"], case["N"], case["K"]
    rows = 2 * N if case["act"] == "swiglu" else N
    st = dict(x=_normal(g, (M, K), 1.0), w=_normal(g, (rows, K), STD), bias=None, row_scale=None,
              residual=None)
    if case["bias"]:
        st["bias"] = _normal(g, (rows,), 0.5, torch.float32)
    if case["scale"]:   # a gate in (0, 1)
        st["row_scale"] = torch.sigmoid(_normal(g, (M,), 1.0, torch.float32))
    if case["residual"] != "none":
        st["residual"] = _normal(g, (M, N), 1.0,
                                 torch.float32 if case["residual"] == "f32" else torch.bfloat16)
    return st


def _codes(gen, n, N, K):
    """Packed e2m1 codes [n, N, K / 2], distributed as a quantised normal
    matrix's."""
    table = torch.repeat_interleave(torch.arange(8, dtype=torch.uint8, device=DEV),
                                    torch.tensor(CODE_SHARE, device=DEV))
    pairs = (table[:, None] | (table[None, :] << 4)).reshape(-1)
    out = torch.empty((n, N, K // 2), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 28) // (N * K // 2))
    for e0 in range(0, n, step):
        part = out[e0:e0 + step]
        r = torch.randint(0, 1 << 18, part.shape, generator=gen, device=DEV, dtype=torch.int32)
        part.copy_(pairs[(r & 0xffff)])
        part |= ((r >> 16) & 1).to(torch.uint8) << 3 | ((r >> 17) & 1).to(torch.uint8) << 7
    return out


def _bytes(gen, shape, lo, hi):
    return torch.randint(lo, hi + 1, shape, generator=gen, device=DEV, dtype=torch.uint8)


def _planes(fmt, gen, n, N, K, halves):
    """Checkpoint planes of n experts' [N, K] matrices of standard deviation
    near STD: (weights, scales, second-level scales)."""
    if fmt == "bf16":
        w = torch.empty((n, N, K), dtype=torch.bfloat16, device=DEV)
        return w.normal_(0, STD, generator=gen), None, None
    if fmt == "fp8":
        w = torch.empty((n, N, K), dtype=torch.float8_e4m3fn, device=DEV)
        for e in range(n):
            w[e] = torch.empty((N, K), device=DEV).normal_(0, 100.0, generator=gen) \
                .clamp_(-448, 448).to(torch.float8_e4m3fn)
        s = torch.empty((n, N // 128, K // 128), device=DEV).uniform_(0.8, 1.25, generator=gen)
        return w.view(torch.uint8), s * (STD / 100.0), None
    c = _codes(gen, n, N, K)
    if fmt == "mxfp4":   # group scales 2^-7 .. 2^-6
        return c, _bytes(gen, (n, N, K // 32), 120, 121), None
    # e4m3 bytes 2^5 .. 1.875 * 2^6 under a second-level scale
    s = _bytes(gen, (n, N, K // 16), 0x60, 0x6f)
    gs = torch.empty((n, 2) if halves else (n,), device=DEV).uniform_(1.0, 2.0, generator=gen)
    return c, s, gs * (0.008 / 64)


def _block_inputs(case, seed):
    s = SHAPES[case["shape"]]
    g = _generator(seed)
    E, H, I, n = s["E"], s["H"], s["I"], s["E"] + s["shared"]
    st = dict(x=_normal(g, (case["T"], H), 1.0), gate=_normal(g, (E, H), STD), bias=None,
              shared_gate=None)
    if s["grouped"]:
        st["bias"] = _normal(g, (E,), 0.02, torch.float32)
    if s["gated"]:
        st["shared_gate"] = _normal(g, (s["shared"], H), STD)
    st["w13"], st["s13"], st["g13"] = _planes(case["fmt"], g, n, 2 * I, H, True)
    st["w2"], st["s2"], st["g2"] = _planes(case["fmt"], g, n, H, I, False)
    return st


def prepare(case, seed):
    if case["op"] == "linear":
        return dict(case=case, **_linear_inputs(case, seed))
    st = dict(case=case, **_block_inputs(case, seed))
    if own:   # the handle a server builds once per layer: weights in the device layout
        st["block"] = _own_block(case, st)
    return st


def _own_block(case, st):
    _path()
    from xtu_moe_amd import formats as F
    from xtu_moe_amd.block import MoeBlock
    from xtu_moe_amd.layer import ExpertWeights

    s = SHAPES[case["shape"]]
    W = ExpertWeights.from_dense(F.fmt_of(case["fmt"]), st["w13"], st["s13"], st["w2"], st["s2"],
                                 st["g13"], st["g2"], n_shared=s["shared"])
    kw = dict(scoring="softmax")
    if s["grouped"]:
        kw = dict(scoring="sigmoid", bias=st["bias"], n_group=8, topk_group=4,
                  routed_scaling_factor=2.5)
    return MoeBlock(st["gate"], W, top_k=s["K"], shared_gate=st["shared_gate"],
                    swiglu_limit=s["limit"], **kw)


def _path():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                     "vllm-xtu-moe_amd")
    if p not in sys.path:
        sys.path.insert(0, p)


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "linear":
        return _plain_linear(case, state)
    return _plain_block(case, state)


def _run_own(case, st):
    if case["op"] == "block":
        out, wts, ids = st["block"](st["x"], return_routing=True)
        return {"out": out, "weights": wts, "ids": ids}
    return _own_linear()(st["x"], st["w"], bias=st["bias"], activation=case["act"],
                         row_scale=st["row_scale"], residual=st["residual"],
                         out_dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)


def _own_linear():
    _path()
    from xtu_moe_amd.linear import linear
    return linear


def _activate(act, z, limit=0.0):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
    if act == "swiglu":
        g, u = z.chunk(2, -1)
        if limit:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g / (1 + torch.exp(-g)) * u
    return z


def _plain_linear(case, st):
    z = st["x"].float() @ st["w"].float().t()
    if st["bias"] is not None:
        z = z + st["bias"]
    y = _activate(case["act"], z)
    if st["row_scale"] is not None:
        y = y * st["row_scale"][:, None]
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y if case["out"] == "f32" else y.to(torch.bfloat16)


def _largest(v, k):
    """Indices of the k largest along the last axis, in order; equal ones go
    to the lowest index."""
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[..., :k]


def _select(s, x, gate, bias):
    """(ids, weights) in 64 bits from the router product."""
    T, E, K = x.shape[0], s["E"], s["K"]
    lg = x.double() @ gate.double().t()
    if not s["grouped"]:
        ids = _largest(lg, K)
        w = torch.exp(lg.gather(1, ids) - lg.amax(1, keepdim=True))
        return ids, w / w.sum(1, keepdim=True)
    p = 1 / (1 + torch.exp(-lg))
    sel = p + bias.double()
    by = sel.view(T, 8, E // 8)
    best = _largest(by.gather(2, _largest(by, 2)).sum(2), 4)
    keep = torch.zeros((T, 8), dtype=torch.bool, device=lg.device).scatter_(1, best, True)
    ids = _largest(sel.masked_fill(~keep.repeat_interleave(E // 8, 1), -float("inf")), K)
    w = p.gather(1, ids)
    return ids, w / w.sum(1, keepdim=True) * 2.5


def _pairs(s, st):
    """Every token's experts and weights, the shared ones behind the routed."""
    x = st["x"]
    ids, wts = _select(s, x, st["gate"], st["bias"])
    all_ids, all_w = ids, wts
    if s["shared"]:
        sh = s["E"] + torch.arange(s["shared"], device=x.device)
        all_ids = torch.cat([ids, sh.expand(x.shape[0], -1)], 1)
        gate = torch.ones((x.shape[0], s["shared"]), dtype=torch.float64, device=x.device)
        if st["shared_gate"] is not None:
            gate = 1 / (1 + torch.exp(-(x.double() @ st["shared_gate"].double().t())))
        all_w = torch.cat([wts, gate], 1)
    return ids.to(torch.int32), wts, all_ids, all_w


def _dequantize(fmt, q, s, gs):
    """Checkpoint planes of some experts as float32 values [n, N, K]."""
    if fmt == "bf16":
        return q.float()
    n, N = q.shape[0], q.shape[1]
    if fmt == "fp8":
        v = q.view(torch.float8_e4m3fn).float().view(n, N // 128, 128, -1, 128)
        return (v * s[:, :, None, :, None]).view(n, N, -1)
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    v = torch.stack([lut[(q & 15).int()], lut[(q >> 4).int()]], -1).view(n, N, -1)
    if fmt == "mxfp4":
        sc = torch.exp2(s.float() - 127)
    else:
        gs = gs.view(n, -1)
        sc = s.view(torch.float8_e4m3fn).float().view(n, gs.shape[1], -1) * gs[:, :, None]
        sc = sc.view(n, N, -1)
    return (v.view(n, N, sc.shape[2], -1) * sc[..., None]).view(n, N, -1)


def _of(st, which, e):
    pick = lambda t: None if t is None else t[e]  # noqa: E731
    return pick(st["w" + which]), pick(st["s" + which]), pick(st["g" + which])


def _plain_block(case, st):
    s, fmt = SHAPES[case["shape"]], case["fmt"]
    ids, wts, all_ids, all_w = _pairs(s, st)
    T, P = all_ids.shape
    e = all_ids.reshape(-1)
    x = st["x"].float().repeat_interleave(P, 0)
    z = (_dequantize(fmt, *_of(st, "13", e)) @ x[:, :, None])[..., 0]
    a = _activate("swiglu", z, s["limit"])
    y = (_dequantize(fmt, *_of(st, "2", e)) @ a[:, :, None])[..., 0]
    out = (y.view(T, P, -1) * all_w.float()[:, :, None]).sum(1)
    return {"out": out.to(torch.bfloat16), "weights": wts.float(), "ids": ids}


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        rows = 2 * N if case["act"] == "swiglu" else N
        nbytes = 2 * (M * K + rows * K) + M * N * (4 if case["out"] == "f32" else 2)
        nbytes += 4 * rows * case["bias"] + 4 * M * case["scale"]
        nbytes += M * N * {"none": 0, "bf16": 2, "f32": 4}[case["residual"]]
        return {"bytes": float(nbytes), "flops": 2.0 * M * rows * K}
    # every active expert's planes once: the expected number of distinct
    # experts of T uniform choices of K
    s = SHAPES[case["shape"]]
    T, E, H, I, K = case["T"], s["E"], s["H"], s["I"], s["K"]
    n = E * (1.0 - (1.0 - K / E) ** T) + s["shared"]
    bits = {"mxfp4": 4 + 8 / 32, "nvfp4": 4 + 8 / 16, "fp8": 8 + 32 / 16384, "bf16": 16}
    nbytes = n * 3 * H * I * bits[case["fmt"]] / 8 + 2 * E * H + T * (4 * H + 8 * K)
    return {"bytes": nbytes, "flops": 2.0 * T * (3 * H * I * (K + s["shared"]) + E * H)}


# ------------------------------------------------------------------ exact
def _exact_linear(case, st):
    x, w = st["x"].double(), st["w"].double()
    y = torch.empty((case["M"], case["N"]), dtype=torch.float64, device=x.device)
    for r in range(0, case["M"], 1024):   # rows at a time
        z = x[r:r + 1024] @ w.t()
        if st["bias"] is not None:
            z += st["bias"].double()
        if case["act"] == "swiglu":
            g, u = z[:, :case["N"]], z[:, case["N"]:]
            z = g * torch.sigmoid(g) * u
        elif case["act"] in ("gelu", "gelu_tanh"):
            z = torch.nn.functional.gelu(z, approximate="tanh" if "tanh" in case["act"] else "none")
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] == "sigmoid":
            z = torch.sigmoid(z)
        elif case["act"] == "relu":
            z = z.clamp(min=0)
        y[r:r + 1024] = z
    if st["row_scale"] is not None:
        y *= st["row_scale"].double()[:, None]
    if st["residual"] is not None:
        y += st["residual"].double()
    return y


def _e4m3_values(b):
    """e4m3 bytes as float64: (1 + m / 8) 2^(e - 7), or m 2^-9 for e = 0."""
    e, m = (b >> 3 & 15).double(), (b & 7).double()
    v = torch.where(e > 0, torch.exp2(e - 7) * (1 + m / 8), m * 2.0 ** -9)
    return torch.where(b >> 7 > 0, -v, v)


def _expert_values(fmt, st, which, e):
    """One expert's matrix as float64 [N, K]."""
    q = st["w" + which][e]
    if fmt == "bf16":
        return q.double()
    s = st["s" + which][e]
    if fmt == "fp8":
        grid = s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        return _e4m3_values(q) * grid
    nib = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.uint8, device=q.device)
    nib[:, 0::2], nib[:, 1::2] = q & 15, q >> 4
    ex, m = (nib >> 1 & 3).double(), (nib & 1).double()
    v = torch.where(ex > 0, torch.exp2(ex - 1) * (1 + m / 2), m / 2)
    v = torch.where(nib > 7, -v, v)
    if fmt == "mxfp4":
        return v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    v *= _e4m3_values(s).repeat_interleave(16, 1)
    gs = st["g" + which][e].double().reshape(-1)
    return v * gs.repeat_interleave(v.shape[0] // gs.numel())[:, None]


def exact(case, seed):
    if case["op"] == "linear":
        return _exact_linear(case, _linear_inputs(case, seed))
    s, fmt, st = SHAPES[case["shape"]], case["fmt"], _block_inputs(case, seed)
    x, E, I, K = st["x"].double(), s["E"], s["I"], s["K"]
    lg = x @ st["gate"].double().t()
    if s["grouped"]:
        p = torch.sigmoid(lg)
        sel = p + st["bias"].double()
        best = sel.view(len(x), 8, -1).topk(2, 2).values.sum(2).topk(4, 1).indices
        keep = torch.zeros((len(x), 8), dtype=torch.bool, device=DEV).scatter_(1, best, True)
        ids = sel.masked_fill(~keep.repeat_interleave(E // 8, 1), -1e9).topk(K, 1).indices
        wts = p.gather(1, ids)
        wts = wts / wts.sum(1, keepdim=True) * 2.5
    else:
        wts, ids = torch.softmax(lg, 1).topk(K, 1)
        wts = wts / wts.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in torch.unique(ids).tolist() + list(range(E, E + s["shared"])):
        if e < E:
            tok, k = (ids == e).nonzero(as_tuple=True)
            w = wts[tok, k]
        else:
            tok = torch.arange(len(x), device=DEV)
            w = torch.ones(len(x), dtype=torch.float64, device=DEV)
            if st["shared_gate"] is not None:
                w = torch.sigmoid(x @ st["shared_gate"][e - E].double())
        gu = x[tok] @ _expert_values(fmt, st, "13", e).t()
        g, u = gu[:, :I], gu[:, I:]
        if s["limit"]:
            g, u = g.clamp(max=s["limit"]), u.clamp(-s["limit"], s["limit"])
        act = g * torch.sigmoid(g) * u
        y = act @ _expert_values(fmt, st, "2", e).t()
        out.index_add_(0, tok, y * w[:, None])
    return {"out": out, "weights": wts, "ids": ids.to(torch.int32)}
