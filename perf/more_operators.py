"""Timed cases of two more operators beside the expert layer: the dense
product with 4-bit weights and group scales (``linear4.linear4``) and the
router's losses, per-expert counts and weights with their gradient
(``router.router_losses``).

linear4: y = residual + row_scale * act(x w^T + bias), bf16 x, w in MXFP4
(e2m1, e8m0 per 32 k), NVFP4 (e2m1, e4m3 per 16 k, second-level scale) or INT4
(code - 8, fp32 scale per 32, 64 or 128 k); "swiglu" takes w as [gate rows; up
rows].

router: of logits [T, E] and the selected ids [T, K] (-1: no expert), one
training step: the selected experts' weights, balance loss, z-loss (softmax),
per-sequence counts and mean probabilities, and the logits' gradient.  Rows
behind the last sequence belong to no sequence.

The plain forms (``own`` false) are elementary torch operations in 32 bits
(sums over tokens in 64).
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
# codes of N(0, 1) draws in units of the group scale, as 256 equally likely
# ones: shares of |v| for a group maximum near 4.5 steps (e2m1), and of
# code - 8 from -8 on for one near 7 (int4)
E2M1_SHARE = (30, 55, 47, 37, 51, 25, 9, 2)
INT4_SHARE = (1, 3, 6, 10, 16, 24, 30, 25, 26, 25, 30, 24, 16, 10, 7, 3)


def _linear(name, fmt, M, N, K, act="none", bias=False, scale=False, residual="none", out="bf16",
            group=0):
    c = dict(op="linear4", fmt=fmt, M=M, N=N, K=K, act=act, bias=bias, scale=scale,
             residual=residual, out=out, group=group)
    if name:
        c["name"] = name
    return c


def _router(name, T, E, K, scoring="softmax", renormalize=True, scale=1.0, sequences=1, pad=0,
            dtype="f32", dropped=False):
    c = dict(op="router", T=T, E=E, K=K, scoring=scoring, renormalize=renormalize, scale=scale,
             sequences=sequences, pad=pad, dtype=dtype, dropped=dropped)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user's decode step: a small shared expert's gate/up (latency)
        _linear("shared-gate-up-m1", "mxfp4", 1, 512, 2048, act="swiglu"),
        # one user, a wide dense layer's gate/up (all bandwidth)
        _linear("wide-gate-up-m1", "mxfp4", 1, 16384, 7168, act="swiglu"),
        # an INT4 checkpoint's projection for a few users, added to the stream
        _linear("projection-int4-m3", "int4", 3, 7168, 2048, residual="bf16", group=128),
        # odd row counts, the finest INT4 groups
        _linear("odd-int4-m7", "int4", 7, 1171, 1184, act="gelu", bias=True, out="f32", group=32),
        # a decode batch through a square projection
        _linear("projection-nvfp4-m16", "nvfp4", 16, 7168, 7168),
        # a ragged decode batch: the large shared expert's down, added to the routed sum
        _linear("shared-down-m47", "nvfp4", 47, 7168, 2048, scale=True, residual="f32"),
        # a prompt through the large shared expert's gate/up
        _linear("shared-gate-up-m2048", "mxfp4", 2048, 2048, 7168, act="swiglu"),
        # a small step over 8 experts
        _router("e8-t128", 128, 8, 2),
        # odd expert count, tokens dropped by capacity, weights as they are
        _router("e60-t1013", 1013, 60, 4, renormalize=False, dropped=True),
        # packed sequences of one micro-batch in bf16 logits, padding behind the last
        _router("packed-e128-t5003", 5003, 128, 8, sequences=17, pad=211, dtype="bf16"),
        # the large model's sigmoid router, a long prompt
        _router("sigmoid-e256-t8192", 8192, 256, 8, scoring="sigmoid", scale=2.5, sequences=2),
        # many small experts, a large micro-batch (all bandwidth)
        _router("e512-t32768", 32768, 512, 10),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    if rng.random() < 0.6:
        fmt = rng.choice(("mxfp4", "nvfp4", "int4"))
        act = rng.choice(ACTS)
        group = rng.choice((32, 64, 128)) if fmt == "int4" else 0
        M = _log(rng, 1, 2048) if rng.random() < 0.4 else _log(rng, 1, 64)
        N = _log(rng, 8, 16384)
        step = group or {"mxfp4": 32, "nvfp4": 16}[fmt]
        K = max(step, _log(rng, 64, 8192) // step * step)
        if rng.random() < 0.6:   # most row counts are multiples of 64
            N = max(64, N // 64 * 64)
        if act == "swiglu":
            N = max(1, N // 2)
        gated = 2 if act == "swiglu" else 1
        while M * N * K * gated > 2048 * 2048 * 7168 * 2 or N * K * gated > 2 * 16384 * 7168:
            M, N = max(1, M // 2), N if M > 1 else N // 2
        return _linear(None, fmt, M, N, K, act=act, bias=rng.random() < 0.5,
                       scale=rng.random() < 0.4, residual=rng.choice(("none", "bf16", "f32")),
                       out=rng.choice(("bf16", "bf16", "f32")), group=group)
    E = rng.choice((8, 16, 32, 60, 64, 72, 128, 160, 256, 384, 512))
    T = _log(rng, 1, 32768)
    scoring = rng.choice(("softmax", "sigmoid"))
    return _router(None, T, E, rng.randint(1, min(10, E)), scoring=scoring,
                   renormalize=rng.random() < 0.7,
                   scale=2.5 if scoring == "sigmoid" and rng.random() < 0.5 else 1.0,
                   sequences=min(T, _log(rng, 1, 64)), pad=rng.choice((0, 0, T // 10)),
                   dtype=rng.choice(("f32", "f32", "bf16")), dropped=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(gen, shape, std, dtype=torch.bfloat16):
    return torch.empty(shape, device=DEV).normal_(0, std, generator=gen).to(dtype)


def _codes(gen, N, K, fmt):
    """Packed codes [N, K / 2] (low nibble = even k), distributed as a
    quantised normal matrix's."""
    share = INT4_SHARE if fmt == "int4" else E2M1_SHARE
    table = torch.repeat_interleave(torch.arange(len(share), dtype=torch.uint8, device=DEV),
                                    torch.tensor(share, device=DEV))
    pairs = (table[:, None] | (table[None, :] << 4)).reshape(-1)
    r = torch.randint(0, 1 << 18, (N, K // 2), generator=gen, device=DEV, dtype=torch.int32)
    out = pairs[(r & 0xffff)]
    if fmt != "int4":   # signs
        out |= ((r >> 16) & 1).to(torch.uint8) << 3 | ((r >> 17) & 1).to(torch.uint8) << 7
    return out


def _bytes(gen, shape, lo, hi):
    return torch.randint(lo, hi + 1, shape, generator=gen, device=DEV, dtype=torch.uint8)


def _linear_inputs(case, seed):
    g = _generator(seed)
    M, N, K, fmt = case["M"], case["N"], case["K"], case["fmt"]
    gated = case["act"] == "swiglu"
    rows = 2 * N if gated else N
    st = dict(x=_normal(g, (M, K), 1.0), codes=_codes(g, rows, K, fmt), gs=None, bias=None,
              row_scale=None, residual=None)
    if fmt == "mxfp4":     # group scales 2^-7 .. 2^-6
        st["scales"] = _bytes(g, (rows, K // 32), 120, 121)
    elif fmt == "nvfp4":   # e4m3 bytes 2^5 .. 1.875 * 2^6 under a second-level scale
        st["scales"] = _bytes(g, (rows, K // 16), 0x60, 0x6f)
        st["gs"] = torch.empty(2 if gated else 1, device=DEV).uniform_(1.0, 2.0, generator=g) \
            * (0.008 / 64)
    else:
        st["scales"] = torch.empty((rows, K // case["group"]), device=DEV) \
            .uniform_(0.8, 1.25, generator=g) * (STD / 3.0)
    if case["bias"]:
        st["bias"] = _normal(g, (rows,), 0.5, torch.float32)
    if case["scale"]:   # a gate in (0, 1)
        st["row_scale"] = torch.sigmoid(_normal(g, (M,), 1.0, torch.float32))
    if case["residual"] != "none":
        st["residual"] = _normal(g, (M, N), 1.0,
                                 torch.float32 if case["residual"] == "f32" else torch.bfloat16)
    return st


def _router_inputs(case, seed):
    g = _generator(seed)
    T, E, K, S = case["T"], case["E"], case["K"], case["sequences"]
    tilt = _normal(g, (E,), 0.5, torch.float32)   # some experts are liked more
    logits = (_normal(g, (T, E), 1.5, torch.float32) + tilt).to(
        torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :K].to(torch.int32)
    if case["dropped"]:   # past an expert's capacity
        ids = torch.where(torch.rand(ids.shape, generator=g, device=DEV) < 0.05, -1, ids)
    # sequence starts: uneven, the last one ends `pad` rows before T
    used = T - case["pad"]
    cuts = torch.rand(S - 1, generator=g, device=DEV).mul(used).long().sort().values
    ends = torch.tensor([used], device=DEV)
    starts = torch.cat([torch.zeros_like(ends), cuts, ends]).to(torch.int32)
    return dict(logits=logits, ids=ids.contiguous(), starts=starts,
                g_weights=_normal(g, (T, K), 1e-3, torch.float32),
                g_balance=torch.full((), 0.01, device=DEV), g_z=torch.full((), 0.001, device=DEV))


def prepare(case, seed):
    if case["op"] == "linear4":
        st = dict(case=case, **_linear_inputs(case, seed))
        if own:   # the weights a server lays out once, when they are loaded
            st["weight"] = _own_weight(case, st)
        return st
    st = dict(case=case, **_router_inputs(case, seed))
    if own:   # what a training step differentiates
        _path()
        st["logits"].requires_grad_(True)
    return st


def _own_weight(case, st):
    _path()
    from xtu_moe_amd.linear4 import Weight4
    return Weight4.from_dense(case["fmt"], st["codes"], st["scales"], st["gs"],
                              gated=case["act"] == "swiglu")


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
    if case["op"] == "linear4":
        return _plain_linear(case, state)
    return _plain_router(case, state)


def _run_own(case, st):
    if case["op"] == "linear4":
        from xtu_moe_amd.linear4 import linear4
        return linear4(st["x"], st["weight"], bias=st["bias"], activation=case["act"],
                       row_scale=st["row_scale"], residual=st["residual"],
                       out_dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
    from xtu_moe_amd.router import router_losses
    r = router_losses(st["logits"], st["ids"], scoring=case["scoring"],
                      renormalize=case["renormalize"], routed_scaling_factor=case["scale"],
                      seq_starts=st["starts"])
    outs, grads = [r.weights, r.balance], [st["g_weights"], st["g_balance"]]
    if r.z is not None:
        outs.append(r.z)
        grads.append(st["g_z"])
    d, = torch.autograd.grad(outs, st["logits"], grads)
    return dict(weights=r.weights.detach(), balance=r.balance.detach(),
                z=None if r.z is None else r.z.detach(), counts=r.counts, probs=r.probs, dlogits=d)


def _activate(act, z):
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
        return g / (1 + torch.exp(-g)) * u
    return z


def _dequantize(case, st):
    """The matrix in 32 bits."""
    q, s, rows = st["codes"], st["scales"], st["codes"].shape[0]
    if case["fmt"] == "int4":
        lut = torch.arange(16, device=q.device).float() - 8
    else:
        lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    v = torch.stack([lut[(q & 15).int()], lut[(q >> 4).int()]], -1).view(rows, s.shape[1], -1)
    if case["fmt"] == "mxfp4":
        s = torch.exp2(s.float() - 127)
    elif case["fmt"] == "nvfp4":
        gs = st["gs"].repeat_interleave(rows // st["gs"].numel())
        s = s.view(torch.float8_e4m3fn).float() * gs[:, None]
    return (v * s[:, :, None]).view(rows, -1)


def _plain_linear(case, st):
    z = st["x"].float() @ _dequantize(case, st).t()
    if st["bias"] is not None:
        z = z + st["bias"]
    y = _activate(case["act"], z)
    if st["row_scale"] is not None:
        y = y * st["row_scale"][:, None]
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y if case["out"] == "f32" else y.to(torch.bfloat16)


def _plain_router(case, st):
    lg, ids, starts = st["logits"].float(), st["ids"].long(), st["starts"].long()
    T, E = lg.shape
    K, S, f = ids.shape[1], starts.numel() - 1, case["scale"]
    soft = case["scoring"] == "softmax"
    # probabilities over all experts
    if soft:
        m = lg.amax(1, keepdim=True)
        e = torch.exp(lg - m)
        total = e.sum(1, keepdim=True)
        p, s = e / total, None
        lse = (m + torch.log(total))[:, 0]
    else:
        s = 1 / (1 + torch.exp(-lg))
        p = s / s.sum(1, keepdim=True)
    # the selected experts' weights
    there = (ids >= 0) & (ids < E)
    at = torch.where(there, ids, torch.zeros_like(ids))
    sel = (p if soft else s).gather(1, at) * there
    if case["renormalize"]:
        norm = sel.sum(1, keepdim=True)
        u = torch.where(norm > 0, sel / norm, torch.zeros_like(sel))
    else:
        u = sel
    # sequences of the rows (S: none), counts and means
    row = torch.arange(T, device=lg.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp(max=S)
    n = starts[1:] - starts[:-1]
    member = (seq[:, None] == torch.arange(S, device=lg.device)).double().t()
    hits = torch.zeros((T, E), dtype=torch.float64, device=lg.device)
    hits = hits.scatter_add(1, at, there.double())
    counts = (member @ hits).to(torch.int32)
    sums = member @ p.double()
    nn = n.clamp(min=1).double()
    probs = sums / nn[:, None]
    Q = (n > 0).sum().clamp(min=1).double()
    balance = ((counts.double() * probs).sum(1) * E / (K * nn)).sum() / Q
    # the gradient
    share = st["g_balance"].double() * E / (K * nn * nn * Q)
    h = torch.cat([counts.double() * share[:, None],
                   torch.zeros((1, E), dtype=torch.float64, device=lg.device)]).float()[seq]
    d = p * (h - (p * h).sum(1, keepdim=True))
    if not soft:
        d = d * (1 - s)
    z = None
    if soft:
        used = seq < S
        count = used.sum().clamp(min=1).double()
        z = (torch.where(used, lse.double() ** 2, 0.0).sum() / count).float()
        dz = torch.where(used, 2 * lse, torch.zeros_like(lse)) * (st["g_z"] / count.float())
        d = d + dz[:, None] * p
    g = st["g_weights"]
    if case["renormalize"]:
        dk = f * u * (g - (u * g).sum(1, keepdim=True))
    else:
        dk = f * u * g
        if soft:
            d = d - dk.sum(1, keepdim=True) * p
    if not soft:
        dk = dk * (1 - s.gather(1, at))
    d = d.scatter_add(1, at, dk * there)
    return dict(weights=f * u, balance=balance.float(), z=z, counts=counts, probs=probs.float(),
                dlogits=d.to(st["logits"].dtype))


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "linear4":
        M, N, K = case["M"], case["N"], case["K"]
        rows = 2 * N if case["act"] == "swiglu" else N
        per = {"mxfp4": 0.5 + 1 / 32, "nvfp4": 0.5 + 1 / 16,
               "int4": 0.5 + 4 / (case["group"] or 128)}[case["fmt"]]
        nbytes = rows * K * per + 2 * M * K + M * N * (4 if case["out"] == "f32" else 2)
        nbytes += 4 * rows * case["bias"] + 4 * M * case["scale"]
        nbytes += M * N * {"none": 0, "bf16": 2, "f32": 4}[case["residual"]]
        return {"bytes": float(nbytes), "flops": 2.0 * M * rows * K}
    # logits, ids and the weights' gradient read; weights and the logits'
    # gradient written; counts and means of the sequences
    T, E, K, S = case["T"], case["E"], case["K"], case["sequences"]
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": float(2 * size * T * E + 12 * T * K + 8 * S * E + 4 * S),
            "flops": 12.0 * T * E}


# ------------------------------------------------------------------ exact
def _exact_linear(case, st):
    q, s, fmt = st["codes"], st["scales"], case["fmt"]
    rows = q.shape[0]
    nib = torch.empty((rows, case["K"]), dtype=torch.uint8, device=q.device)
    nib[:, 0::2], nib[:, 1::2] = q & 15, q >> 4
    if fmt == "int4":
        w = nib.double() - 8
        w *= s.double().repeat_interleave(case["group"], 1)
    else:
        ex, m = (nib >> 1 & 3).double(), (nib & 1).double()
        w = torch.where(ex > 0, torch.exp2(ex - 1) * (1 + m / 2), m / 2)
        w = torch.where(nib > 7, -w, w)
        if fmt == "mxfp4":
            w *= torch.exp2(s.double() - 127).repeat_interleave(32, 1)
        else:
            ex, m = (s >> 3 & 15).double(), (s & 7).double()
            sc = torch.where(ex > 0, torch.exp2(ex - 7) * (1 + m / 8), m * 2.0 ** -9)
            w *= torch.where(s > 127, -sc, sc).repeat_interleave(16, 1)
            gs = st["gs"].double()
            w *= gs.repeat_interleave(rows // gs.numel())[:, None]
    y = torch.empty((case["M"], case["N"]), dtype=torch.float64, device=q.device)
    x = st["x"].double()
    for r in range(0, case["M"], 1024):   # rows at a time
        z = x[r:r + 1024] @ w.t()
        if st["bias"] is not None:
            z += st["bias"].double()
        if case["act"] == "swiglu":
            z = torch.nn.functional.silu(z[:, :case["N"]]) * z[:, case["N"]:]
        elif case["act"] in ("gelu", "gelu_tanh"):
            z = torch.nn.functional.gelu(z, approximate="tanh" if "tanh" in case["act"] else "none")
        elif case["act"] == "silu":
            z = torch.nn.functional.silu(z)
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


def _exact_router(case, st):
    """The losses and weights in 64 bits, their gradient by autograd."""
    T, E, K = case["T"], case["E"], case["K"]
    soft = case["scoring"] == "softmax"
    lg = st["logits"].double().requires_grad_(True)
    p = torch.softmax(lg, 1) if soft else torch.sigmoid(lg)
    ids = st["ids"].long()
    miss = ids < 0
    w = p.gather(1, ids.clamp(min=0)).masked_fill(miss, 0.0)
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = w / total.masked_fill(total == 0, 1.0)
    w = w * case["scale"]
    if not soft:
        p = p / p.sum(1, keepdim=True)
    b = st["starts"].tolist()
    counts, probs, losses = [], [], []
    for lo, hi in zip(b[:-1], b[1:]):
        sub = ids[lo:hi]
        c = torch.bincount(sub[sub >= 0], minlength=E)
        m = p[lo:hi].sum(0) / max(hi - lo, 1)
        counts.append(c)
        probs.append(m)
        if hi > lo:
            losses.append((c.double() / (K * (hi - lo)) * m).sum() * E)
    balance = torch.stack(losses).mean() if losses else lg.sum() * 0
    total = (w * st["g_weights"].double()).sum() + balance * st["g_balance"].double()
    z = None
    if soft:
        n = b[-1] - b[0]
        z = (torch.logsumexp(lg[b[0]:b[-1]], 1) ** 2).sum() / max(n, 1)
        total = total + z * st["g_z"].double()
    d, = torch.autograd.grad(total, lg)
    return dict(weights=w.detach(), balance=balance.detach(), z=None if z is None else z.detach(),
                counts=torch.stack(counts).to(torch.int32), probs=torch.stack(probs).detach(),
                dlogits=d)


def exact(case, seed):
    if case["op"] == "linear4":
        return _exact_linear(case, _linear_inputs(case, seed))
    return _exact_router(case, _router_inputs(case, seed))
