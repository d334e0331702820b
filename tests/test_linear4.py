"""The dense product with 4-bit weights: the packed layout, and everything that
is turned away on the host, before a launch."""
import os

import pytest
import torch

from xtu_moe_amd import _lib, formats as F
from xtu_moe_amd.linear import ACTIVATIONS
from xtu_moe_amd.linear4 import ARGS, Weight4, linear4

BF = torch.bfloat16
GROUPS = [(F.FMT_MXFP4, 32), (F.FMT_NVFP4, 16), (F.FMT_INT4, 32), (F.FMT_INT4, 64),
          (F.FMT_INT4, 128)]


def _dense(fmt, rows, K, group, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8)
    if fmt == F.FMT_INT4:
        s = torch.rand((rows, K // group), generator=g) + 0.5
    else:
        s = torch.randint(100, 120, (rows, K // group), generator=g, dtype=torch.uint8)
    return codes, s, 0.25 if fmt == F.FMT_NVFP4 else None


# (kernel, K split or not) -> M, N, K of a product that takes it, for every format;
# gated ones have the same number of rows
FORMS = {
    (0, False): [(1, 300, 512), (5, 296, 128), (2, 12000, 640), (1, 150, 9600)],
    (1, False): [(1, 16, 1792), (3, 4000, 2176), (7, 182, 1536), (16, 534, 1280), (24, 2037, 768),
                 (42, 407, 640), (50, 102, 384), (64, 1500, 2176), (36, 112, 3712),
                 (65, 16, 128), (137, 1140, 384), (71, 16, 896), (123, 504, 2816),   # parts of
                 (300, 1700, 640), (97, 3000, 512), (70, 8000, 256), (5000, 34, 256),   # x
                 (80, 6500, 512), (128, 2000, 640)],
    (2, False): [(20, 16864, 128), (30, 18111, 512), (44, 21292, 128), (51, 18559, 128)],
    (2, True): [(10, 16, 7808), (13, 40, 9600), (33, 17986, 2944)],
    (3, False): [(68, 8420, 128), (579, 4514, 256)],
    (3, True): [(97, 8196, 2304), (1685, 68, 4736)],
    (4, False): [(1224, 3405, 256), (1838, 2228, 512)],
    (4, True): [(65, 4186, 7296)],
    None: [(26, 396, 8448), (64, 148, 9216), (65, 5888, 5248)],   # not the same for all
}


def forms(fmt, group, gated):
    """(form, M, N, K) of this format: INT4's finer groups have no kernel 4."""
    for form, sizes in FORMS.items():
        if form is None or form[0] != 4 or fmt != F.FMT_INT4 or group == 128:
            for M, N, K in sizes:
                yield form, M, N // 2 if gated else N, K


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
@pytest.mark.parametrize("fmt,group", GROUPS)
@pytest.mark.parametrize("gated", [False, True])
def test_forms_are_taken(fmt, group, gated):
    for form, M, N, K in forms(fmt, group, gated):
        plan = _lib.load().xtu_linear4_plan(M, N, K, 6 if gated else 0, fmt, group)
        assert form in ((plan % 16, plan >= 32), None), (M, N, K, plan % 16, plan // 16)


def _w(fmt="mxfp4", rows=4, K=32, gated=False):
    group = {"mxfp4": 32, "nvfp4": 16, "int4": 32}[fmt]
    c, s, gs = _dense(F.fmt_of(fmt), rows, K, group)
    return Weight4.from_dense(fmt, c, s, gs, gated=gated)


@pytest.mark.parametrize("fmt,group", GROUPS)
@pytest.mark.parametrize("gated", [False, True])
def test_records(fmt, group, gated):
    """Every code and scale at the place that the kernels read it from."""
    for N, K in ((1, 128), (16, 256), (21, 384), (35, 3 * group)):
        halves = 2 if gated else 1
        codes, s, gs = _dense(fmt, N * halves, K, group, seed=N)
        W = Weight4.from_dense(fmt, codes, s, gs, gated=gated)
        P, B = (N + 15) // 16, (K + 127) // 128
        rec = {F.FMT_MXFP4: 1088, F.FMT_NVFP4: 1152, F.FMT_INT4: 1024 + 8192 // group}[fmt]
        assert W.data.shape == (P * halves, B, rec) and W.data.is_contiguous()
        assert (W.N, W.K, W.group, W.gated) == (N, K, group, gated)
        if os.path.exists(_lib.LIB_PATH):
            assert _lib.load().xtu_linear4_weight_bytes(N, K, 6 if gated else 0, fmt, group) == W.nbytes
        n, k = torch.meshgrid(torch.arange(P * 16), torch.arange(B * 128), indexing="ij")
        b, kk = k // 128, k % 128
        j, q = kk // 32, kk // 8 % 4
        i = kk % 8
        byte, high = (4 * j + i % 4, i // 4) if fmt == F.FMT_INT4 else (4 * j + i // 2, i % 2)
        for h in range(halves):
            pan = (n // 16) * halves + h
            got = W.data[pan, b, (q * 16 + n % 16) * 16 + byte] >> (4 * high) & 15
            want = torch.zeros(P * 16, B * 128, dtype=torch.uint8)
            nib = torch.stack([codes & 15, codes >> 4], -1).view(halves, N, K)[h]
            want[:N, :K] = torch.where(nib >= 8, nib - 8, 15 - nib) if fmt == F.FMT_INT4 else nib
            assert torch.equal(got, want)
            sv = torch.full((P * 16, B * 128), 127 if fmt == F.FMT_MXFP4 else 0, dtype=s.dtype)
            sv[:N, :K] = s.view(halves, N, -1)[h].repeat_interleave(group, 1)
            if fmt == F.FMT_INT4:
                planes = W.data[..., 1024:].contiguous().view(torch.float32)
                got = planes[pan, b, kk // group * 16 + n % 16]
            elif fmt == F.FMT_MXFP4:
                got = W.data[pan, b, 1024 + (n % 16) * 4 + j]
            else:
                got = W.data[pan, b, 1024 + q // 2 * 64 + (n % 16) * 4 + j]
            assert torch.equal(got, sv)


def _refused_w(match, *args, **kw):
    with pytest.raises(ValueError, match=match):
        Weight4.from_dense(*args, **kw)


def test_weights_refused():
    c, s, _ = _dense(F.FMT_MXFP4, 4, 64, 32)
    _refused_w("4-bit", "bf16", c, s)
    _refused_w("4-bit", "fp8", c, s)
    _refused_w("codes", "mxfp4", c[0], s)
    _refused_w("codes", "mxfp4", c.int(), s)
    _refused_w("codes", "mxfp4", c[:0], s[:0])
    _refused_w("scales", "mxfp4", c, s[:3])
    _refused_w("scales", "mxfp4", c, s[0])
    _refused_w("groups", "mxfp4", c, s[:, :1])
    _refused_w("split", "mxfp4", c, s[:, :0])
    _refused_w("bytes", "mxfp4", c, s.float())
    _refused_w("no second-level", "mxfp4", c, s, 1.0)
    _refused_w("equal number", "mxfp4", c[:3], s[:3], gated=True)
    for bad in (253, 255):
        _refused_w("e8m0", "mxfp4", c, torch.full_like(s, bad))
    Weight4.from_dense("mxfp4", c, torch.full_like(s, 252))
    n = torch.full((4, 4), 0x38, dtype=torch.uint8)
    _refused_w("second-level", "nvfp4", c, n)
    _refused_w("second-level", "nvfp4", c, n, torch.ones(2))
    _refused_w("second-level", "nvfp4", c, n, torch.ones(3), gated=True)
    for bad in (0x7f, 0xff):
        _refused_w("NaN", "nvfp4", c, torch.full_like(n, bad), 1.0)
    w = Weight4.from_dense("nvfp4", c, n.view(torch.float8_e4m3fn), torch.tensor([2.0, 3.0]), gated=True)
    assert w.gs.tolist() == [2.0, 3.0] and w.N == 2
    assert Weight4.from_dense("nvfp4", c, n, 2.0, gated=True).gs.tolist() == [2.0, 2.0]
    f = torch.ones((4, 2))
    _refused_w("fp32", "int4", c, f.double())
    _refused_w("fp32", "int4", c, f.int())
    for bad in (float("nan"), float("inf"), 2.0 ** 123):
        _refused_w("finite", "int4", c, f * bad)
    _refused_w("groups", "int4", c, torch.ones((4, 4)))
    for t in (torch.float32, torch.float16, BF):
        assert Weight4.from_dense("int4", c, f.to(t)).data.shape == (1, 1, 1024 + 256)


def test_weights_in_other_orders():
    """Checkpoint tensors as views: transposed storage, slices, torch's scale types."""
    for fmt, group in GROUPS:
        codes, s, gs = _dense(fmt, 40, 256, group, seed=5)
        want = Weight4.from_dense(fmt, codes, s, gs, gated=True)
        wide = torch.zeros((40, 200), dtype=torch.uint8)
        wide[:, 7:135] = codes
        for c, z in ((codes.t().contiguous().t(), s.t().contiguous().t()), (wide[:, 7:135], s)):
            got = Weight4.from_dense(fmt, c, z, gs, gated=True)
            assert torch.equal(got.data, want.data)
    codes, s, _ = _dense(F.FMT_MXFP4, 40, 256, 32, seed=5)
    assert torch.equal(Weight4.from_dense("mxfp4", codes, s.view(torch.float8_e8m0fnu)).data,
                       Weight4.from_dense("mxfp4", codes, s).data)


def test_weights_do_not_change():
    """The kernels take the records' size from N and K: other records are refused."""
    import dataclasses
    w = _w("nvfp4", 36, 160, gated=True)
    for field in ("data", "gs", "N", "K"):
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(w, field, getattr(w, field))
    for kw in (dict(data=w.data[:1]), dict(data=w.data.int()), dict(N=40), dict(K=512),
               dict(gated=False), dict(data=w.data.flip(0).transpose(0, 1)), dict(gs=None),
               dict(gs=w.gs[:1]), dict(gs=w.gs.double()), dict(fmt=F.FMT_MXFP4, group=32)):
        with pytest.raises(ValueError, match="must be"):
            dataclasses.replace(w, **kw)
    moved = w.to("cpu")
    assert torch.equal(moved.data, w.data) and moved.nbytes == w.nbytes


def _refused(match, *args, **kw):
    with pytest.raises(ValueError, match=match):
        linear4(*args, **kw)


def test_operands_refused():
    x, w = torch.zeros((3, 32), dtype=BF), _w()
    _refused("Weight4", x, torch.zeros((4, 32), dtype=BF))
    _refused("2-D", x[0], w)
    _refused("2-D", x.float(), w)
    _refused("columns", x[:, :31], w)
    _refused("contiguous", torch.zeros((32, 3), dtype=BF).t(), w)
    _refused("CUDA", x, w)
    _refused("rows", x[:1].expand((1 << 31) - 511, 32), w)
    _refused("unknown activation", x, w, activation="tanh")
    _refused("swiglu", x, w, activation="swiglu")
    _refused("swiglu", x, _w(gated=True))
    for name in ACTIVATIONS:   # each gets as far as the device check
        _refused("CUDA", x, _w(gated=name == "swiglu"), activation=name)


def test_epilogue_operands_refused():
    x, w = torch.zeros((3, 32), dtype=BF), _w()
    f32 = torch.float32
    _refused("bias", x, w, bias=torch.zeros(3))
    _refused("bias", x, w, bias=torch.zeros(4, dtype=torch.float16))
    _refused("bias", x, w, bias=torch.zeros(8)[::2])
    _refused("bias", x, _w(gated=True), bias=torch.zeros(2), activation="swiglu")   # 2N values
    _refused("row_scale", x, w, row_scale=torch.zeros(4))
    _refused("row_scale", x, w, row_scale=torch.zeros(3, dtype=BF))
    _refused("residual", x, w, residual=torch.zeros((2, 4), dtype=f32))
    _refused("columns", x, w, residual=torch.zeros((3, 3), dtype=f32))
    _refused("residual", x, w, residual=torch.zeros((3, 4), dtype=torch.float64))
    _refused("residual", x, w, residual=torch.zeros((4, 3), dtype=f32).t())
    _refused("output type", x, w, out_dtype=torch.float16)
    _refused("output type", x, w, out=torch.zeros((3, 4), dtype=BF), out_dtype=f32)
    _refused("does not hold", x, w, out=torch.zeros((2, 4), dtype=BF))
    _refused("does not hold", x, w, out=torch.zeros((1, 4), dtype=BF).expand(3, 4))
    _refused("columns", x, w, out=torch.zeros((3, 5), dtype=BF))
    both = torch.zeros((3, 40), dtype=BF)
    _refused("overlaps x", both[:, :32], w, out=both[:, 30:34])
    _refused("overlaps residual", x, w, residual=both[:, 0:4], out=both[:, 2:6])
    _refused("overlaps w", x, w, out=w.data.view(-1)[:24].view(BF).view(3, 4))
    _refused("CUDA", x, w, residual=both[:, :4], out=both[:, :4])   # in place: allowed


def test_gradients_refused():
    """There is no backward: a result without one would train nothing, silently."""
    x, w = torch.zeros((3, 32), dtype=BF), _w()
    for kw in (dict(bias=torch.zeros(4)), dict(row_scale=torch.zeros(3)),
               dict(residual=torch.zeros((3, 4)))):
        t = next(iter(kw.values())).requires_grad_(True)
        _refused("no backward", x, w, **kw)
        with torch.no_grad():
            _refused("CUDA", x, w, **kw)
        assert t.requires_grad
    _refused("no backward", x.requires_grad_(True), w)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_entry_refuses_on_the_host():
    lib = _lib.load()

    def rc(x=16, w=16, gs=0, bias=0, out=16, ws=0, ldx=32, ldr=0, ldo=8, sst=0, M=1, N=1, K=32,
           act=0, fmt=2, group=32):
        return lib.xtu_linear4(ARGS.pack(x, w, gs, bias, 0, 0, out, ws, ldx, ldr, ldo, sst, 0, M, N,
                                         K, act, fmt, group, 0, 0, 1, 0.0, 1.0, 0.0), None)

    assert lib.xtu_linear4(None, None) == 1
    assert rc(M=0) == 0                       # nothing to do, nothing launched
    for bad in (dict(x=0), dict(x=17), dict(w=0), dict(w=8), dict(out=0), dict(M=-1), dict(N=0),
                dict(K=0), dict(act=7), dict(act=-1), dict(ldx=-1), dict(ldr=-1), dict(sst=-1),
                dict(ws=8), dict(M=2, N=9), dict(N=1 << 29), dict(K=1 << 29), dict(fmt=0),
                dict(fmt=1), dict(fmt=5), dict(group=16), dict(fmt=3, group=16), dict(gs=16),
                dict(fmt=3, group=32, gs=16), dict(fmt=4, group=16), dict(K=48),
                dict(fmt=4, group=64, K=96), dict(M=(1 << 31) - 511),
                dict(M=1 << 30, N=1 << 20, ldo=1 << 20)):
        assert rc(**bad) == 1, bad
    assert lib.xtu_linear4_workspace_bytes(0, 1, 32, 0, 2, 32, 1) == 0
    assert lib.xtu_linear4_workspace_bytes(1, 1, 33, 0, 2, 32, 1) == 0
    assert lib.xtu_linear4_workspace_bytes(5, 1, 96, 0, 2, 32, 0) == 5 * 96 * 2   # a copy of x
    assert lib.xtu_linear4_plan(0, 1, 32, 0, 2, 32) == lib.xtu_linear4_plan(1, 1, 48, 0, 2, 32) == -1
    assert lib.xtu_linear4_weight_bytes(1, 32, 0, 1, 32) == 0


def test_tangents_refused():
    """Nor a forward-mode derivative, which requires_grad does not show."""
    from torch.autograd import forward_ad
    w, zeros = _w(), torch.zeros((3, 32), dtype=BF)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                _refused("forward-mode", dual(zeros), w)
                for kw in (dict(bias=torch.zeros(4)), dict(row_scale=torch.zeros(3)),
                           dict(residual=torch.zeros((3, 4))), dict(out=torch.zeros((3, 4)))):
                    _refused("forward-mode", zeros, w, **{k: dual(v) for k, v in kw.items()})
                    _refused("CUDA", zeros, w, **kw)


def test_unaligned_rows_are_not_read_as_aligned():
    """The kernel for rows of x at any 2-byte address takes them with a load that claims
    no more: an access through a 16-byte-aligned type would be right by luck only."""
    import re
    src = os.path.join(os.path.dirname(_lib.__file__), "..", "csrc", "linear4_tile.hip")
    text = open(src).read()
    loads = [line for line in text.splitlines() if "xrow[i]" in line and "xv[i]" in line]
    assert len(loads) == 1
    fn = re.search(r"xv\[i\] = (\w+)\(", loads[0]).group(1)
    body = re.search(r"u32x4_t " + fn + r"\(.*?\n}", text, re.S).group(0)
    assert "__builtin_memcpy" in body and "reinterpret_cast" not in body


def test_second_level_scales_are_checked():
    c, n = torch.zeros((4, 32), dtype=torch.uint8), torch.full((4, 4), 0x38, dtype=torch.uint8)
    for bad in (float("nan"), float("inf"), -float("inf"), 1e39):
        _refused_w("finite", "nvfp4", c, n, bad)
        _refused_w("finite", "nvfp4", c, n, torch.tensor([1.0, bad]), gated=True)
    for good in (0.0, -2.0, 3e38):
        assert Weight4.from_dense("nvfp4", c, n, good).gs.tolist() == [torch.tensor(good).item()]


def test_weights_are_constants():
    """Parameters are packed as they are now; records that claim a gradient are refused."""
    import dataclasses
    c, n = torch.zeros((4, 32), dtype=torch.uint8), torch.full((4, 4), 0x38, dtype=torch.uint8)
    p = torch.nn.Parameter(torch.tensor([2.0]))
    w = Weight4.from_dense("nvfp4", c, n, p)
    assert not w.gs.requires_grad and w.gs.tolist() == [2.0]
    with torch.no_grad():
        p.fill_(5.0)
    assert w.gs.tolist() == [2.0]
    w.gs.requires_grad_(False)
    with pytest.raises(ValueError, match="without a gradient"):
        dataclasses.replace(w, gs=torch.nn.Parameter(w.gs.clone()))
    s = torch.nn.Parameter(torch.ones((4, 2)))
    got = Weight4.from_dense("int4", c, s)
    assert not got.data.requires_grad
    assert torch.equal(got.data, Weight4.from_dense("int4", c, s.detach()).data)
