"""Norms, 8-bit rows and matrix products.

CPU: every refusal of the C entry points and of the Python calls.
GPU: against the float64 oracle, within bounds derived here.

Norm: s is one float32 addition (2^-24), the sum of squares a float32 sum of at
most 32 terms a thread and 10 pairwise steps (below 2^-18), its root halves
that, and three products follow: y is within 2^-18 |y| before its rounding of
half a step (bfloat16 2^-8, float32 2^-24).  Codes: half a step of the exact
scale plus that (127 steps of 2^-18 are below 2^-10 of one); e4m3 half a step
is 2^-4 of the value, 2^-10 of the scale below its normal range.

Product: each product of two bfloat16 (e4m3) values is exact in float32; a
matrix instruction adds 16 (32) of them to the sum, and each of these additions
loses at most 2^-22 of the sum of magnitudes M, so K / 16 + 8 of them lose
(K / 16 + 8) 2^-22 M.  int8 sums are exact.  Scales, bias, activation (slope at
most 1.13) and residual: 2^-20 of their magnitudes; then half a step of the
output's type.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from flashnext_b200 import _lib
from oracle import dense as od

KINDS = ("int8", "e4m3")
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


# ---- CPU: refusals ----


def _set(a, **kw):
    b = type(a).from_buffer_copy(a)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def test_norm_refuses_before_any_device_call():
    lib = _lib.load()
    a = _lib.FnNormArgs(_lib.ABI_VERSION, 0, 4, 64, 0, 0, 0, 0, 1e-6, 0, 0x1000, 64, 0x2000, 64, 0x3000, 0x4000, 0x5000,
                        0x6000, 0x7000)
    run = lambda b: lib.fnmoe_add_rms_norm(ctypes.byref(b), None)  # noqa: E731
    for kw, code in (({"abi_version": 3}, _lib.ERR_ABI), ({"dim": 0}, _lib.ERR_SHAPE), ({"dim": 16385}, _lib.ERR_SHAPE),
                     ({"rows": 1 << 31}, _lib.ERR_SHAPE), ({"x_dtype": 2}, _lib.ERR_UNSUPPORTED),
                     ({"residual_dtype": 2}, _lib.ERR_UNSUPPORTED), ({"weight_dtype": 7}, _lib.ERR_UNSUPPORTED),
                     ({"code_type": 2}, _lib.ERR_UNSUPPORTED), ({"eps": -1e-6}, _lib.ERR_VALUE),
                     ({"eps": float("nan")}, _lib.ERR_VALUE), ({"eps": float("inf")}, _lib.ERR_VALUE),
                     ({"x": None}, _lib.ERR_NULL), ({"weight": None}, _lib.ERR_NULL),
                     ({"y": None, "codes": None}, _lib.ERR_NULL), ({"scales": None}, _lib.ERR_NULL),
                     ({"residual": None}, _lib.ERR_NULL), ({"x_stride": 63}, _lib.ERR_SHAPE),
                     ({"residual_stride": 63}, _lib.ERR_SHAPE), ({"x": 0x1001}, _lib.ERR_VALUE),
                     ({"scales": 0x7002}, _lib.ERR_VALUE), ({"weight": 0x3002, "weight_dtype": 1}, _lib.ERR_VALUE)):
        assert run(_set(a, **kw)) == code, kw
    assert run(_set(a, rows=0)) == _lib.OK
    assert lib.fnmoe_add_rms_norm(None, None) == _lib.ERR_NULL


def test_dequantize_refuses_before_any_device_call():
    lib = _lib.load()
    a = _lib.FnRowCodesArgs(_lib.ABI_VERSION, 4, 64, 0, 0, 0, 0x1000, 0x2000, 0x3000)
    for kw, code in (({"abi_version": 0}, _lib.ERR_ABI), ({"dim": 0}, _lib.ERR_SHAPE), ({"code_type": 2}, _lib.ERR_UNSUPPORTED),
                     ({"out_dtype": 2}, _lib.ERR_UNSUPPORTED), ({"codes": None}, _lib.ERR_NULL),
                     ({"scales": None}, _lib.ERR_NULL), ({"out": None}, _lib.ERR_NULL), ({"scales": 0x2001}, _lib.ERR_VALUE),
                     ({"out": 0x3001}, _lib.ERR_VALUE)):
        assert lib.fnmoe_dequantize_rows(ctypes.byref(_set(a, **kw)), None) == code, kw
    assert lib.fnmoe_dequantize_rows(ctypes.byref(_set(a, rows=0)), None) == _lib.OK


def test_linear_refuses_before_any_device_call():
    lib = _lib.load()
    a = _lib.FnLinearArgs(_lib.ABI_VERSION, _lib.LINEAR_BF16, 4, 64, 48, 0, 0, 0, 0, 0, 0x1000, 64, 0x2000, 64, None, None,
                          0x5000, 0x6000, 48, 0x7000)
    q = {"type": _lib.LINEAR_INT8, "x_scale": 0x8000, "weight_scale": 0x9000}
    for kw, code in (({"abi_version": 0}, _lib.ERR_ABI), ({"type": 3}, _lib.ERR_UNSUPPORTED),
                     ({"activation": 4}, _lib.ERR_UNSUPPORTED), ({"bias_dtype": 2}, _lib.ERR_UNSUPPORTED),
                     ({"out_dtype": 2}, _lib.ERR_UNSUPPORTED), ({"residual_dtype": 2}, _lib.ERR_UNSUPPORTED),
                     ({"in_width": 0}, _lib.ERR_SHAPE), ({"out_width": 0}, _lib.ERR_SHAPE),
                     ({"in_width": 131072}, _lib.ERR_SHAPE), ({"rows": 0x7FFFFF01}, _lib.ERR_SHAPE),
                     ({"x": None}, _lib.ERR_NULL), ({"weight": None}, _lib.ERR_NULL), ({"out": None}, _lib.ERR_NULL),
                     ({"x_scale": 0x8000}, _lib.ERR_NULL), (dict(q, x_scale=None), _lib.ERR_NULL),
                     (dict(q, weight_scale=None), _lib.ERR_NULL), ({"x_stride": 56}, _lib.ERR_SHAPE),
                     ({"weight_stride": 56}, _lib.ERR_SHAPE), ({"residual_stride": 47}, _lib.ERR_SHAPE),
                     ({"x": 0x1008}, _lib.ERR_VALUE), ({"weight": 0x2002}, _lib.ERR_VALUE),
                     ({"x_stride": 68}, _lib.ERR_VALUE), ({"weight_stride": 65}, _lib.ERR_VALUE),
                     (dict(q, x_stride=72), _lib.ERR_VALUE), (dict(q, x_scale=0x8002), _lib.ERR_VALUE),
                     ({"bias": 0x5001}, _lib.ERR_VALUE), ({"residual": 0x6002, "residual_dtype": 1}, _lib.ERR_VALUE),
                     ({"out": 0x7001}, _lib.ERR_VALUE)):
        assert lib.fnmoe_linear(ctypes.byref(_set(a, **kw)), None) == code, kw
    assert lib.fnmoe_linear(ctypes.byref(_set(a, rows=0)), None) == _lib.OK


def test_python_refuses_cpu_tensors_and_types():
    import torch

    from flashnext_b200 import dense

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: dense.add_rms_norm(x, x[0]), lambda: dense.quantize_rows(x), lambda: dense.linear(x, x),
                 lambda: dense.dequantize_rows(x.to(torch.int8), torch.ones(2)),
                 lambda: dense.add_rms_norm(x.half(), x[0]), lambda: dense.quantize_rows(x.double()),
                 lambda: dense.linear(x, x.float()), lambda: dense.linear(x.half(), x.half()),
                 lambda: dense.dequantize_rows(x, torch.ones(2))):
        with pytest.raises(TypeError):
            call()


# ---- GPU ----

gpu = pytest.mark.gpu


def _types():
    import torch

    return {"bf16": torch.bfloat16, "f32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _np(t):
    return t.detach().float().double().cpu().numpy()


def _gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _cut(x, pad, at=0):
    """x as columns ``at`` .. of rows that are ``pad`` wider."""
    import torch

    if not pad:
        return x
    wide = torch.zeros(x.shape[0], (x.shape[1] + pad) * x.element_size(), dtype=torch.uint8, device=x.device).view(x.dtype)
    wide.view(torch.uint8).fill_(0xFF)  # what lies beside the rows is not a number (bfloat16, float32, e4m3)
    wide[:, at:at + x.shape[1]] = x
    return wide[:, at:at + x.shape[1]]


def _held(codes, scales, y, kind):
    """Codes and scales of the rows y (float64), within their bounds."""
    want = od.row_scales(y, kind)
    scales = _np(scales)
    np.testing.assert_allclose(scales, want, rtol=2.0 ** -17)
    got = _np(codes) * scales[:, None]
    slack = np.abs(y) * 2.0 ** -16
    half = 0.5 * want[:, None] if kind == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, want[:, None] * 2.0 ** -10)
    assert (np.abs(got - y) <= half * (1 + 2.0 ** -10) + slack).all()


@gpu
@pytest.mark.parametrize("rows,dim,pad,at", [(1, 1, 0, 0), (3, 7, 5, 1), (1, 64, 0, 0), (5, 64, 8, 8), (4, 200, 0, 0),
                                             (129, 256, 0, 0), (2, 257, 0, 0), (7, 2048, 16, 8), (9, 2561, 3, 2),
                                             (3, 4104, 0, 0), (2, 8192, 0, 0), (2, 12000, 0, 0), (2, 16383, 0, 0),
                                             (3, 16384, 0, 0), (700, 512, 0, 0)])
@pytest.mark.parametrize("xd,rd,wd,offset,kind", [("bf16", "bf16", "bf16", False, "int8"), ("bf16", "f32", "f32", True, "e4m3"),
                                                  ("f32", None, "bf16", True, "int8"), ("f32", "bf16", "f32", False, "e4m3"),
                                                  ("bf16", None, "f32", False, None), ("f32", "f32", "bf16", True, None)])
def test_norm(cuda_lib, rows, dim, pad, at, xd, rd, wd, offset, kind):
    import torch

    from flashnext_b200 import dense

    t, g = _types(), _gen(rows * 31 + dim)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = _cut((randn(rows, dim) * torch.exp(2 * randn(rows, 1))).to(t[xd]), pad, at)
    res = None if rd is None else _cut(randn(rows, dim).to(t[rd]), pad, at)
    w = (1 - offset + 0.3 * randn(dim)).to(t[wd])
    got = dense.add_rms_norm(x, w, res, 1e-5, unit_offset=offset, codes=None if kind is None else t[kind], keep=True)
    y, s = od.add_rms_norm(_np(x), _np(w), None if res is None else _np(res), 1e-5, offset)
    assert got.y.dtype is t[xd]
    assert (np.abs(_np(got.y) - y) <= np.abs(y) * (HALF[xd] + 2.0 ** -18) + 1e-37).all()
    if rd is None:
        assert got.residual is None
    else:
        assert got.residual.dtype is t[rd]
        assert (np.abs(_np(got.residual) - s) <= np.abs(s) * (HALF[rd] + 2.0 ** -23) + 1e-37).all()
    if kind:
        _held(got.codes, got.scales, y, kind)
        alone = dense.add_rms_norm(x, w, res, 1e-5, unit_offset=offset, codes=t[kind])
        assert alone.y is None and torch.equal(alone.codes.view(torch.uint8), got.codes.view(torch.uint8))
        assert torch.equal(alone.scales, got.scales)


@gpu
def test_norm_in_place_residual_and_misaligned_starts(cuda_lib):
    import torch

    from flashnext_b200 import dense

    g = _gen(5)
    x = torch.randn(6, 96, device="cuda", generator=g).bfloat16()
    r = torch.randn(6, 96, device="cuda", generator=g)
    w = torch.randn(97, device="cuda", generator=g).bfloat16()
    want = dense.add_rms_norm(x, w[:96], r)
    buf = r.clone()
    got = dense.add_rms_norm(x, w[:96], buf, residual_out=buf)
    assert got.residual is buf and torch.equal(buf, want.residual) and torch.equal(got.y, want.y)
    # a weight, rows and a residual that start off a 16-byte boundary
    off = torch.empty(97, dtype=torch.bfloat16, device="cuda")[1:].copy_(w[:96])
    xo = torch.empty(6 * 96 + 3, dtype=torch.bfloat16, device="cuda")[3:].view(6, 96).copy_(x)
    ro = torch.empty(6 * 96 + 1, device="cuda")[1:].view(6, 96).copy_(r)
    # columns are dealt to threads in another order, so the sum of squares may differ in its last bits
    got = dense.add_rms_norm(xo, off, ro, residual_out=ro)
    assert torch.equal(ro, want.residual)
    assert (got.y.float() - want.y.float()).abs().max() <= want.y.float().abs().max() * 2.0 ** -7


@gpu
@pytest.mark.parametrize("dim", [96, 97, 2048, 16384])
def test_norm_far_magnitudes(cuda_lib, dim):
    """Rows whose squares or products leave float32's range, in one call with ordinary ones, and eps 0."""
    import torch

    from flashnext_b200 import dense

    g = _gen(dim)
    size = torch.tensor([1.0, 1e30, 3e37, 1e-30, 1e-37, 2.0 ** 64, 2.0 ** -64, 1e19], device="cuda")[:, None]
    x = torch.randn(8, dim, device="cuda", generator=g).clamp(-5, 5) * size
    w = torch.rand(dim, device="cuda", generator=g) + 0.5
    for eps in (0.0, 1e-6, 1e-38):
        for weight in (w, w * 2.0 ** 60):
            got = dense.add_rms_norm(x, weight, eps=eps, codes=torch.int8, keep=True)
            y, _ = od.add_rms_norm(_np(x), _np(weight), None, float(np.float32(eps)))
            # below float32's normal range a value keeps an absolute error of its last bit
            assert (np.abs(_np(got.y) - y) <= np.abs(y) * 2.0 ** -17 + 2.0 ** -140).all()
            np.testing.assert_allclose(_np(got.scales), od.row_scales(y, "int8"), rtol=2.0 ** -17)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_zero_or_not_finite(cuda_lib, kind):
    import torch

    from flashnext_b200 import dense

    x = torch.randn(6, 72, device="cuda")
    x[1] = 0.0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = 2.0 ** -120
    w = torch.ones(72, device="cuda")
    for r in (dense.add_rms_norm(x, w, codes=_types()[kind], keep=True), None):
        codes, scales = (r.codes, r.scales) if r else dense.quantize_rows(x, _types()[kind])
        assert torch.isnan(scales[2:4]).all() and torch.isfinite(scales[[0, 1, 4, 5]]).all()
        assert (codes[1:4].float() == 0).all()
        assert (scales[1] > 0) and (dense.dequantize_rows(codes, scales)[1] == 0).all()
        assert torch.isnan(dense.dequantize_rows(codes, scales)[2:4]).all()
        if r:
            assert torch.isnan(r.y[3]).all() and torch.isnan(r.y[2, 5]) and (r.y[1] == 0).all()
    np.testing.assert_allclose(float(scales[4]), 2.0 ** -100 / od.TOP[kind], rtol=1e-6)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,dim,pad", [(1, 1, 0), (3, 33, 2), (64, 4096, 0), (65, 2561, 0), (2, 16384, 8), (1001, 24, 0)])
@pytest.mark.parametrize("xd", ["bf16", "f32"])
def test_quantize_and_back(cuda_lib, kind, rows, dim, pad, xd):
    import torch

    from flashnext_b200 import dense

    t = _types()
    x = _cut((torch.randn(rows, dim, device="cuda", generator=_gen(dim)) * 3).to(t[xd]), pad)
    codes, scales = dense.quantize_rows(x, t[kind])
    _held(codes, scales, _np(x), kind)
    for out in ("bf16", "f32"):
        back = dense.dequantize_rows(codes, scales, t[out])
        want = _np(codes) * _np(scales)[:, None]
        assert back.dtype is t[out] and (np.abs(_np(back) - want) <= np.abs(want) * HALF[out] + 1e-40).all()
    assert torch.equal(dense.dequantize_rows(codes, scales, out=torch.empty(rows, dim, device="cuda")),
                       dense.dequantize_rows(codes, scales, torch.float32))


def _product(m, k, n, kind, seed, pad=0, wpad=0):
    import torch

    t, g = _types(), _gen(seed)
    x = torch.randn(m, k, device="cuda", generator=g) * 2
    w = torch.randn(n, k, device="cuda", generator=g) * k ** -0.5
    if kind == "bf16":
        return _cut(x.bfloat16(), pad), _cut(w.bfloat16(), wpad), None, None
    if kind == "int8":  # every code, the ends among them
        x, w = (torch.randint(-127, 128, s.shape, device="cuda", generator=g).to(torch.int8) for s in (x, w))
    else:
        x, w = (x * 50).clamp(-448, 448).to(t[kind]), (w * 1000).clamp(-448, 448).to(t[kind])
    return (_cut(x, pad), _cut(w, wpad), torch.rand(m, device="cuda", generator=g) + 0.1,
            (torch.rand(n, device="cuda", generator=g) + 0.1) * 1e-3)


def _check_linear(x, w, xs, ws, kind, out, bias=None, act=None, residual=None, **kw):
    import torch

    from flashnext_b200 import dense

    f = lambda v: None if v is None else _np(v)  # noqa: E731
    got = dense.linear(x, w, bias, activation=act, residual=residual, x_scale=xs, weight_scale=ws, out_dtype=_types()[out],
                       **kw)
    want, mag = od.linear(_np(x), _np(w), f(bias), act, f(residual), f(xs), f(ws))
    k = x.shape[1]
    sums = 0.0 if kind == "int8" else (k / 16 + 8) * 2.0 ** -22 * mag
    rest = mag if kind != "int8" else np.abs(od.linear(_np(x), _np(w), None, None, None, f(xs), f(ws))[0])
    rest = rest + (0 if bias is None else np.abs(f(bias))) + (0 if residual is None else np.abs(f(residual)))
    bound = 1.13 * sums + 2.0 ** -20 * rest + HALF[out] * np.abs(want) + 1e-37
    bad = np.abs(_np(got) - want) > bound
    assert not bad.any(), (np.argwhere(bad)[:5], _np(got)[bad][:5], want[bad][:5])
    return got


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (1, 16, 129), (2, 2048, 512), (16, 528, 300), (17, 64, 128), (31, 1024, 1000),
                                   (33, 4096, 2048), (64, 80, 77), (65, 2048, 130), (128, 160, 384), (129, 512, 200),
                                   (256, 336, 257), (257, 1024, 513), (700, 2576, 1003), (1, 16384, 640)])
def test_linear(cuda_lib, kind, m, k, n):
    _check_linear(*_product(m, k, n, kind, m + k + n), kind, "f32")


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("bd,rd,out", [(None, None, "bf16"), ("bf16", "f32", "bf16"), ("f32", "bf16", "f32"),
                                       (None, "f32", "f32"), ("bf16", None, "f32")])
@pytest.mark.parametrize("m,k,n,pad,rpad", [(5, 2064, 520, 0, 0), (150, 272, 1001, 16, 3)])
def test_linear_epilogue(cuda_lib, kind, act, bd, rd, out, m, k, n, pad, rpad):
    import torch

    t, g = _types(), _gen(m + n)
    bias = None if bd is None else torch.randn(n, device="cuda", generator=g).to(t[bd])
    res = None if rd is None else _cut((3 * torch.randn(m, n, device="cuda", generator=g)).to(t[rd]), rpad)
    _check_linear(*_product(m, k, n, kind, n, pad, 2 * pad), kind, out, bias, act, res)


@gpu
def test_linear_many_tiles_and_rows(cuda_lib):
    """More tiles than CTAs (accumulators and rings wrap), wide and tall."""
    _check_linear(*_product(16, 128, 60000, "bf16", 1), "bf16", "f32")
    _check_linear(*_product(9000, 64, 300, "int8", 2), "int8", "bf16")
    _check_linear(*_product(3000, 144, 2100, "e4m3", 3), "e4m3", "bf16")


@gpu
def test_linear_values_that_are_not_finite_stay_in_their_row_and_column(cuda_lib):
    import torch

    from flashnext_b200 import dense

    x, w, _, _ = _product(20, 128, 140, "bf16", 4)
    clean = dense.linear(x, w, out_dtype=torch.float32)
    x, w = x.clone(), w.clone()
    x[3, 5] = float("nan")
    x[4, 5] = float("inf")
    w[7, 9] = float("inf")
    got = dense.linear(x, w, out_dtype=torch.float32)
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[4]).any() and not torch.isfinite(got[:, 7]).any()
    rows = [i for i in range(20) if i not in (3, 4)]
    cols = [i for i in range(140) if i != 7]
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    relu = dense.linear(x, w, activation="relu", out_dtype=torch.float32)
    assert torch.isnan(relu[3]).all()


@gpu
def test_linear_in_place_residual_is_the_same_and_repeats(cuda_lib):
    import torch

    from flashnext_b200 import dense

    for m, k, n in ((3, 2048, 256), (300, 512, 1000)):
        x, w, xs, ws = _product(m, k, n, "int8", m)
        r = torch.randn(m, n, device="cuda")
        want = dense.linear(x, w, residual=r, x_scale=xs, weight_scale=ws, out_dtype=torch.float32)
        buf = r.clone()
        got = dense.linear(x, w, residual=buf, x_scale=xs, weight_scale=ws, out=buf)
        assert got is buf and torch.equal(buf, want)
        x, w, _, _ = _product(m, k, n, "bf16", m)
        assert torch.equal(dense.linear(x, w), dense.linear(x, w))


@gpu
def test_refusals_of_tensors(cuda_lib):
    import torch

    from flashnext_b200 import dense

    dev = {"device": "cuda"}
    x = torch.zeros(4, 64, dtype=torch.bfloat16, **dev)
    w = torch.zeros(8, 64, dtype=torch.bfloat16, **dev)
    q, s4, s8 = torch.zeros(4, 64, dtype=torch.int8, **dev), torch.ones(4, **dev), torch.ones(8, **dev)
    wq = torch.zeros(8, 64, dtype=torch.int8, **dev)
    for call in (lambda: dense.linear(x.t(), w), lambda: dense.linear(x[:, :60], w), lambda: dense.linear(x, w, activation="tanh"),
                 lambda: dense.linear(x[0], w), lambda: dense.linear(x[:1].expand(4, 64), w),
                 lambda: dense.linear(q, wq), lambda: dense.linear(q, wq, x_scale=s8, weight_scale=s8),
                 lambda: dense.linear(q, wq, x_scale=s4, weight_scale=s4), lambda: dense.linear(x, w, x_scale=s4),
                 lambda: dense.linear(x, w, bias=s4), lambda: dense.linear(x, w, residual=x),
                 lambda: dense.linear(x, w, out=torch.zeros(4, 9, **dev)),
                 lambda: dense.linear(x[:, 1:], w[:, 1:]), lambda: dense.linear(x[:, :63].contiguous(), w[:, :63].contiguous()),
                 lambda: dense.add_rms_norm(x, s8), lambda: dense.add_rms_norm(x, x[0], x[:3]),
                 lambda: dense.add_rms_norm(x, x[0], keep=False), lambda: dense.add_rms_norm(x, x[0], eps=-1.0),
                 lambda: dense.add_rms_norm(x, x[0], residual_out=x), lambda: dense.add_rms_norm(x.t(), x[0, :4]),
                 lambda: dense.quantize_rows(torch.zeros(1, 16385, **dev)), lambda: dense.dequantize_rows(q, s8),
                 lambda: dense.dequantize_rows(q[:, ::2], s4)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: dense.linear(x, w, bias=torch.zeros(8, dtype=torch.float16, **dev)), lambda: dense.linear(x, w.cpu()),
                 lambda: dense.linear(x, w, out_dtype=torch.float16), lambda: dense.linear(x, wq),
                 lambda: dense.add_rms_norm(x, x[0], codes=torch.uint8), lambda: dense.quantize_rows(x, None),
                 lambda: dense.add_rms_norm(x, x[0], x.half()), lambda: dense.dequantize_rows(q, s4.double())):
        with pytest.raises(TypeError):
            call()


@gpu
def test_empty_calls(cuda_lib):
    import torch

    from flashnext_b200 import dense

    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    assert dense.linear(x, w).shape == (0, 8)
    r = dense.add_rms_norm(x, w[0], x, codes=torch.int8, keep=True)
    assert r.y.shape == r.residual.shape == r.codes.shape == (0, 64) and r.scales.shape == (0,)
    assert dense.dequantize_rows(r.codes, r.scales).shape == (0, 64)


@gpu
def test_other_streams_and_graphs(cuda_lib):
    """A norm, an 8-bit product and a bfloat16 one in order on a side stream and in two graphs that replay in turn."""
    import torch

    from flashnext_b200 import dense

    g = _gen(9)
    w1 = torch.ones(512, device="cuda")
    wq, ws = dense.quantize_rows(torch.randn(768, 512, device="cuda", generator=g))
    w2 = torch.randn(512, 768, device="cuda", generator=g).bfloat16()

    def step(x):
        n = dense.add_rms_norm(x, w1, codes=torch.int8)
        h = dense.linear(n.codes, wq, activation="silu", x_scale=n.scales, weight_scale=ws)
        return dense.linear(h, w2, residual=x, out_dtype=torch.bfloat16)

    xs = [torch.randn(m, 512, device="cuda", generator=g).bfloat16() for m in (3, 200)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x, y in zip(xs, want):
            assert torch.equal(step(x), y)
    graphs = []
    for x in xs:
        gr, held = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(gr):
            out = step(held)
        graphs.append((gr, held, out))
    for _ in range(3):
        for (gr, held, out), x, y in zip(graphs, xs, want):
            held.copy_(x)
            gr.replay()
            assert torch.equal(out, y)
            held.zero_()
            gr.replay()
            assert not torch.equal(out, y)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 65])
def test_weights_that_are_not_finite_show_in_the_scales(cuda_lib, kind, dim):
    import torch

    from flashnext_b200 import dense

    x = torch.randn(400, dim, device="cuda")
    for bad in (float("nan"), float("inf"), -float("inf")):
        w = torch.ones(dim, device="cuda")
        w[dim - 2] = bad
        r = dense.add_rms_norm(x, w, codes=_types()[kind], keep=True)
        assert torch.isnan(r.scales).all() and (r.codes.float() == 0).all() and not torch.isfinite(r.y[:, dim - 2]).any()


def test_outputs_that_overlap_inputs_are_refused():
    lib = _lib.load()
    a = _lib.FnLinearArgs(_lib.ABI_VERSION, _lib.LINEAR_BF16, 4, 64, 64, 0, 0, 0, 0, 0, 0x1000, 64, 0x2000, 64, None, None,
                          None, 0x8000, 64, 0x9000)
    run = lambda **kw: lib.fnmoe_linear(ctypes.byref(_set(a, **kw)), None)  # noqa: E731
    # x, the weight, a residual one row on, a residual of another type or stride in the same place
    for kw in ({"out": 0x1000}, {"out": 0x11F0}, {"out": 0x2100}, {"residual": 0x9080}, {"residual": 0x8FF0},
               {"residual": 0x9000, "residual_dtype": 1}, {"residual": 0x9000, "residual_stride": 72}):
        assert run(**kw) == _lib.ERR_VALUE, kw
        assert "overlap" in _lib.last_error(lib)
    n = _lib.FnNormArgs(_lib.ABI_VERSION, 0, 4, 64, 0, 0, 0, 0, 1e-6, 0, 0x10000, 64, 0x20000, 64, 0x30000, 0x40000, 0x50000,
                        0x60000, 0x70000)
    run = lambda **kw: lib.fnmoe_add_rms_norm(ctypes.byref(_set(n, **kw)), None)  # noqa: E731
    for kw in ({"residual_out": 0x20080}, {"residual_out": 0x10080}, {"y": 0x20100}, {"y": 0x10002}, {"codes": 0x10000},
               {"y": 0x50000}, {"codes": 0x40010}, {"scales": 0x60000}, {"y": 0x30000},
               {"residual_out": 0x20000, "residual_stride": 72}, {"y": 0x10000, "x_stride": 72}):
        assert run(**kw) == _lib.ERR_VALUE, kw
        assert "overlap" in _lib.last_error(lib)


def test_int8_widths_whose_sums_pass_32_bits_are_refused():
    """128^2 x 131072 is 2^31: rows of -128, which no quantiser here makes, would wrap."""
    lib = _lib.load()
    a = _lib.FnLinearArgs(_lib.ABI_VERSION, _lib.LINEAR_INT8, 1, 131072, 1, 0, 0, 0, 0, 0, 0x100000, 131072, 0x200000, 131072,
                          0x1000, 0x2000, None, None, 0, 0x3000)
    assert lib.fnmoe_linear(ctypes.byref(a), None) == _lib.ERR_SHAPE


@gpu
@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("dim", [*range(1, 42), 252, 253, 255, 1021, 2053, 2559, 4101, 8189, 16373, 16375, 16376])
def test_norm_of_contiguous_rows_of_any_width(cuda_lib, rows, dim):
    """Rows laid end to end start at every offset from a boundary of eight and end at every other."""
    import torch

    from flashnext_b200 import dense

    if rows * dim > 2_000_000:
        rows = 17
    t, g = _types(), _gen(dim)
    w = torch.randn(dim, device="cuda", generator=g)
    for xd, rd in (("bf16", None), ("f32", None), ("bf16", "bf16"), ("f32", "bf16")):
        x = torch.randn(rows, dim, device="cuda", generator=g).to(t[xd])
        res = None if rd is None else torch.randn(rows, dim, device="cuda", generator=g).to(t[rd])
        got = dense.add_rms_norm(x, w, res, 1e-5, codes=torch.int8, keep=True)
        y, s = od.add_rms_norm(_np(x), _np(w), None if res is None else _np(res), 1e-5)
        assert (np.abs(_np(got.y) - y) <= np.abs(y) * (HALF[xd] + 2.0 ** -18) + 1e-37).all()
        if rd:
            assert (np.abs(_np(got.residual) - s) <= np.abs(s) * (HALF[rd] + 2.0 ** -23) + 1e-37).all()
        _held(got.codes, got.scales, y, "int8")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,dim,pad", [(3, 4096, 0), (3, 4097, 0), (5, 4096, 3), (700, 4096, 0), (700, 1027, 1)])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 2.0 ** -79])
def test_weights_whose_products_leave_the_normal_range(cuda_lib, kind, rows, dim, pad, eps):
    """Rows and weights whose products are subnormal, or 0, although y is not."""
    import torch

    from flashnext_b200 import dense

    g = _gen(dim + rows)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    sign = lambda *s: torch.where(rand(*s) < 0.5, -1.0, 1.0)  # noqa: E731
    for size, small in ((2.0 ** -45, 2.0 ** -100), (2.0 ** -41, 2.0 ** -98), (2.0 ** -30, 2.0 ** -110), (1.0, 2.0 ** -104)):
        x = _cut((1 + rand(rows, dim)) * sign(rows, dim) * size, pad)
        w = (1 + rand(dim)) * small
        got = dense.add_rms_norm(x, w, None, eps, codes=_types()[kind], keep=True)
        y, _ = od.add_rms_norm(_np(x), _np(w), None, float(np.float32(eps)))
        assert (np.abs(_np(got.y) - y) <= np.abs(y) * 2.0 ** -17 + 2.0 ** -140).all()
        _held(got.codes, got.scales, y, kind)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,dim", [(2, 64), (3, 65), (600, 2048)])
@pytest.mark.parametrize("size", [1.5, 1e-20, 3e38])
def test_weights_next_to_the_largest_float(cuda_lib, kind, rows, dim, size):
    """y is finite although a row's own values times the weight are not."""
    import torch

    from flashnext_b200 import dense

    g = _gen(dim + rows)
    x = (1.0 - 2.0 ** -10 * torch.rand(rows, dim, device="cuda", generator=g)) * size
    w = torch.full((dim,), 3.3e38, device="cuda")
    got = dense.add_rms_norm(x, w, None, 0.0, codes=_types()[kind], keep=True)
    y, _ = od.add_rms_norm(_np(x), _np(w), None, 0.0)
    assert (np.abs(_np(got.y) - y) <= np.abs(y) * 2.0 ** -17).all()
    _held(got.codes, got.scales, y, kind)


def test_values_that_overlap_codes_or_scales_are_refused():
    lib = _lib.load()
    a = _lib.FnRowCodesArgs(_lib.ABI_VERSION, 4, 64, 0, 0, 0, 0x1000, 0x2000, 0x3000)
    run = lambda **kw: lib.fnmoe_dequantize_rows(ctypes.byref(_set(a, **kw)), None)  # noqa: E731
    # 256 codes, 16 bytes of scales, 512 or 1024 bytes of values
    for kw in ({"out": 0x1000}, {"out": 0x10FE}, {"out": 0xE02}, {"out": 0xC04, "out_dtype": 1}, {"out": 0x2000},
               {"out": 0x200E}, {"out": 0x1E02}, {"out": 0x1C04, "out_dtype": 1}):
        assert run(**kw) == _lib.ERR_VALUE, kw
        assert "overlap" in _lib.last_error(lib)


@gpu
def test_values_out_and_out_dtype_have_to_agree(cuda_lib):
    import torch

    from flashnext_b200 import dense

    codes, scales = dense.quantize_rows(torch.randn(3, 48, device="cuda"))
    out = torch.empty(3, 48, device="cuda")
    for call in (dense.dequantize_rows, lambda *a, **kw: dense.dequantize_rows(a[0].float().to(torch.float8_e4m3fn), *a[1:], **kw)):
        with pytest.raises(TypeError):
            call(codes, scales, torch.bfloat16, out)
        with pytest.raises(TypeError):
            call(codes, scales, out_dtype=torch.float32, out=out.bfloat16())
        assert call(codes, scales, torch.float32, out) is out
        assert call(codes, scales).dtype is torch.bfloat16 and call(codes, scales, out=out).dtype is torch.float32
    buf = torch.zeros(3 * 48 * 4, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError):  # values over their own codes
        dense.dequantize_rows(buf[:144].view(3, 48), scales, out=buf.view(torch.float32).view(3, 48))


@gpu
def test_gelu_of_large_negative_values(cuda_lib):
    """bfloat16 results: erfc to 2^-12 of itself, its exponential and quotient to 2^-13 (-v^2 / 2 down to -84.5, twice
    rounded), then half a step of bfloat16."""
    import torch

    from flashnext_b200 import dense

    v = -torch.arange(0, 1664, device="cuda").float() / 128
    v = v.bfloat16().unique()
    w = torch.zeros(v.numel(), 16, dtype=torch.bfloat16, device="cuda")
    w[:, 3] = v
    for rows in (3, 300):
        x = torch.zeros(rows, 16, dtype=torch.bfloat16, device="cuda")
        x[:, 3] = 1.0
        got = dense.linear(x, w, activation="gelu")
        want, _ = od.linear(_np(x), _np(w), None, "gelu")
        assert (np.abs(_np(got) - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -11) + 1e-37).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,dim,pad", [(3, 512, 0), (3, 513, 0), (4, 512, 3), (700, 512, 0), (3, 1, 0)])
def test_norm_where_eps_is_far_above_the_squares(cuda_lib, kind, rows, dim, pad):
    """s / sqrt(eps) is subnormal, or 0, and the weight large: y and its codes are not; rows of zeros among them."""
    import torch

    from flashnext_b200 import dense

    g = _gen(dim + rows)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    for size, large, eps in ((2.0 ** -119, 2.0 ** 59, 7e14), (2.0 ** -90, 2.0 ** 97, 2e25), (2.0 ** -130, 2.0 ** 110, 1e-6),
                             (2.0 ** -140, 2.0 ** 120, 1e38), (2.0 ** -130, 1.0, 1e-20), (2.0 ** -130, 2.0 ** 110, 0.0),
                             (2.0 ** -60, 2.0 ** 126, 3e38), (2.0 ** -148, 2.0 ** -100, 0.0)):
        x = (1 + rand(rows, dim)) * torch.where(rand(rows, dim) < 0.5, -size, size)
        if eps:
            x[1] = 0.0
        x, w = _cut(x, pad), (1 + rand(dim)) * large
        got = dense.add_rms_norm(x, w, None, eps, codes=_types()[kind], keep=True)
        y, _ = od.add_rms_norm(_np(x), _np(w), None, float(np.float32(eps)))
        bound = np.abs(y) * 2.0 ** -17 + 2.0 ** -140
        bad = np.isfinite(_np(got.y)) != (np.abs(y) < 2.0 ** 128)
        live = (np.abs(y) < 2.0 ** 127.99).all(1)
        assert not bad[live].any() and (np.abs(_np(got.y) - y) <= bound)[live].all()
        _held(got.codes[torch.from_numpy(live).cuda()], got.scales[torch.from_numpy(live).cuda()], y[live], kind)


@gpu
@pytest.mark.parametrize("dim", [10209, 10247, 12209, 12215, 12217, 12250, 12279, 12281, 12287, 12289])
def test_norm_of_widths_whose_weights_nearly_fill_48_kb(cuda_lib, dim):
    """The weights that lie in shared memory and the kernel's own variables there pass 48 KB together."""
    import torch

    from flashnext_b200 import dense

    w = 1 + 0.1 * torch.randn(dim, device="cuda", generator=_gen(dim))
    for rows, pad in ((3, 0), (3, 1), (400, 0), (400, 1)):
        x = _cut(torch.randn(rows, dim, device="cuda", generator=_gen(rows)), pad)
        y, _ = od.add_rms_norm(_np(x), _np(w))
        assert (np.abs(_np(dense.add_rms_norm(x, w).y) - y) <= np.abs(y) * (HALF["f32"] + 2.0 ** -18) + 1e-37).all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("m,k,n,rpad", [(3000, 528, 2100, 0), (5000, 2064, 1003, 5), (4000, 144, 2050, 1)])
def test_linear_float32_results_of_several_items_a_pair(cuda_lib, kind, m, k, n, rpad):
    """Chunks summed in registers, with accumulators and ring handed from item to item across a pair of CTAs."""
    import torch

    g = _gen(m + n)
    res = _cut(torch.randn(m, n, device="cuda", generator=g), rpad)
    x, w, xs, ws = _product(m, k, n, kind, m)
    got = _check_linear(x, w, xs, ws, kind, "f32", None, "silu", res)
    assert torch.equal(_check_linear(x, w, xs, ws, kind, "f32", None, "silu", res), got)


@gpu
@pytest.mark.parametrize("rows,dim,pad,at", [(297, 513, 3, 1), (1200, 100, 1, 0), (700, 1027, 5, 3), (320, 2560, 1, 1),
                                             (300, 4099, 2, 0), (297, 8200, 1, 1), (301, 15001, 3, 2)])
@pytest.mark.parametrize("xd,rd,kind", [("bf16", None, "int8"), ("bf16", "bf16", "e4m3"), ("f32", None, "e4m3"),
                                        ("f32", "f32", "int8"), ("bf16", "f32", None)])
def test_norm_of_many_rows_off_boundaries(cuda_lib, rows, dim, pad, at, xd, rd, kind):
    """Padded rows that start at any value, enough of them for a thread to hold several chunks of a row."""
    import torch

    from flashnext_b200 import dense

    t, g = _types(), _gen(rows + dim)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = _cut(randn(rows, dim).to(t[xd]), pad, at)
    res = None if rd is None else _cut(randn(rows, dim).to(t[rd]), pad, at)
    w = (1 + 0.3 * randn(dim)).bfloat16()
    got = dense.add_rms_norm(x, w, res, 1e-5, codes=None if kind is None else t[kind], keep=True)
    y, s = od.add_rms_norm(_np(x), _np(w), None if res is None else _np(res), 1e-5)
    assert (np.abs(_np(got.y) - y) <= np.abs(y) * (HALF[xd] + 2.0 ** -18) + 1e-37).all()
    if rd:
        assert (np.abs(_np(got.residual) - s) <= np.abs(s) * (HALF[rd] + 2.0 ** -23) + 1e-37).all()
    if kind:
        _held(got.codes, got.scales, y, kind)
        codes, scales = dense.quantize_rows(x, t[kind])
        _held(codes, scales, _np(x), kind)


@gpu
def test_products_of_four_threads_at_once(cuda_lib):
    """A split by clusters, tiles of one CTA and pairs side by side on streams of their own."""
    import threading

    import torch

    from flashnext_b200 import dense

    def job(m, k, n, kind):
        x, w, xs, ws = _product(m, k, n, kind, m)
        return lambda: dense.linear(x, w, x_scale=xs, weight_scale=ws, out_dtype=torch.float32)

    jobs = [job(3, 2048, 1024, "bf16"), job(64, 512, 20000, "int8"), job(700, 1024, 2100, "e4m3"), job(300, 528, 1000, "bf16")]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(jobs)), []

    def work(j, out):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(40):
                    got = [j() for _ in range(25)]
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(g, out) for g in got):
                        wrong.append("another result")
        except Exception as e:  # noqa: BLE001
            wrong.append(str(e))

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for a in threads:
        a.start()
    for a in threads:
        a.join()
    assert not wrong
    assert _lib.read_device_errors() == 0
