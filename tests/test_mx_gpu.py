"""Microscaled quantisation, the residual + RMS norm and the mxfp4 products against the float64 oracle.

Tolerances. Quantisation of a given input has one right answer: codes and scales are compared bit for bit.
The norm works in fp32: v takes at most three roundings of its terms, its sum of squares a tree of fp32 additions, so y is
within NORM_REL = 64 * 2^-24 of the exact y plus v's own error; a type's rounding adds half a step. A quantised y is within
half an element's step of the exact one (or at the saturated end) beyond that.
A product's terms are exact in fp32. Each tensor-core step adds 32 or 64 of them to the running sum and may drop what lies
below a last place of the largest term: 2^-22 of the sum of magnitudes S per step covers it with the final additions,
(K / 32 + 8) * 2^-22 * S in all.
"""
from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

import oracle.mx as OM
from kernelopt_b200 import _lib
from kernelopt_b200 import kernels as K

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # a subnormal's step
NORM_REL = 64 * 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
FMTS = ("mxfp4", "mxfp8")


def acts(rows, k, seed, dtype, device):
    """Channels of different size, a few far out, some rows of zeros."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, k)) * np.exp(r.standard_normal(k)) * (1 + 30 * (r.standard_normal(k) > 2.3))
    if rows > 4:
        x[r.integers(0, rows, 2)] = 0
    return torch.from_numpy(x.astype(np.float32)).to(device).to(dtype)


def np64(t):
    return t.detach().double().cpu().numpy()


def codes_of(q):
    """One code per element, and the scale bytes by row, of an MXTensor, its fill included."""
    c = q.codes.view(torch.uint8).cpu().numpy()
    if q.fmt == "mxfp4":
        c = np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)
    return c, q.scales.view(torch.uint8).cpu().numpy()


def check_quantized(q, x64, what=""):
    want_c, want_s = OM.quantize(x64, q.fmt)
    got_c, got_s = codes_of(q)
    assert np.array_equal(got_s, OM.scale_tiles(want_s)), f"{what}: scales"
    sign = 8 if q.fmt == "mxfp4" else 128
    zero = (want_c & (sign - 1)) == 0                   # the sign of a zero is free
    assert np.array_equal(np.where(zero, got_c & (sign - 1), got_c), np.where(zero, 0, want_c)), f"{what}: codes"


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (2, 33), (127, 128), (128, 129), (129, 384), (301, 1001),
                                    (5, 4096), (1000, 200)])
def test_quantize_bit_exact(cuda, rows, k, dtype, fmt):
    x = acts(rows, k, rows * 7 + k, dtype, cuda)
    q = K.quantize_mx(x, fmt)
    assert q.shape == x.shape and q.dtype == dtype and q.fmt == fmt
    check_quantized(q, np64(x), f"{rows}x{k}")
    want = OM.round_trip(np64(x), fmt)
    for out in DTYPES:
        v = q.dequantize(out)
        assert v.dtype == out and v.shape == x.shape
        w = torch.from_numpy(want).to(cuda).to(out)
        assert torch.equal(v, w), f"dequantize to {out}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_every_16_bit_value(cuda, fmt, dtype):
    """All finite patterns, subnormals and both ends included, in blocks of 32 consecutive patterns."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype).to(cuda)
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).reshape(64, 1024)
    check_quantized(K.quantize_mx(x, fmt), np64(x))
    y = x.t().contiguous()                               # the same values beside others of every size
    check_quantized(K.quantize_mx(y, fmt), np64(y))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_and_extremes(cuda, fmt):
    t = OM.TABLE[fmt]
    mid = (t[1:] + t[:-1]) / 2
    for e in (0, 100, -100, -120, 115):
        vals = np.concatenate([t, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), [t[-1] * 1.14]])
        vals = np.concatenate([vals, -vals])
        vals = np.pad(vals, (0, -len(vals) % 31))
        blocks = np.concatenate([vals.reshape(-1, 31), np.full((len(vals) // 31, 1), t[-1])], 1) * 2.0 ** e
        x = torch.from_numpy(blocks.astype(np.float32)).to(cuda)
        check_quantized(K.quantize_mx(x, fmt), np64(x), f"2^{e}")
    x = torch.tensor([[3.4028235e38, -1.0] + [0.0] * 30, [2.0 ** -149] * 32, [-0.0] * 32], device=cuda)
    check_quantized(K.quantize_mx(x, fmt), np64(x), "largest, smallest, zero")


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_not_finite(cuda, fmt):
    x = torch.ones(4, 96, device=cuda)
    x[0, 40], x[1, 5], x[2, 95] = float("nan"), float("inf"), -float("inf")
    q = K.quantize_mx(x, fmt)
    check_quantized(q, np64(x))
    v = q.dequantize()
    bad = torch.zeros(4, 96, dtype=torch.bool, device=cuda)
    bad[0, 32:64], bad[1, :32], bad[2, 64:] = True, True, True
    assert torch.equal(torch.isnan(v), bad) and bool((v[~bad] == 1).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_slices_and_shapes(cuda, dtype):
    wide = acts(60, 300, 3, dtype, cuda)
    for lo, hi in ((0, 128), (8, 264), (1, 130), (7, 300), (299, 300)):
        check_quantized(K.quantize_mx(wide[:, lo:hi]), np64(wide[:, lo:hi]), f"{lo}:{hi}")
    cube = wide.view(3, 20, 300)[:, :, 16:80]
    q = K.quantize_mx(cube)
    assert q.shape == (3, 20, 64) and q.dequantize().shape == (3, 20, 64)
    check_quantized(q, np64(cube).reshape(60, 64))
    assert K.quantize_mx(wide[0, :64]).dequantize().shape == (64,)
    assert K.quantize_mx(wide[:0]).dequantize().shape == (0, 300)
    for bad in (wide.t(), wide[:, ::2], wide[:1].expand(3, 300), wide.double()):
        with pytest.raises(ValueError):
            K.quantize_mx(bad)


# ---- norm ----
def norm_inputs(rows, c, seed, dtype, device, affine):
    h, o = acts(rows, c, seed, dtype, device), acts(rows, c, seed + 1, dtype, device)
    r = np.random.default_rng(seed + 2)
    p = [torch.from_numpy(a.astype(np.float32)).to(device).to(dtype)
         for a in (0.1 * r.standard_normal(c), 0.5 + 0.1 * r.standard_normal(c), 1 + 0.1 * r.standard_normal(c))]
    return h, o, p[0] if affine else None, p[1] if affine else None, p[2]


def norm_oracle(h, o, bias, scale, gamma, eps):
    f = lambda t: None if t is None else np64(t)  # noqa: E731
    v, y = OM.residual_rmsnorm(f(h), f(o), f(bias), f(scale), f(gamma), eps)
    terms = np.abs(f(h))
    if o is not None:
        terms = terms + (np.abs(f(o)) + (0 if bias is None else np.abs(f(bias)))) * (1 if scale is None else np.abs(f(scale)))
    dv = 3 * 2.0 ** -24 * terms                          # v's error before its rounding to the output's type
    rms = np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    with np.errstate(divide="ignore", invalid="ignore"):
        # dv moves y directly and through the mean; the mean's relative move is at most 2 |dv| / |v| in 2-norm
        move = np.linalg.norm(dv, axis=-1, keepdims=True) / (np.sqrt(v.shape[-1]) * rms)
        dy = np.abs(f(gamma)) * dv / rms + np.abs(y) * (move + NORM_REL)
    return v, dv, y, dy


def check_norm_quantized(q, y, dy, what=""):
    fmt, (rows, c) = q.fmt, y.shape
    got_c, got_t = codes_of(q)
    tiles = got_t.transpose(0, 3, 2, 1, 4).reshape(got_t.shape[0] * 128, -1)      # back to [rows, blocks]
    scales = tiles[:rows]
    assert not tiles[rows:].any(), f"{what}: scales of the filling rows"
    _, low = OM.quantize(np.sign(y) * np.maximum(np.abs(y) - dy, 0), fmt)
    _, high = OM.quantize(np.sign(y) * (np.abs(y) + dy), fmt)
    assert ((scales >= low) & (scales <= high)).all(), f"{what}: scales"
    assert not got_c[:, c:].any(), f"{what}: codes beyond the width"
    s = np.repeat(OM.POWERS[scales], 32, axis=1)[:, :c]
    got = OM.values(got_c, scales, fmt, c)
    mant, emin = (1, 0) if fmt == "mxfp4" else (3, -6)
    with np.errstate(divide="ignore"):
        ex = np.maximum(np.floor(np.log2((np.abs(y) + dy) / s)), emin)
    half = np.maximum(2.0 ** (ex - mant) / 2, (np.abs(y) + dy) / s - OM.TABLE[fmt][-1]) * s
    assert (np.abs(got - y) <= half + dy).all(), f"{what}: values"


@pytest.mark.parametrize("out", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,affine", [(1, 1, False), (1, 32, True), (5, 33, True), (130, 384, True),
                                           (17, 385, False), (33, 1000, True), (3, 1024, False), (5, 1025, True),
                                           (9, 2048, False), (4, 4095, True), (2, 4096, False), (3, 8192, True),
                                           (2, 8200, False), (2, 16392, False), (1, 32768, True), (300, 128, False),
                                           (41, 200, True), (6, 256, False), (9, 512, True)])
def test_residual_rmsnorm(cuda, rows, c, affine, dtype, out):
    args = norm_inputs(rows, c, rows + c, dtype, cuda, affine)
    v, dv, y, dy = norm_oracle(*args, 1e-6)
    got_v, got_y = K.residual_rmsnorm(*args, 1e-6, quantize=out)
    half, tiny = HALF[dtype], TINY[dtype]
    assert got_v.dtype == dtype and got_v.shape == args[0].shape
    assert (np.abs(np64(got_v) - v) <= dv + half * (np.abs(v) + dv) + tiny).all(), "v"
    if out is None:
        assert got_y.dtype == dtype
        assert (np.abs(np64(got_y) - y) <= dy + half * (np.abs(y) + dy) + tiny).all(), "y"
    else:
        check_norm_quantized(got_y, y, dy)
    # without the residual
    _, _, y, dy = norm_oracle(args[0], None, None, None, args[4], 1e-6)
    got = K.rmsnorm(args[0], args[4], 1e-6, quantize=out)
    if out is None:
        assert (np.abs(np64(got) - y) <= dy + half * (np.abs(y) + dy) + tiny).all(), "rmsnorm"
    else:
        check_norm_quantized(got, y, dy, "rmsnorm")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rmsnorm_slices_in_place_and_shapes(cuda, dtype):
    wide = acts(40, 700, 5, dtype, cuda)
    gamma = torch.ones(256, dtype=dtype, device=cuda)
    for lo in (0, 8, 3):
        h, o = wide[:, lo:lo + 256], wide[:, 300 + lo:556 + lo]
        a = K.residual_rmsnorm(h, o, None, None, gamma, 1e-5, quantize="mxfp8")
        b = K.residual_rmsnorm(h.contiguous(), o.contiguous(), None, None, gamma, 1e-5, quantize="mxfp8")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1].buf, b[1].buf)
    h = wide[:, :256].contiguous().view(4, 10, 256)
    o = wide[:, 300:556].contiguous().view(4, 10, 256)
    v, y = K.residual_rmsnorm(h, o, None, None, gamma, 1e-5)
    mine = h.clone()
    v2, y2 = K.residual_rmsnorm(mine, o, None, None, gamma, 1e-5, h_out=mine)
    assert v2 is mine and torch.equal(v, v2) and torch.equal(y, y2) and v.shape == (4, 10, 256)
    mine = o.clone()
    v2, y2 = K.residual_rmsnorm(h, mine, None, None, gamma, 1e-5, h_out=mine)
    assert torch.equal(v, v2) and torch.equal(y, y2)
    flat = torch.zeros(12 * 256, dtype=dtype, device=cuda)
    with pytest.raises(ValueError, match="overlaps"):
        K.residual_rmsnorm(flat[:2560].view(10, 256), o[0], None, None, gamma, 1e-5, h_out=flat[256:2816].view(10, 256))
    assert K.rmsnorm(h[:0], gamma, 1e-5).shape == (0, 10, 256)
    assert K.rmsnorm(h[:0], gamma, 1e-5, quantize="mxfp8").shape == (0, 10, 256)


def test_rmsnorm_zero_rows_and_not_finite(cuda):
    x = torch.ones(6, 100, device=cuda)
    x[1] = 0
    x[2, 7], x[3, 99] = float("nan"), float("inf")
    g = torch.ones(100, device=cuda)
    y = K.rmsnorm(x, g, 1e-6)
    assert bool((y[1] == 0).all()) and bool(torch.isnan(y[2]).all())
    assert bool((y[3, :99] == 0).all()) and bool(torch.isnan(y[3, 99]))  # 1 / inf, and inf / inf
    q = K.rmsnorm(x, g, 1e-6, quantize="mxfp8").dequantize()
    assert bool((q[1] == 0).all()) and bool(torch.isnan(q[2]).all())
    assert bool((q[3, :96] == 0).all()) and bool(torch.isnan(q[3, 96:]).all())
    for r in (0, 4, 5):
        # y = (1 + 1e-6)^(-1/2) is below 1, so its block's scale is 2^(-1 - 8), and 511.99 saturates at 448: 0.875
        assert bool((y[r] == y[0]).all()) and bool((q[r] == 0.875).all())
    z = K.rmsnorm(x, g, 0.0, quantize="mxfp8").dequantize()             # eps 0: a row of zeros is 0 * inf
    assert bool(torch.isnan(z[1]).all()) and bool((z[0] == 1).all())


def test_rmsnorm_refusals(cuda):
    h = torch.zeros(4, 64, device=cuda)
    g = torch.ones(64, device=cuda)
    for call in (lambda: K.residual_rmsnorm(h, h[:2], None, None, g, 1e-6),
                 lambda: K.residual_rmsnorm(h, h.bfloat16(), None, None, g, 1e-6),
                 lambda: K.residual_rmsnorm(h, h, g[:3], None, g, 1e-6),
                 lambda: K.residual_rmsnorm(h, h, None, g.half(), g, 1e-6),
                 lambda: K.residual_rmsnorm(h, h, None, None, None, 1e-6),
                 lambda: K.residual_rmsnorm(h, h, None, None, g, 1e-6, quantize="int8"),
                 lambda: K.residual_rmsnorm(h, h, None, None, g, -1e-6),
                 lambda: K.residual_rmsnorm(h, h, None, None, g, 1e-6, h_out=h[:2]),
                 lambda: K.rmsnorm(torch.zeros(2, 32769, device=cuda), torch.ones(32769, device=cuda), 1e-6)):
        with pytest.raises(ValueError):
            call()


# ---- products ----
def weight(k, n, seed, dtype, device):
    r = np.random.default_rng(seed)
    w = torch.from_numpy((r.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)).to(device).to(dtype)
    return w, torch.from_numpy((0.1 * r.standard_normal(n)).astype(np.float32)).to(device).to(dtype)


def check_linear(got, a, w, bias, act, what=""):
    """got against act(a @ w + bias), a [rows, K] and w [K, N] the quantised values in float64."""
    k = a.shape[1]
    s = np.abs(a) @ np.abs(w)
    pre = a @ w + (0 if bias is None else bias)
    d = (k / 32 + 8) * 2.0 ** -22 * (s + (0 if bias is None else np.abs(bias)))
    want = OM.act(pre, act)
    # GELU's slope is at most 1.13. Its own error: erf by A&S 7.1.26 is within 1.5e-7, halved and times |v|; the fp32
    # evaluation of erfc / 2 <= 1/2 is within 2^-20 of itself, so |v| 2^-21
    d = 1.13 * d + (np.abs(pre) * (0.75e-7 + 2.0 ** -21) if act == "gelu" else 0)
    half, tiny = HALF[got.dtype], TINY[got.dtype]
    err = np.abs(np64(got).reshape(want.shape) - want)
    assert (err <= d + half * (np.abs(want) + d) + tiny).all(), \
        f"{what}: off by {np.nanmax(err):.3g}, {np.mean(~(err <= d + half * (np.abs(want) + d) + tiny)):.2%} of the outputs"


SHAPES = [(1, 1, 1), (1, 32, 8), (3, 33, 5), (127, 128, 129), (128, 256, 128), (129, 320, 257), (300, 1000, 517),
          (1, 4096, 1024), (2, 2048, 100), (65, 64, 1024), (16, 512, 384), (9, 8192, 72), (513, 1152, 640),
          (1000, 384, 1536), (1111, 700, 2049), (5001, 300, 2560), (300, 136, 5003), (700, 1300, 2601),
          (2600, 1100, 4704), (700, 96, 8), (2000, 40, 12), (600, 4096, 16), (100, 8192, 260), (90, 512, 1000),
          (1500, 1300, 2051), (1501, 1300, 2056)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_mxfp4(cuda, m, k, n, fmt):
    dtype = DTYPES[(m + k + n) % 3]
    act = (None, "gelu", "relu")[(m + n) % 3]
    x = acts(m, k, m + k, dtype, cuda)
    w, b = weight(k, n, n + k, dtype, cuda)
    with_bias = (m + k) % 2 == 0
    pw = K.pack_weight_mxfp4(w, b if with_bias else None)
    wq = OM.round_trip(np64(w).T, "mxfp4").T
    assert np.array_equal(np64(pw.dequantize()), wq), "packed weight"
    aq = OM.round_trip(np64(x), fmt)
    for out_dtype in DTYPES:
        got = K.linear_mxfp4(K.quantize_mx(x, fmt), pw, act, out_dtype)
        K.check_device_status(cuda)
        assert got.shape == (m, n) and got.dtype == out_dtype
        check_linear(got, aq, wq, np64(b) if with_bias else None, act, f"{m}x{k}x{n} {fmt} {out_dtype}")
    if fmt == "mxfp4":
        a, b2 = K.linear_mxfp4(x, pw, act), K.linear_mxfp4(K.quantize_mx(x), pw, act)
        assert a.dtype == dtype and torch.equal(a, b2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16])
def test_linear_fused_rows(cuda, m, dtype):
    """Up to 16 rows are quantised inside the product's kernel: the same bits as quantising first, for any width, pitch and
    content."""
    for k, n in ((1, 3), (31, 40), (256, 130), (300, 129), (4097, 256), (2048, 1000)):
        wide = acts(m, k + 9, m * k, dtype, cuda)
        w, b = weight(k, n, n + k, dtype, cuda)
        pw = K.pack_weight_mxfp4(w, b)
        for x in (wide[:, :k], wide[:, 8:k + 8], wide[:, 3:k + 3].contiguous()):
            assert torch.equal(K.linear_mxfp4(x, pw, "gelu"), K.linear_mxfp4(K.quantize_mx(x), pw, "gelu")), (k, n)
        x = wide[:, :k].clone()
        x[m // 2, k // 2] = float("nan")
        got, want = K.linear_mxfp4(x, pw), K.linear_mxfp4(K.quantize_mx(x), pw)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(got[m // 2]).all())
        keep = [r for r in range(m) if r != m // 2]
        assert torch.equal(got[keep], want[keep])
    K.check_device_status(cuda)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 40, 200, 600])
def test_linear_rows_do_not_meet(cuda, m, fmt):
    """A row or a weight column that is not finite stays in its own outputs, rows of zeros give the bias, and what lies
    behind the output is left as it was."""
    k, n = 300, 200
    x = acts(m, k, 8, torch.float32, cuda)
    w, b = weight(k, n, 9, torch.float32, cuda)
    base = K.linear_mxfp4(K.quantize_mx(x, fmt), K.pack_weight_mxfp4(w, b))
    w2 = w.clone()
    w2[17, 3], w2[299, 150] = float("nan"), float("inf")
    got = K.linear_mxfp4(K.quantize_mx(x, fmt), K.pack_weight_mxfp4(w2, b))
    cols = torch.zeros(n, dtype=torch.bool, device=cuda)
    cols[3] = cols[150] = True
    assert bool(torch.isnan(got[:, cols]).all()) and torch.equal(got[:, ~cols], base[:, ~cols])
    y = x.clone()
    y[m // 2] = 0
    y[m - 1, 299] = float("nan")
    got = K.linear_mxfp4(K.quantize_mx(y, fmt), K.pack_weight_mxfp4(w, b))
    assert bool(torch.isnan(got[m - 1]).all())
    if m > 2:
        assert torch.equal(got[m // 2], b)
        keep = [r for r in range(m - 1) if r != m // 2]
        assert torch.equal(got[keep], base[keep])
    buf = torch.full((m + 2, n), 7.0, device=cuda)
    K.linear_mxfp4(K.quantize_mx(x, fmt), K.pack_weight_mxfp4(w, b), out=buf[1:m + 1])
    assert torch.equal(buf[1:m + 1], base) and bool((buf[0] == 7).all()) and bool((buf[m + 1] == 7).all())
    K.check_device_status(cuda)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 70, 300])
def test_linear_output_anywhere(cuda, m, dtype):
    """An output that starts on its own element's alignment only, with its neighbours left as they were."""
    k, n = 320, 264
    x = acts(m, k, 3, dtype, cuda)
    w, b = weight(k, n, 4, dtype, cuda)
    pw = K.pack_weight_mxfp4(w, b)
    want = K.linear_mxfp4(x, pw, "relu")
    flat = torch.full((m * n + 9,), 7.0, dtype=dtype, device=cuda)
    for lead in (1, 2, 8):
        flat.fill_(7.0)
        K.linear_mxfp4(x, pw, "relu", out=flat[lead:lead + m * n].view(m, n))
        assert torch.equal(flat[lead:lead + m * n].view(m, n), want)
        assert bool((flat[:lead] == 7).all()) and bool((flat[lead + m * n:] == 7).all())
    x0 = torch.zeros(m, 256, dtype=dtype, device=cuda)
    with pytest.raises(ValueError, match="overlaps"):
        K.linear_mxfp4(x0, K.pack_weight_mxfp4(w[:256, :256].contiguous()), out=x0)
    K.check_device_status(cuda)


def test_gelu_at_the_ends(cuda):
    """Infinities, NaN, and values far on both sides, reached through the bias of a product of zeros."""
    v = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0, 100.0, -100.0, 1e-30, -1e-30, 6.0, -6.0, -5.5, -9.0],
                     device=cuda)
    want = 0.5 * v.double() * torch.special.erfc(-v.double() / 2 ** 0.5)
    for m in (1, 20, 100):
        got = K.linear_mxfp4(torch.zeros(m, 64, device=cuda), K.pack_weight_mxfp4(torch.ones(64, 12, device=cuda), v), "gelu")
        assert bool((got == got[0]).logical_or(torch.isnan(got)).all())
        g = got[0].double()
        assert g[0] == float("inf") and g[1] == 0 and bool(torch.isnan(g[2])) and g[3] == 0
        # |v| q within 8e-8, and q within 3e-5 of itself up to 6; beyond that q is below 1e-9
        assert bool(((g - want)[3:].abs() <= 1e-7 + want[3:].abs() * 2.0 ** -22).all())
        assert bool(((g - want)[9:11].abs() <= want[9:11].abs() * 4e-5).all())


def test_more_than_2_to_the_31_elements(cuda):
    """The last rows of tensors whose offsets pass 32 bits, against the same rows on their own."""
    rows, k = 70001, 32768                                     # 2.3e9 elements
    x = torch.empty((rows, k), dtype=torch.bfloat16, device=cuda)
    x[:-4] = 1
    x[-4:] = acts(4, k, 5, torch.bfloat16, cuda)
    for fmt in FMTS:
        q, part = K.quantize_mx(x, fmt), K.quantize_mx(x[-4:], fmt)
        assert torch.equal(q.codes[-4:].view(torch.uint8), part.codes.view(torch.uint8))
        v = q.dequantize(torch.bfloat16)
        assert torch.equal(v[-4:], part.dequantize(torch.bfloat16)) and bool((v[-5] == 1).all())
        del q, v
    gamma = torch.ones(k, dtype=torch.bfloat16, device=cuda)
    v, y = K.residual_rmsnorm(x, x, None, None, gamma, 1e-6, quantize="mxfp8")
    v4, y4 = K.residual_rmsnorm(x[-4:], x[-4:], None, None, gamma, 1e-6, quantize="mxfp8")
    assert torch.equal(v[-4:], v4) and torch.equal(y.codes[-4:].view(torch.uint8), y4.codes.view(torch.uint8))
    del v, y
    a = acts(rows, 32, 6, torch.bfloat16, cuda)                # sums of 32 terms are exact in every form of the product
    pw = K.pack_weight_mxfp4(weight(32, k, 7, torch.bfloat16, cuda)[0])
    got = K.linear_mxfp4(a, pw)
    assert torch.equal(got[-4:], K.linear_mxfp4(a[-4:], pw)) and torch.equal(got[:4], K.linear_mxfp4(a[:4], pw))
    K.check_device_status(cuda)


@pytest.mark.parametrize("m,k,n", [(1, 4096, 512), (70, 4096, 300), (600, 1024, 512)])
def test_linear_same_result_every_time(cuda, m, k, n):
    x = K.quantize_mx(acts(m, k, 1, torch.bfloat16, cuda))
    w, b = weight(k, n, 2, torch.bfloat16, cuda)
    pw = K.pack_weight_mxfp4(w, b)
    first = K.linear_mxfp4(x, pw, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(K.linear_mxfp4(x, pw, out_dtype=torch.float32), first)
    # a row's result does not depend on the rows beside it where the same kernel form runs
    assert K.linear_mxfp4(acts(0, k, 1, torch.bfloat16, cuda), pw).shape == (0, n)


def test_linear_refusals(cuda):
    x = torch.zeros(4, 64, device=cuda)
    w, b = weight(64, 24, 1, torch.float32, cuda)
    pw = K.pack_weight_mxfp4(w, b)
    for call in (lambda: K.linear_mxfp4(x[:, :32], pw), lambda: K.linear_mxfp4(K.quantize_mx(x[:, :32]), pw),
                 lambda: K.linear_mxfp4(x.cpu(), pw), lambda: K.linear_mxfp4(x, pw, act="silu"),
                 lambda: K.linear_mxfp4(x, pw, out_dtype=torch.float64),
                 lambda: K.linear_mxfp4(x, pw, out=torch.zeros(4, 23, device=cuda)),
                 lambda: K.linear_mxfp4(x, pw, out=torch.zeros(24, 4, device=cuda).t()),
                 lambda: K.pack_weight_mxfp4(w.t()), lambda: K.pack_weight_mxfp4(w, b[:3]),
                 lambda: K.pack_weight_mxfp4(w[:, :0]), lambda: K.pack_weight_mxfp4(w.double())):
        with pytest.raises(ValueError):
            call()


# ---- the operators together ----
@pytest.mark.parametrize("rows", [1, 7, 401])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_run(cuda, dtype, rows):
    """residual + norm -> mxfp8 -> up projection with GELU -> mxfp4 -> down projection, each against the oracle on the
    operands that it was given."""
    c, f = 384, 1536
    h, o, bias, scale, gamma = norm_inputs(rows, c, 31, dtype, cuda, True)
    w1, b1 = weight(c, f, 32, dtype, cuda)
    w2, b2 = weight(f, c, 33, dtype, cuda)
    p1, p2 = K.pack_weight_mxfp4(w1, b1), K.pack_weight_mxfp4(w2, b2)
    v, y = K.residual_rmsnorm(h, o, bias, scale, gamma, 1e-6, quantize="mxfp8")
    m = K.linear_mxfp4(y, p1, "gelu")
    out = K.linear_mxfp4(m, p2)
    K.check_device_status(cuda)
    assert m.dtype == out.dtype == dtype and out.shape == h.shape
    _, _, ey, edy = norm_oracle(h, o, bias, scale, gamma, 1e-6)
    check_norm_quantized(y, ey, edy)
    check_linear(m, np64(y.dequantize()), np64(p1.dequantize()), np64(b1), "gelu", "up")
    check_linear(out, OM.round_trip(np64(m), "mxfp4"), np64(p2.dequantize()), np64(b2), None, "down")


@pytest.mark.parametrize("rows", [5, 50, 700])
def test_streams_threads_and_graphs(cuda, rows):
    """The same results on another stream, from two threads at once, and captured into graphs that run side by side."""
    c, n = 512, 640
    h, o, _, _, gamma = norm_inputs(rows, c, 41, torch.bfloat16, cuda, False)
    w, b = weight(c, n, 42, torch.bfloat16, cuda)
    pw = K.pack_weight_mxfp4(w, b)

    def layer(h, o):
        v, y = K.residual_rmsnorm(h, o, None, None, gamma, 1e-6, quantize="mxfp8")
        return v, K.linear_mxfp4(y, pw, "gelu"), K.linear_mxfp4(v, pw)

    want = layer(h, o)
    h2, o2 = h.flip(0).contiguous(), o.flip(0).contiguous()
    want2 = layer(h2, o2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer(h, o)
    side.synchronize()
    assert all(torch.equal(a, x) for a, x in zip(got, want))

    res = {}

    def work(i, h, o):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                res[i] = layer(h, o)
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work, args=(i, *a)) for i, a in enumerate(((h, o), (h2, o2)))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert all(torch.equal(a, x) for a, x in zip(res[0], want)) and all(torch.equal(a, x) for a, x in zip(res[1], want2))

    graphs, outs, ins = [], [], []
    for _ in range(2):
        hh, oo = h.clone(), o.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(hh, oo))
        graphs.append(g)
        ins.append((hh, oo))
    ins[1][0].copy_(h2)
    ins[1][1].copy_(o2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, x) for a, x in zip(outs[0], want)) and all(torch.equal(a, x) for a, x in zip(outs[1], want2))
    K.check_device_status(cuda)


FIRST_IN_CAPTURE = """
import torch
from kernelopt_b200 import kernels as K
g = torch.cuda.CUDAGraph()
x = torch.randn(ROWS, 512, device="cuda")
pw = K.pack_weight_mxfp4(torch.randn(512, 640, device="cuda"))
gamma = torch.ones(512, device="cuda")
s = torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    v, y = K.residual_rmsnorm(x, x, None, None, gamma, 1e-6, quantize="mxfp8")
    a, b = K.linear_mxfp4(y, pw, "gelu"), K.linear_mxfp4(v, pw)
    d = y.dequantize()
g.replay()
torch.cuda.synchronize()
v2, y2 = K.residual_rmsnorm(x, x, None, None, gamma, 1e-6, quantize="mxfp8")
assert torch.equal(v, v2) and torch.equal(d, y2.dequantize())
assert torch.equal(a, K.linear_mxfp4(y2, pw, "gelu")) and torch.equal(b, K.linear_mxfp4(v2, pw))
K.check_device_status()
print("captured")
"""


@pytest.mark.parametrize("rows", [3, 40, 700])
def test_first_call_inside_a_capture(cuda, rows):
    """A process whose first use of the kernels is being captured."""
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE.replace("ROWS", str(rows))], capture_output=True, text=True,
                       timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_launch_counts(cuda):
    _lib.launch_count.clear()
    x = torch.ones(4, 64, device=cuda)
    pw = K.pack_weight_mxfp4(torch.ones(64, 8, device=cuda))
    K.linear_mxfp4(x, pw)
    K.rmsnorm(x, torch.ones(64, device=cuda), 1e-6, quantize="mxfp8").dequantize()
    K.linear_mxfp4(x.repeat(5, 1), pw)
    K.linear_mxfp4(K.quantize_mx(x), pw)
    assert _lib.launch_count == {"ko_pack_weight_mxfp4": 1, "ko_linear_quantize_mxfp4": 3, "ko_residual_rmsnorm": 1,
                                 "ko_dequantize_mx": 1, "ko_quantize_mx": 1, "ko_linear_mxfp4": 1}
