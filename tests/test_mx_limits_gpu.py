"""The microscaled operators at the ends of what they take: products that run longer than any one wait of their kernels may,
and norms whose outputs take the place of their inputs."""
from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

from kernelopt_b200 import _lib
from kernelopt_b200 import kernels as K

import test_mx_gpu as T

pytestmark = pytest.mark.gpu


def repeated(mx, rows):
    """mx, 256 rows, as an MXTensor of `rows` rows that hold them over and over."""
    big = K.MXTensor((rows, mx.k), mx.fmt, mx.dtype, mx.device)
    n = rows // 256
    for of in (lambda t: t.codes, lambda t: t.scales):
        small = of(mx).view(torch.uint8)
        of(big).view(torch.uint8).view(n, *small.shape).copy_(small.expand(n, *small.shape))
    return big


def test_product_longer_than_a_wait(cuda):
    """9.0e15 operations, about three seconds: every wait of the kernel has a limit of two, and each covers a tile's work,
    not the product's. Sums of products of -1, 0 and 1 are exact, and rows and columns repeat every 256."""
    m, k, n = 1 << 17, 1 << 18, 1 << 17
    torch.cuda.empty_cache()
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randint(-1, 2, (256, k), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.randint(-1, 2, (k, 256), generator=g, device=cuda).to(torch.bfloat16)
    want = (x.double() @ w.double()).to(torch.bfloat16)
    a, b = repeated(K.quantize_mx(x, "mxfp8"), m), repeated(K.pack_weight_mxfp4(w).mx, n)
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device=cuda)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    _lib.call("ko_linear_mxfp4", *a._ptrs(), _lib.KO_MXFP8, *b._ptrs(), None, m, k, n, _lib.KO_ACT_NONE, out.data_ptr(),
              _lib.KO_BF16, K.status_word(cuda).data_ptr(), torch.cuda.current_stream().cuda_stream)
    end.record()
    K.check_device_status(cuda)
    assert start.elapsed_time(end) > 2000, "the product is too short to show anything"
    for r in range(0, m, 4096):
        assert bool((out[r:r + 4096].view(16, 256, n // 256, 256) == want[None, :, None, :]).all()), r


@pytest.mark.parametrize("dtype,code", [(torch.float32, _lib.KO_F32), (torch.bfloat16, _lib.KO_BF16)])
@pytest.mark.parametrize("rows,c", [(1, 33), (5, 384), (130, 1000), (7, 4096), (3, 16392), (3, 32768)])
def test_norm_output_in_place(cuda, rows, c, dtype, code):
    """y in the place of h or of o, and v in the other's."""
    g = torch.Generator(device=cuda).manual_seed(rows + c)
    h, o = (torch.randn((rows, c), generator=g, device=cuda).to(dtype) for _ in range(2))
    gamma = (1 + 0.1 * torch.randn(c, generator=g, device=cuda)).to(dtype)
    v, y = K.residual_rmsnorm(h, o, None, None, gamma, 1e-6)
    for swap in (False, True):
        a, b = h.clone(), o.clone()
        v_at, y_at = (b, a) if swap else (a, b)
        _lib.call("ko_residual_rmsnorm", a.data_ptr(), c, b.data_ptr(), c, None, None, gamma.data_ptr(), code, 1e-6, rows, c,
                  v_at.data_ptr(), y_at.data_ptr(), 0, None, None, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(v_at, v) and torch.equal(y_at, y)


def test_outputs_over_operands_are_refused(cuda):
    """Through the Python entry points, which take `out` and `h_out` from the caller."""
    x = torch.randn((64, 256), device=cuda)
    pw = K.pack_weight_mxfp4(torch.randn((256, 32), device=cuda), torch.randn(32, device=cuda))
    q = K.quantize_mx(x, "mxfp8")
    over_codes = q.buf.view(torch.uint8).view(-1)[:64 * 32 * 4].view(torch.float32).view(64, 32)
    over_x = x.view(-1)[256 * 64 - 2048:].view(64, 32)
    for a, out in ((q, over_codes), (x, over_x)):
        with pytest.raises(ValueError, match="overlap"):
            K.linear_mxfp4(a, pw, out=out)
    with pytest.raises(ValueError, match="overlap"):
        K.linear_mxfp4(x[:1], pw, out=pw.bias.view(1, 32))
    both = torch.ones(65 * 256, device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        K.residual_rmsnorm(x, x, None, None, both[64 * 256:], 1e-6, h_out=both[256:].view(64, 256))


@pytest.mark.parametrize("m", [1, 40])
def test_a_copied_weight_outlives_the_original(cuda, m):
    g = torch.Generator(device=cuda).manual_seed(9)
    x, w = torch.randn((m, 256), generator=g, device=cuda), torch.randn((256, 200), generator=g, device=cuda)
    pw = K.pack_weight_mxfp4(w, torch.randn(200, generator=g, device=cuda))
    want = K.linear_mxfp4(x, pw)
    other = copy.deepcopy(pw)
    pw.mx.buf.zero_()
    pw.bias.zero_()
    assert torch.equal(K.linear_mxfp4(x, other), want) and not K.linear_mxfp4(x, pw).any()


@pytest.mark.parametrize("m,n", [(2300, 1000), (2300, 1100), (290, 6200), (130, 10300)])
@pytest.mark.parametrize("fmt,k", [("mxfp8", 10400), ("mxfp4", 20700)])
def test_long_k_beside_many_tiles(cuda, fmt, k, m, n):
    """No more tiles than stages of K, with 128 x 128 tiles for one round of the SMs and for more. Sums of products of -1, 0
    and 1 are exact in every form of the product."""
    g = torch.Generator(device=cuda).manual_seed(m + n)
    x = torch.randint(-1, 2, (m, k), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.randint(-1, 2, (k, n), generator=g, device=cuda).to(torch.bfloat16)
    got = K.linear_mxfp4(K.quantize_mx(x, fmt), K.pack_weight_mxfp4(w), out_dtype=torch.float32)
    K.check_device_status(cuda)
    assert torch.equal(got.double(), x.double() @ w.double())


@pytest.mark.parametrize("m", [1, 20, 100])
def test_gelu_below_zero_keeps_its_digits(cuda, m):
    """Relative to the result, reached through the bias of a product of zeros. On [-6, 0) the kernel's erfc is a fit within 3e-5
    of itself times an exponential whose argument, up to 26, is off by two roundings: 26 * 2^-23; the products and the sum
    add less than 2^-20. Beyond -6 it is the value at 6 times that exponential, so too small by 1 - 6 g(6) / (|v| g(|v|))."""
    from scipy.special import erfc

    v = np.concatenate([-np.geomspace(1e-6, 6, 400), -np.linspace(6.01, 13.1, 400)]).astype(np.float32)
    pw = K.pack_weight_mxfp4(torch.ones((64, 800), device=cuda), torch.from_numpy(v).to(cuda))
    got = K.linear_mxfp4(torch.zeros((m, 64), device=cuda), pw, "gelu")
    K.check_device_status(cuda)
    assert bool((got == got[0]).all())
    v = v.astype(np.float64)
    off = got[0].double().cpu().numpy() / (0.5 * v * erfc(-v / np.sqrt(2.0))) - 1
    assert np.abs(off[:400]).max() <= 3e-5 + 26 * 2.0 ** -23 + 2.0 ** -20
    at = lambda x: x * erfc(x / np.sqrt(2.0)) / 2 * np.exp(x * x / 2)  # noqa: E731  |v| g(|v|)
    small = 1 - at(6.0) / at(-v[400:])
    assert small[-1] < 0.026 and np.abs(off[400:] + small).max() <= 3e-5 + 124 * 2.0 ** -23 + 2.0 ** -20


@pytest.mark.parametrize("m", [1, 40, 300, 700])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("ex,ew", [(-126, 126), (126, -126), (127, -126), (-126, 127), (-127, 100), (100, -127), (-133, 60)])
def test_block_scales_at_both_ends(cuda, fmt, m, ex, ew):
    """Products of blocks whose scale bytes are the lowest (0) or near the highest (252 and 246), down to subnormal elements:
    -1, 0 and 1 times 2^ex and 2^ew, whose sums are exact."""
    k, n = 640, 520
    g = torch.Generator(device=cuda).manual_seed(m)
    x = torch.randint(-1, 2, (m, k), generator=g, device=cuda).double()
    w = torch.randint(-1, 2, (k, n), generator=g, device=cuda).double()
    a, b = ((t * 2.0 ** e).to(torch.float32) for t, e in ((x, ex), (w, ew)))
    least = -128 if fmt == "mxfp4" else -136          # the smallest element beside the scale 2^-127
    q, pw = K.quantize_mx(a, fmt), K.pack_weight_mxfp4(b)
    assert int(q.scales.view(torch.uint8).max()) == max(127 + ex - (2 if fmt == "mxfp4" else 8), 0)
    want = (x @ w) * 2.0 ** (ex + ew) if ex >= least else torch.zeros((m, n), dtype=torch.float64, device=cuda)
    assert torch.equal(K.linear_mxfp4(q, pw, out_dtype=torch.float32).double(), want)
    if fmt == "mxfp4":
        assert torch.equal(K.linear_mxfp4(a, pw).double(), want)
    K.check_device_status(cuda)


@pytest.mark.parametrize("m", [1, 40, 700])
def test_a_product_over_the_range_is_infinite(cuda, m):
    x = torch.zeros((m, 256), device=cuda)
    x[:, 7] = 2.0 ** 127
    w = torch.zeros((256, 16), device=cuda)
    w[7, :8], w[7, 8:] = 2.0 ** 3, -2.0 ** 3
    got = K.linear_mxfp4(x, K.pack_weight_mxfp4(w))
    assert bool((got[:, :8] == float("inf")).all()) and bool((got[:, 8:] == -float("inf")).all())


@pytest.mark.parametrize("out", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", T.DTYPES)
@pytest.mark.parametrize("rows,c,affine", [(3, 16385, True), (2, 20001, False), (2, 32767, True)])
def test_norm_of_the_widest_rows_element_by_element(cuda, rows, c, affine, dtype, out):
    args = T.norm_inputs(rows, c, rows + c, dtype, cuda, affine)
    v, dv, y, dy = T.norm_oracle(*args, 1e-6)
    got_v, got_y = K.residual_rmsnorm(*args, 1e-6, quantize=out)
    half, tiny = T.HALF[dtype], T.TINY[dtype]
    assert (np.abs(T.np64(got_v) - v) <= dv + half * (np.abs(v) + dv) + tiny).all(), "v"
    if out is None:
        assert (np.abs(T.np64(got_y) - y) <= dy + half * (np.abs(y) + dy) + tiny).all(), "y"
    else:
        T.check_norm_quantized(got_y, y, dy)


@pytest.mark.parametrize("m", [1, 20, 100])
def test_gelu_next_to_zero_keeps_its_digits(cuda, m):
    """Relative to the result on both sides of zero. There q = erfc / 2 is near 1/2, so an error of |v| times 2.4e-7 in |v| q
    is one of 4.8e-7 at most of the result, at |v| = 1/2 on the negative side of 7.8e-7; the polynomial's twelve steps, of
    partial sums below 0.6, add 12 * 0.6 * 2^-24 to q and the other five roundings 2^-24 of it each, both doubled at zero
    and over 0.31 at |v| = 1/2."""
    from scipy.special import erfc

    v = np.geomspace(1e-30, 0.5, 400)
    v = np.concatenate([v, -v]).astype(np.float32)
    pw = K.pack_weight_mxfp4(torch.ones((64, 800), device=cuda), torch.from_numpy(v).to(cuda))
    got = K.linear_mxfp4(torch.zeros((m, 64), device=cuda), pw, "gelu")
    K.check_device_status(cuda)
    assert bool((got == got[0]).all())
    v = v.astype(np.float64)
    off = got[0].double().cpu().numpy() / (0.5 * v * erfc(-v / np.sqrt(2.0))) - 1
    q = np.minimum(0.5 * erfc(np.abs(v) / np.sqrt(2.0)), 0.5 * erfc(-v / np.sqrt(2.0)))
    assert (np.abs(off) <= (2.4e-7 + (12 * 0.6 + 5) * 2.0 ** -24) / q).all(), np.abs(off).max()
