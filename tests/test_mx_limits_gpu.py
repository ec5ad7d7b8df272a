"""The microscaled operators at the ends of what they take: products that run longer than any one wait of their kernels may."""
from __future__ import annotations

import pytest
import torch

from kernelopt_b200 import _lib
from kernelopt_b200 import kernels as K

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
