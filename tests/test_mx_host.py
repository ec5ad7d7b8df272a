"""The microscaled entry points refuse bad arguments on the host, before any device work, and the oracle of their
formats holds against hand-computed values. No GPU needed."""
from __future__ import annotations

import copy
import io
import pickle

import numpy as np
import pytest
import torch

import oracle.mx as OM
from kernelopt_b200 import _lib
from kernelopt_b200 import kernels as K

A = 4096  # a stand-in for an aligned device pointer: every call below is refused before it is used


@pytest.mark.parametrize("name,args", [
    ("ko_quantize_mx", (A, 0, -1, 64, 64, 0, A, A, None)),                # rows < 0
    ("ko_quantize_mx", (A, 0, 4, 0, 64, 0, A, A, None)),                  # K = 0
    ("ko_quantize_mx", (A, 0, 4, 64, 63, 0, A, A, None)),                 # pitch below the width
    ("ko_quantize_mx", (A, 3, 4, 64, 64, 0, A, A, None)),                 # unknown element type
    ("ko_quantize_mx", (A, 0, 4, 64, 64, 2, A, A, None)),                 # unknown format
    ("ko_quantize_mx", (A + 2, 0, 4, 64, 64, 0, A, A, None)),             # x not aligned to its elements
    ("ko_quantize_mx", (A, 0, 4, 64, 64, 0, A + 8, A, None)),             # codes unaligned
    ("ko_quantize_mx", (A, 0, 4, 64, 64, 0, A, None, None)),              # no scales
    ("ko_quantize_mx", (A, 0, 1 << 31, 1 << 24, 1 << 24, 0, A, A, None)),  # more blocks than a grid holds
    ("ko_dequantize_mx", (A, A, 0, 4, 0, A, 0, None)),                    # K = 0
    ("ko_dequantize_mx", (A, A, 5, 4, 64, A, 0, None)),                   # unknown format
    ("ko_dequantize_mx", (A, A, 0, 4, 64, None, 0, None)),                # no output
    ("ko_dequantize_mx", (A, A + 4, 0, 4, 64, A, 0, None)),               # scales unaligned
    ("ko_pack_weight_mxfp4", (A, 0, 0, 64, A, A, None)),                  # K = 0
    ("ko_pack_weight_mxfp4", (A, 0, 64, 0, A, A, None)),                  # N = 0
    ("ko_pack_weight_mxfp4", (A, 7, 64, 64, A, A, None)),                 # unknown element type
    ("ko_pack_weight_mxfp4", (None, 0, 64, 64, A, A, None)),              # no weight
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, 1e-6, 4, 0, A, A, 0, None, None, None)),      # C = 0
    ("ko_residual_rmsnorm", (A, 1 << 16, A, 1 << 16, None, None, A, 0, 1e-6, 4, 32769, A, A, 0, None, None, None)),
    ("ko_residual_rmsnorm", (A, 63, A, 64, None, None, A, 0, 1e-6, 4, 64, A, A, 0, None, None, None)),     # ldh < C
    ("ko_residual_rmsnorm", (A, 64, A, 63, None, None, A, 0, 1e-6, 4, 64, A, A, 0, None, None, None)),     # ldo < C
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, -1.0, 4, 64, A, A, 0, None, None, None)),     # eps < 0
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, float("nan"), 4, 64, A, A, 0, None, None, None)),
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, None, 0, 1e-6, 4, 64, A, A, 0, None, None, None)),  # no gamma
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, 1e-6, 4, 64, A, A, 0, A, A, None)),           # y and codes
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, 1e-6, 4, 64, A, None, 0, A, None, None)),     # no scales
    ("ko_residual_rmsnorm", (A, 64, A, 64, None, None, A, 0, 1e-6, 4, 64, A, None, 9, A, A, None)),        # format
    ("ko_residual_rmsnorm", (A, 64, None, 0, A, None, A, 0, 1e-6, 4, 64, A, A, 0, None, None, None)),      # bias, no o
    ("ko_residual_rmsnorm", (A, 72, A, 64, None, None, A, 0, 1e-6, 4, 64, A, A, 0, None, None, None)),     # h_out is a
    ("ko_residual_rmsnorm", (A, 64, 2 * A, 64, None, None, A, 0, 1e-6, 4, 64, A + 256, 9 * A, 0, None, None, None)),  # h_out
    ("ko_residual_rmsnorm", (9 * A, 64, A, 65, None, None, A, 0, 1e-6, 4, 64, A, 5 * A, 0, None, None, None)),  # overlaps
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 4, 64, 64, 0, A + 512, 0, None, 0, None, None)),  # out in x
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 4, 64, 64, 0, A - 512, 0, None, 0, None, None)),  # x in out
    ("ko_residual_rmsnorm", (A, 64, A + 1, 64, None, None, A, 1, 1e-6, 4, 64, A, A, 0, None, None, None)),  # strided h
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, -1, 64, 64, 0, A, 0, None, None)),   # M < 0
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, 4, 0, 64, 0, A, 0, None, None)),     # K = 0
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, 4, 64, 0, 0, A, 0, None, None)),     # N = 0
    ("ko_linear_mxfp4", (A, A, 2, A, A, None, 4, 64, 64, 0, A, 0, None, None)),    # unknown format
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, 4, 64, 64, 3, A, 0, None, None)),    # SiLU not offered
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, 4, 64, 64, 0, A, 4, None, None)),    # unknown output type
    ("ko_linear_mxfp4", (A, A, 0, A, None, None, 4, 64, 64, 0, A, 0, None, None)),  # no weight scales
    ("ko_linear_mxfp4", (A + 8, A, 0, A, A, None, 4, 64, 64, 0, A, 0, None, None)),  # codes unaligned
    ("ko_linear_mxfp4", (A, A, 0, A, A, A + 2, 4, 64, 64, 0, A, 0, None, None)),   # bias unaligned
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, 4, 64, 64, 0, A + 1, 1, None, None)),  # out unaligned
    ("ko_linear_mxfp4", (A, A, 0, A + 16, A, None, 4, 64, 64, 0, A, 0, None, None)),  # weight codes not on 32 bytes
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 17, 64, 64, 0, A, 0, None, 0, None, None)),  # no workspace
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 17, 64, 64, 0, A, 0, A, 1599, None, None)),  # too small
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 17, 64, 64, 0, A, 0, A + 8, 9999, None, None)),  # unaligned
    ("ko_linear_quantize_mxfp4", (A, 0, 63, A, A, None, 4, 64, 64, 0, A, 0, None, 0, None, None)),   # pitch < width
    ("ko_linear_quantize_mxfp4", (A, 5, 64, A, A, None, 4, 64, 64, 0, A, 0, None, 0, None, None)),   # element type
    ("ko_linear_quantize_mxfp4", (None, 0, 64, A, A, None, 4, 64, 64, 0, A, 0, None, 0, None, None)),  # no x
    ("ko_linear_quantize_mxfp4", (A + 1, 1, 64, A, A, None, 4, 64, 64, 0, A, 0, None, 0, None, None)),  # x unaligned
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, 4, 64, 64, 9, A, 0, None, 0, None, None)),   # unknown act
])
def test_bad_arguments_are_refused_on_the_host(name, args):
    with pytest.raises(ValueError, match=name):
        _lib.call(name, *args)


@pytest.mark.parametrize("name,args", [
    ("ko_quantize_mx", (None, 0, 0, 64, 64, 0, None, None, None)),
    ("ko_dequantize_mx", (None, None, 0, 0, 64, None, 0, None)),
    ("ko_residual_rmsnorm", (None, 64, None, 0, None, None, None, 0, 1e-6, 0, 64, None, None, 0, None, None, None)),
    ("ko_linear_mxfp4", (None, None, 0, None, None, None, 0, 64, 64, 0, None, 0, None, None)),
])
def test_no_rows_is_no_work(name, args):
    assert _lib.call(name, *args) == _lib.KO_OK


def test_sizes():
    lib = _lib.lib()
    assert lib.ko_mx_codes_bytes(3, 100, _lib.KO_MXFP4) == 3 * 64
    assert lib.ko_mx_codes_bytes(3, 129, _lib.KO_MXFP8) == 3 * 256
    assert lib.ko_mx_scales_bytes(129, 129) == 256 * 8
    assert lib.ko_mx_codes_bytes(3, 0, 0) == lib.ko_mx_codes_bytes(-1, 8, 0) == lib.ko_mx_codes_bytes(3, 8, 2) == -1
    assert lib.ko_linear_quantize_mxfp4_workspace_bytes(16, 64) == 0
    assert lib.ko_linear_quantize_mxfp4_workspace_bytes(17, 64) == 17 * 64 + 128 * 4 == 1600
    assert lib.ko_linear_quantize_mxfp4_workspace_bytes(17, 0) == -1
    assert lib.ko_mx_scales_bytes(-1, 8) == lib.ko_mx_scales_bytes(1, 0) == -1


def test_python_entry_points_refuse_cpu_tensors_and_unknown_names():
    x, w = torch.zeros(4, 64), torch.zeros(64, 8)
    for call in (lambda: K.quantize_mx(x), lambda: K.residual_rmsnorm(x, x, None, None, x[0], 1e-6),
                 lambda: K.rmsnorm(x, x[0], 1e-6), lambda: K.pack_weight_mxfp4(w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="act"):
        K.linear_mxfp4(x, None, act="silu")
    with pytest.raises(ValueError, match="format"):
        K.MXTensor((4, 64), "mxfp6", torch.float32, "cpu")


def test_row_pitch_rules():
    """The pitch of evenly spaced rows, and the refusals, on tensors without a device (the check for CUDA apart)."""
    class Fake(torch.Tensor):
        is_cuda = True

    t = torch.zeros(6, 4, 40).as_subclass(Fake)
    assert K._rows(t, "t") == (24, 40)
    assert K._rows(t[..., 8:], "t") == (24, 40)
    assert K._rows(t[:, :1, 3:7], "t") == (6, 160)
    assert K._rows(t[0, 0, 3:7], "t") == (1, 4)
    assert K._rows(t[:0], "t") == (0, 40)
    assert K._rows(t[..., :1], "t") == (24, 40)
    for bad in (t[:, :3], t.transpose(1, 2), t[..., ::2], t[:1, :1].expand(2, 3, 40), t[0, 0, 0], t[..., :0]):
        with pytest.raises(ValueError):
            K._rows(bad, "t")
    with pytest.raises(ValueError):
        K._rows(t.double(), "t")


def test_calls_go_to_the_device_of_their_tensors(monkeypatch):
    """_call_on launches on the current stream of the tensors' device, and makes that device current for the call only
    where it is not."""
    seen, entered = [], []

    class Guard:
        def __init__(self, device):
            entered.append(device)

        def __enter__(self):
            pass

        def __exit__(self, *exc):
            entered.append("left")

    monkeypatch.setattr(K, "call", lambda name, *args: seen.append((name, args)))
    monkeypatch.setattr(K, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    K._call_on(torch.device("cuda:0"), "f", 1, 2)
    assert seen == [("f", (1, 2, 1000))] and not entered
    K._call_on(torch.device("cuda:1"), "g", 3)
    assert seen[1] == ("g", (3, 1001)) and entered == [torch.device("cuda:1"), "left"]


def test_oracle_against_hand_computed_blocks():
    v = np.zeros((1, 64))
    v[0, :8] = [6, 5, 2.5, 1.75, 0.25, 0.75, -3.5, 7.9]       # ties: 5 -> 4, 2.5 -> 2, 1.75 -> 2, 0.25 -> 0, 0.75 -> 1
    v[0, 32:36] = [2.0 ** -140, -(2.0 ** -128), 0, 2.0 ** -129]
    q = OM.round_trip(v, "mxfp4")
    assert q[0, :8].tolist() == [6, 4, 2, 2, 0, 1, -4, 6]
    assert q[0, 32:36].tolist() == [0, -(2.0 ** -128), 0, 0]
    codes, scales = OM.quantize(v, "mxfp4")
    assert scales.tolist() == [[127, 0, 0, 0]] and codes[0, 6] == 8 + 6
    v[0, :4] = [500, 448, 1.0625, 2.0 ** -9]
    q = OM.round_trip(v, "mxfp8")
    assert q[0, :4].tolist() == [448, 448, 1.0, 2.0 ** -9]    # saturated; 1.0625 is a tie and goes to the even 1
    v[0, 1] = np.inf
    assert np.isnan(OM.round_trip(v, "mxfp8")[0, :32]).all() and np.isfinite(OM.round_trip(v, "mxfp8")[0, 32:]).all()


BIG = 1 << 31
HUGE = 1 << 60  # a pitch whose product with the rows leaves 64 bits


@pytest.mark.parametrize("name,args,why", [
    ("ko_quantize_mx", (A, 0, 16, 64, HUGE, 0, A, A, None), "pitch"),
    ("ko_residual_rmsnorm", (A, HUGE, A, 64, None, None, A, 0, 1e-6, 16, 64, A, A, 0, None, None, None), "pitch"),
    ("ko_residual_rmsnorm", (A, 64, A, HUGE, None, None, A, 0, 1e-6, 16, 64, A, A, 0, None, None, None), "pitch"),
    ("ko_linear_quantize_mxfp4", (A, 0, HUGE, A, A, None, 16, 64, 64, 0, A, 0, None, 0, None, None), "pitch"),
    ("ko_linear_quantize_mxfp4", (A, 0, 64, A, A, None, BIG, 64, BIG, 0, A, 0, A, HUGE, None, None), "tiles"),
    ("ko_linear_mxfp4", (A, A, 0, A, A, None, BIG, 64, BIG, 0, A, 0, None, None), "tiles"),
    ("ko_linear_mxfp4", (A, A, 1, A, A, None, 1 << 30, 64, 1 << 13, 0, A, 0, None, None), "tiles"),
])
def test_sizes_whose_products_leave_the_range_are_refused(name, args, why):
    """Before their extents are compared with anything, and before anything is launched: there is no device here to refuse
    a launch with another reason."""
    with pytest.raises(ValueError, match=why):
        _lib.call(name, *args)


def norm_call(h=A, ldh=64, o=9 * A, ldo=64, bias=None, scale=None, gamma=20 * A, rows=4, c=64, h_out=11 * A, y=13 * A, fmt=0,
              codes=None, scales=None):
    return (h, ldh, o, ldo, bias, scale, gamma, 0, 1e-6, rows, c, h_out, y, fmt, codes, scales, None)


ROW = 64 * 4          # bytes of a row of the calls below


@pytest.mark.parametrize("args", [
    norm_call(y=A + ROW), norm_call(y=A - ROW), norm_call(y=9 * A + ROW), norm_call(y=A + 4),      # shifted over h or o
    norm_call(ldh=72, y=A), norm_call(o=A, ldo=72, h_out=None, y=A),                               # in place of strided rows
    norm_call(y=11 * A), norm_call(y=11 * A + 3 * ROW), norm_call(h_out=A, y=A),                   # over h_out
    norm_call(h_out=20 * A), norm_call(y=20 * A - 4 * ROW + 4), norm_call(bias=13 * A + 64),       # over gamma and bias
    norm_call(scale=11 * A + 4 * ROW - 16),
    norm_call(y=None, codes=A + 512, scales=14 * A), norm_call(y=None, codes=14 * A, scales=9 * A + 16),   # over h, o
    norm_call(y=None, codes=11 * A + 992, scales=14 * A), norm_call(y=None, codes=14 * A, scales=11 * A),  # over h_out
    norm_call(y=None, codes=14 * A, scales=14 * A), norm_call(y=None, fmt=1, codes=14 * A, scales=14 * A + 496),
    norm_call(y=None, codes=20 * A + 240, scales=14 * A),
])
def test_norm_outputs_that_overlap_are_refused(args):
    with pytest.raises(ValueError, match="overlaps"):
        _lib.call("ko_residual_rmsnorm", *args)


@pytest.mark.parametrize("args", [
    norm_call(), norm_call(y=A), norm_call(y=9 * A), norm_call(h_out=A, y=9 * A), norm_call(h_out=9 * A, y=A),
    norm_call(o=A, h_out=None, y=A), norm_call(rows=1, ldh=72, y=A), norm_call(o=None, ldo=0, h_out=None, y=A),
    norm_call(o=None, ldo=1 << 62),
    norm_call(y=A + 4 * ROW), norm_call(y=A - 4 * ROW), norm_call(y=11 * A + 4 * ROW),
    norm_call(y=None, codes=14 * A, scales=14 * A + 256), norm_call(y=None, fmt=1, codes=A + 4 * ROW, scales=A + 4 * ROW + 512),
])
def test_norm_outputs_in_place_or_apart_pass_the_checks(args):
    if torch.cuda.is_available():
        pytest.skip("would launch on made-up addresses")
    with pytest.raises(_lib.KernelError):
        _lib.call("ko_residual_rmsnorm", *args)


def at(i):
    return 16 * A + i * 64 * A      # far from each other, for the small operands below


# x or w 64 x 64 float32 (16384 bytes), its codes 64 x 64 bytes (mxfp4; Kp 128), scales 512 bytes; out 64 x 64 float32
@pytest.mark.parametrize("name,args", [
    ("ko_quantize_mx", (at(0), 0, 64, 64, 64, 0, at(0) + 16368, at(1), None)),                  # codes over x
    ("ko_quantize_mx", (at(0), 0, 64, 64, 64, 0, at(1), at(0) - 496, None)),                    # scales over x
    ("ko_quantize_mx", (at(0), 0, 64, 64, 64, 0, at(1), at(1) + 4080, None)),                   # scales over codes
    ("ko_quantize_mx", (at(0), 0, 64, 64, 128, 1, at(0) + 32256 - 16, at(1), None)),            # codes over strided x's end
    ("ko_dequantize_mx", (at(0), at(1), 0, 64, 64, at(0) + 4092, 0, None)),                     # out over codes
    ("ko_dequantize_mx", (at(0), at(1), 0, 64, 64, at(1) + 508, 0, None)),                      # out over scales
    ("ko_pack_weight_mxfp4", (at(0), 0, 64, 64, at(0) - 4080, at(1), None)),                    # codes over w
    ("ko_pack_weight_mxfp4", (at(0), 0, 64, 64, at(1), at(0) + 16368, None)),                   # scales over w
    ("ko_pack_weight_mxfp4", (at(0), 0, 64, 64, at(1), at(1), None)),                           # scales over codes
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(2), at(3), at(4), 64, 64, 64, 0, at(0) + 4092, 0, None, None)),   # a's codes
    ("ko_linear_mxfp4", (at(0), at(1), 1, at(2), at(3), at(4), 64, 64, 64, 0, at(0) + 8188, 0, None, None)),
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(2), at(3), at(4), 64, 64, 64, 0, at(1) + 508, 0, None, None)),    # a's scales
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(2), at(3), at(4), 64, 64, 64, 0, at(2) - 16380, 0, None, None)),  # weight
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(2), at(3), at(4), 64, 64, 64, 0, at(3), 0, None, None)),
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(2), at(3), at(4), 64, 64, 64, 0, at(4) + 252, 0, None, None)),    # bias
    ("ko_linear_quantize_mxfp4", (at(0), 0, 64, at(2), at(3), at(4), 4, 64, 64, 0, at(2), 0, None, 0, None, None)),
    ("ko_linear_quantize_mxfp4", (at(0), 0, 64, at(2), at(3), at(4), 4, 64, 64, 0, at(3), 0, None, 0, None, None)),
    ("ko_linear_quantize_mxfp4", (at(0), 0, 64, at(2), at(3), at(4), 4, 64, 64, 0, at(4), 0, None, 0, None, None)),
    # 64 rows: a workspace of 4096 + 512 bytes, over x, out, the weight, its scales, the bias
    *[("ko_linear_quantize_mxfp4", (at(0), 0, 64, at(2), at(3), at(4), 64, 64, 64, 0, at(5), 0, at(i) - 4592, 4608, None,
                                    None)) for i in (0, 2, 3, 4, 5)],
])
def test_outputs_that_overlap_operands_are_refused(name, args):
    with pytest.raises(ValueError, match="overlap"):
        _lib.call(name, *args)


@pytest.mark.parametrize("name,args", [
    ("ko_quantize_mx", (at(0), 0, 64, 64, 64, 0, at(0) + 16384, at(0) - 512, None)),
    ("ko_dequantize_mx", (at(0), at(1), 0, 64, 64, at(0) + 4096, 0, None)),
    ("ko_pack_weight_mxfp4", (at(0), 0, 64, 64, at(0) - 4096, at(0) + 16384, None)),
    ("ko_linear_mxfp4", (at(0), at(1), 0, at(0), at(1), None, 64, 64, 64, 0, at(0) + 4096, 0, None, None)),   # x @ x^T
    ("ko_linear_quantize_mxfp4", (at(0), 0, 64, at(2), at(3), at(4), 64, 64, 64, 0, at(5), 0, at(0) - 4608, 4608, None, None)),
])
def test_operands_that_only_touch_pass_the_checks(name, args):
    if torch.cuda.is_available():
        pytest.skip("would launch on made-up addresses")
    with pytest.raises(_lib.KernelError):
        _lib.call(name, *args)


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle", "save"])
@pytest.mark.parametrize("bias", [False, True])
def test_copies_of_a_packed_weight_have_their_own_addresses(monkeypatch, how, bias):
    """A product passes the addresses that the packed weight keeps, so a copy that kept the original's would read memory that
    is freed with the original."""
    monkeypatch.setattr(K, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    pw = K._packed_weight_mx(K.MXTensor((8, 64), "mxfp4", torch.bfloat16, "cpu"), 64, 8, torch.arange(8.0) if bias else None)
    pw.mx.buf.fill_(7)
    if how == "save":
        f = io.BytesIO()
        torch.save(pw, f)
        f.seek(0)
        other = torch.load(f, weights_only=False)
    else:
        other = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda p: pickle.loads(pickle.dumps(p))}[how](pw)
    assert (other.k, other.n, other.mx.fmt, other.mx.shape, other.mx.dtype) == (64, 8, "mxfp4", (8, 64), torch.bfloat16)
    assert torch.equal(other.mx.buf, pw.mx.buf)
    assert other.ptrs == (*other.mx._ptrs(), other.bias.data_ptr() if bias else None)
    assert (other.mx.buf.data_ptr() == pw.mx.buf.data_ptr()) == (how == "copy")
    if bias:
        assert torch.equal(other.bias, pw.bias)
        with pytest.raises(AttributeError):
            pw.bias = torch.zeros(8)
