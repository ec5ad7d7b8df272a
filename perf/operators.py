"""What the microscaled operators compute, and the cases they are measured on.

Microscaled (MX) data: along the reduced axis every 32 consecutive elements share one power of two, 2**e with
e = floor(log2(max |v|)) - emax held to -127 or above, and each element is v / 2**e rounded to the nearest value
of a small float (ties to even, saturating). "mxfp4" has 4-bit e2m1 elements (largest value 6, emax 2), "mxfp8" has
8-bit e4m3 elements (largest 448, emax 8). A block without a finite largest value has the scale NaN.

    norm     h_out = h + (o + bias) * scale, y = h_out / sqrt(mean(h_out^2) + eps) * gamma, y as mxfp8 or as values
    quant    x as mxfp4 / mxfp8 and back to values
    linear   act(q(x) @ q(w) + bias), both sides mxfp4
    block    norm to mxfp8, then act(y @ q(w) + bias) with the weight in mxfp4

`run` with own = False is the plain form in elementary torch operations; with own = True it makes the calls of
kernelopt_b200.kernels.
"""
import math

import torch

own = False

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8}
EPS = 1e-6


def listed():
    """Widths 384 / 1536 and the row counts 25600 / 25664 are the detector backbone's at 16 frames; the others are
    generic transformer sizes."""
    return [
        # one decoding token through the norm in front of a layer
        dict(name="norm_token", op="norm", m=1, k=4096, dtype="bfloat16", fmt="mxfp8", affine=False, slice=False),
        # the backbone's residual stream with bias and layer scale, in its own fp32
        dict(name="norm_frames", op="norm", m=25664, k=384, dtype="float32", fmt="mxfp8", affine=True, slice=False),
        # a long prompt of a wide model
        dict(name="norm_rows", op="norm", m=16384, k=8192, dtype="bfloat16", fmt="mxfp8", affine=False, slice=False),
        # the backbone's fc2 input, checked for what four bits lose
        dict(name="quant_frames", op="quant", m=25600, k=1536, dtype="float32", fmt="mxfp4", slice=False),
        # an odd column slice of a wider projection
        dict(name="quant_ragged", op="quant", m=1203, k=1001, dtype="bfloat16", fmt="mxfp4", slice=True),
        # one decoding token through a square projection: the weight's bytes count
        dict(name="linear_token", op="linear", m=1, k=4096, n=4096, dtype="bfloat16", act="none", slice=False),
        # a decoding batch through a wide projection
        dict(name="linear_batch", op="linear", m=48, k=8192, n=8192, dtype="bfloat16", act="none", slice=False),
        # the backbone's fc1 with its GELU, fp32 in and out
        dict(name="linear_fc1", op="linear", m=25664, k=384, n=1536, dtype="float32", act="gelu", slice=False),
        # sizes that divide by nothing
        dict(name="linear_ragged", op="linear", m=301, k=1000, n=517, dtype="float16", act="relu", slice=True),
        # a long prompt through a square projection of a wide model
        dict(name="linear_rows", op="linear", m=8192, k=8192, n=8192, dtype="bfloat16", act="none", slice=False),
        # four decoding tokens: the norm and the up projection after it
        dict(name="block_token", op="block", m=4, k=4096, n=8192, dtype="float16", act="none", affine=False),
        # a prompt: the same with a GELU
        dict(name="block_rows", op="block", m=8000, k=4096, n=8192, dtype="bfloat16", act="gelu", affine=False),
    ]


def draw(rng):
    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return min(hi, max(lo, n if rng.random() < 0.5 else -(-n // 32) * 32))

    op = rng.choice(["norm", "norm", "quant", "linear", "linear", "block"])
    if op == "norm":
        m, k = size(1, 16384), size(32, 8192)
        return dict(op=op, m=m, k=k, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    fmt=rng.choice(["mxfp8", "none"]), affine=rng.random() < 0.5, slice=rng.random() < 0.25)
    if op == "quant":
        m, k = size(1, 25600), size(32, 4096)
        return dict(op=op, m=m, k=k, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    fmt=rng.choice(["mxfp4", "mxfp8"]), slice=rng.random() < 0.25)
    m, k, n = size(1, 8192), size(32, 8192), size(8, 8192)
    act = rng.choice(["none", "gelu", "relu"])
    if op == "linear":
        return dict(op=op, m=m, k=k, n=n, dtype=rng.choice(["float32", "bfloat16", "float16"]), act=act,
                    slice=rng.random() < 0.25)
    return dict(op=op, m=m, k=k, n=n, dtype=rng.choice(["bfloat16", "float16"]), act=act, affine=rng.random() < 0.5)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    m, k, n = case["m"], case["k"], case.get("n", 0)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rows(width):
        """Activations: channels of different size, a few of them far out, and now and then a padded row of zeros."""
        x = normal(m, width) * torch.exp(0.5 * normal(width)) * (1 + 20 * (normal(width) > 2.5))
        x *= torch.rand((m, 1), generator=g, device="cuda") > 0.02 if m > 8 else 1.0
        return x.to(dt)

    s = dict(case, dt=dt)
    if case["op"] in ("norm", "block"):
        pad = 16 if case.get("slice") else 0
        s["h"], s["o"] = rows(k + pad)[:, pad:], rows(k + pad)[:, :k]
        s["gamma"] = (1 + 0.1 * normal(k)).to(dt)
        s["bias"] = (0.1 * normal(k)).to(dt) if case["affine"] else None
        s["scale"] = (0.5 + 0.1 * normal(k)).to(dt) if case["affine"] else None
    else:
        pad = 24 if case["slice"] else 0
        s["x"] = rows(k + pad)[:, pad:]
    if case["op"] in ("linear", "block"):
        s["w"], s["b"] = (normal(k, n) / math.sqrt(k)).to(dt), (0.1 * normal(n)).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if "w" not in s:
        return s
    w, b = s.pop("w"), s.pop("b")
    if own:  # the weight is laid out once, as a user's program does when it loads its model
        from kernelopt_b200 import kernels as K
        s["weight"] = K.pack_weight_mxfp4(w, b)
    else:    # and so is the plain form's: the values that the 4-bit weight stands for
        s["weight"] = (_values(*_quantize(w.float().t(), "mxfp4")).t().contiguous(), b.float())
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from kernelopt_b200 import kernels as K
    if s["op"] == "quant":
        return K.quantize_mx(s["x"], s["fmt"]).dequantize(s["dt"])
    if s["op"] == "linear":
        return K.linear_mxfp4(s["x"], s["weight"], act=s["act"])
    fmt = "mxfp8" if s["op"] == "block" else s["fmt"]
    h, y = K.residual_rmsnorm(s["h"], s["o"], s["bias"], s["scale"], s["gamma"], EPS,
                              quantize=None if fmt == "none" else fmt)
    if s["op"] == "block":
        return h, K.linear_mxfp4(y, s["weight"], act=s["act"], out_dtype=s["dt"])
    return (h, y) if fmt == "none" else (h, y.codes[:, :s["k"]], y.scales)


# ---- the plain form: 32 bits throughout, rounded once at the end ----
def _pow2(e):
    """2**e for whole -127 <= e <= 127, from the bits: torch.pow and torch.ldexp can be a last place off."""
    return torch.where(e < -126, 2.0 ** -127, ((e.int() + 127) << 23).view(torch.float32))


def _quantize(v, fmt):
    """v [rows, k] -> (elements [rows, k], exponents [rows, ceil(k / 32)]): what each element stands for before its
    block's power of two, NaN in a block whose exponent is NaN."""
    rows, k = v.shape
    nb = -(-k // BLOCK)
    v = torch.nn.functional.pad(v, (0, nb * BLOCK - k)).reshape(rows, nb, BLOCK)
    top = v.abs().amax(-1)
    e = (torch.frexp(top).exponent - 1).float() - EMAX[fmt]
    e = torch.where(top > 0, e.clamp(min=-127), -127.0)
    t = v * _pow2(-e)[..., None]
    mant, emin, most = (1, 0, 6.0) if fmt == "mxfp4" else (3, -6, 448.0)
    step = _pow2((torch.frexp(t).exponent - 1).clamp(min=emin) - mant)
    q = (torch.round(t / step) * step).clamp(-most, most)
    fine = torch.isfinite(top)
    q = torch.where(fine[..., None], q, 0.0)
    return q.reshape(rows, -1)[:, :k], torch.where(fine, e, math.nan)


def _values(q, e):
    k = q.shape[1]
    scale = torch.where(torch.isnan(e), math.nan, _pow2(e.nan_to_num()))
    return q * scale.repeat_interleave(BLOCK, 1)[:, :k]


def _scale_tiles(e, rows):
    """Exponents [rows, ceil(k / 32)] as scales in the products' layout: [row tile of 128][k tile of 128][32][4][4],
    element (i, j, b) of a tile the scale of row 32 j + i and block b, what lies beyond the data 2**-127."""
    tr, tk = -(-rows // 128), -(-e.shape[1] // 4)
    full = torch.full((tr * 128, tk * 4), -127.0, device=e.device)
    full[:rows, :e.shape[1]] = e
    code = torch.where(torch.isnan(full), 255.0, full + 127).to(torch.uint8)
    return code.reshape(tr, 4, 32, tk, 4).permute(0, 3, 2, 1, 4).contiguous().view(torch.float8_e8m0fnu)


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(v / -math.sqrt(2))  # 1 + erf(v / sqrt 2) without its cancellation
    return v.clamp(min=0) if act == "relu" else v


def _linear(x, w, act, dt):
    return _act(x @ w[0] + w[1], act).to(dt)


def _run_plain(s):
    dt = s["dt"]
    if s["op"] == "quant":
        return _values(*_quantize(s["x"].float(), s["fmt"])).to(dt)
    if s["op"] == "linear":
        return _linear(_values(*_quantize(s["x"].float(), "mxfp4")), s["weight"], s["act"], dt)
    o = s["o"].float()
    if s["bias"] is not None:
        o = o + s["bias"].float()
    if s["scale"] is not None:
        o = o * s["scale"].float()
    v = s["h"].float() + o
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["gamma"].float()
    if s["op"] == "block":
        return v.to(dt), _linear(_values(*_quantize(y, "mxfp8")), s["weight"], s["act"], dt)
    if s["fmt"] == "none":
        return v.to(dt), y.to(dt)
    q, e = _quantize(y, s["fmt"])
    return v.to(dt), q.to(torch.float8_e4m3fn), _scale_tiles(e, s["m"])


# ---- work: each input read once, each output written once ----
def work(case):
    m, k, n = case["m"], case["k"], case.get("n", 0)
    size = 4 if case["dtype"] == "float32" else 2
    bits = {"mxfp4": 4.25 / 8, "mxfp8": 8.25 / 8, "none": size}
    weight = n * k * bits["mxfp4"] + n * 4
    if case["op"] == "norm":
        return dict(bytes=m * k * (3 * size + bits[case["fmt"]]) + (3 if case["affine"] else 1) * k * size,
                    flops=8 * m * k)
    if case["op"] == "quant":
        return dict(bytes=m * k * (2 * size + bits[case["fmt"]]), flops=2 * m * k)
    if case["op"] == "linear":
        return dict(bytes=m * k * size + weight + m * n * size, flops=2 * m * n * k)
    return dict(bytes=3 * m * k * size + weight + m * n * size, flops=2 * m * n * k + 8 * m * k)


# ---- the definition in 64 bits, by search in the table of values that an element can have ----
def _table(fmt, device):
    values = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    if fmt == "mxfp8":  # subnormals and the eight steps of 15 binades, without the code of the NaN
        values = [f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (x - 10) for x in range(1, 16) for f in range(8)]
        values.pop()
    return torch.tensor(values, dtype=torch.float64, device=device)


def _powers(device):
    return torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64, device=device)


def _exact_quantize(v, fmt):
    rows, k = v.shape
    nb = (k + BLOCK - 1) // BLOCK
    blocks = torch.zeros((rows, nb * BLOCK), dtype=torch.float64, device=v.device)
    blocks[:, :k] = v
    blocks = blocks.view(rows, nb, BLOCK)
    top = blocks.abs().max(-1).values
    powers = _powers(v.device)
    # the largest power of two not above `top`, found in the list of them, then emax steps down
    at = torch.searchsorted(powers, top, right=True) - 1
    e = (at - 127 - EMAX[fmt]).clamp(min=-127)
    t = blocks.div_(powers[e + 127][..., None])
    table = _table(fmt, v.device)
    middle = (table[1:] + table[:-1]) / 2
    low = torch.searchsorted(middle, t.abs())                # a tie stays at the lower value
    high = torch.searchsorted(middle, t.abs(), right=True)   # a tie goes to the upper one
    q = table[torch.where(low % 2 == 0, low, high)] * torch.sign(t)
    return q.view(rows, -1)[:, :k], e


def _exact_values(v, fmt):
    q, e = _exact_quantize(v, fmt)
    return q * _powers(v.device)[e + 127].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def exact(case, seed):
    s = _inputs(case, seed)
    d = lambda t: None if t is None else t.double()  # noqa: E731
    act = dict(none=lambda v: v, relu=lambda v: torch.where(v > 0, v, 0.0),
               gelu=lambda v: v * torch.special.ndtr(v))[case.get("act", "none")]

    def product(a):
        return act(a @ _exact_values(d(s["w"]).t().contiguous(), "mxfp4").t() + d(s["b"]))

    if case["op"] == "quant":
        return _exact_values(d(s["x"]), case["fmt"])
    if case["op"] == "linear":
        return product(_exact_values(d(s["x"]), "mxfp4"))
    o = d(s["o"]) + (0 if s["bias"] is None else d(s["bias"]))
    h = d(s["h"]) + o * (1 if s["scale"] is None else d(s["scale"]))
    y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * d(s["gamma"])
    if case["op"] == "block":
        return h, product(_exact_values(y, "mxfp8"))
    if case["fmt"] == "none":
        return h, y
    q, e = _exact_quantize(y, case["fmt"])
    del y
    rows, nb = e.shape
    tiles = torch.full((-(-rows // 128), -(-nb // 4), 32, 4, 4), 2.0 ** -127, dtype=torch.float64, device=q.device)
    r, b = torch.meshgrid(torch.arange(rows, device=q.device), torch.arange(nb, device=q.device), indexing="ij")
    tiles[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = _powers(q.device)[e + 127]
    return h, q, tiles
