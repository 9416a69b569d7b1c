"""Every form of the real-valued products under forced plans: 16-bit results with residuals, and activations against 64 bits.

The forms: few rows on warp-level MMAs; a CTA per tile, K over a cluster, pairs of SMs on tcgen05, each with an epilogue for 16-bit results
(turned through shared memory) and one for fp32 results, the cluster's its own for both."""
import contextlib
import math

import pytest
import torch

from tcbnn_b200 import lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FORMS = [(16, 1), (48, 1), (80, 1), (144, 1), (208, 1), (256, 1), (16, 2), (48, 2), (96, 4), (128, 8), (240, 4), (32, -2), (96, -2), (160, -2), (256, -2)]


@contextlib.contextmanager
def plan(cols, splits):
    ops.set_linear_plan(cols, splits)
    try:
        yield
        assert ops.linear_status() == 0
    finally:
        ops.set_linear_plan()


def exists(packed, cols, splits):
    return not packed or (splits != -2 and (splits == 1 or cols <= 128))


def whole(g, shape, most, dtype, cuda):
    return torch.randint(-most, most + 1, shape, generator=g, device=cuda).to(dtype)


@pytest.mark.parametrize("packed,cols,splits", [(p, c, s) for p in (False, True) for c, s in FORMS if exists(p, c, s)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,N,K", [(1, 128, 64), (300, 700, 200), (530, 1301, 520), (40, 129, 640), (2000, 3000, 72), (16, 30000, 64)])
def test_16_bit_results_of_every_form(cuda, packed, cols, splits, dtype, M, N, K):
    """Whole numbers, every sum below 2^11 in magnitude and so exact in either type in any order: results are compared for equality.
    Rows of the result and of the residual on 16 bytes, and not; in place."""
    g = torch.Generator(device=cuda)
    g.manual_seed(M + N + K)
    x = whole(g, (M, K), 1, dtype, cuda)
    if packed:
        w = torch.randint(-2 ** 31, 2 ** 31, (N, ops.step128_words(K)), generator=g, device=cuda).to(torch.int32)
        k = torch.arange(K, device=cuda)
        w32 = (w[:, k // 32] >> (31 - k % 32) & 1).float() * 2 - 1
        call = lambda **kw: ops.bit_linear(x, w, None, bias, "relu", **kw)  # noqa: E731
    else:
        w = whole(g, (N, K), 1, dtype, cuda)
        w32 = w.float()
        call = lambda **kw: ops.linear(x, w, bias, "relu", **kw)  # noqa: E731
    bias = whole(g, (N,), 50, FP32, cuda)
    want32 = (x.float() @ w32.t() + bias).clamp(min=0)
    pad = (-N) % 8
    for width, first in ((N + pad, 0), (N + pad + 3, 1)):
        buf = whole(g, (M, width), 100, dtype, cuda)
        res = buf[:, first:first + N]
        want = (want32 + res.float()).to(dtype)
        rest = buf.clone()
        with plan(cols, splits):
            got = call(residual=res)
            assert torch.equal(got, want)
            call(residual=res, out=res)
        rest[:, first:first + N] = want
        assert torch.equal(buf, rest)


def steps(z, name, short):
    """(value in 64 bits, what its fp32 evaluation may be off by relative to it), in units of u = 2^-24, a rounding's half step.
    silu and gelu_tanh, z / (1 + e^-v): expf 2 ulp = 4 u, the quick division 2 ulp = 4 u, a sum and a product 1 u each; gelu_tanh's exponent v of
    six roundings, which weigh |v|.  gelu, z e^(-z^2/2) Q: polynomial 5 u, its 1 / (1 + k|z|) 2 u, expf 4 u, three products 3 u; the
    exponent's rounding weighs z^2 / 2.  Short forms: __expf is off by 2 + 1.173 |v| ulp; gelu's polynomial by 68 u, the exponential by 4 u, its
    exponent by 2.5 u."""
    z = z.double()
    v = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    if name == "gelu":
        want, off = z * 0.5 * torch.special.erfc(-z / math.sqrt(2)), 77 + 1.25 * z * z if short else 14 + 0.5 * z * z
        off = torch.where(z > 0, 80 if short else 16, off)             # (1 - q, and q at most 1/2)
    else:
        e = z if name == "silu" else v
        want, off = z * torch.sigmoid(e), 10 + (0 if name == "silu" else 6) * e.abs() + (2.4 * e.abs() if short else 0)
        off = torch.where(z > 0, 10 + off * torch.exp(-e.abs()), off)   # (what e^-|v| is off by counts as far as that does against 1)
    return want, off * 2.0 ** -24


Z = torch.cat([torch.linspace(-14, 14, 4001), torch.tensor([0.0, -0.0]), torch.logspace(-30, -1, 40), -torch.logspace(-30, -1, 40),
               torch.linspace(-100, -14, 200), torch.linspace(14, 100, 20), torch.tensor([-1e4, -1e13, -1e30, 1e4, 1e13, 1e30])]).float()


@pytest.mark.parametrize("packed,cols,splits", [(p, c, s) for p in (False, True) for c, s in [(0, 0), (48, 1), (256, 1), (32, 4), (64, -2)] if exists(p, c, s)])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (FP16, FP16), (BF16, FP32)])
def test_activations_of_every_form(cuda, packed, cols, splits, name, dtype, out):
    """z is the bias: sums are 0.  Relative to the result everywhere, in the far negative tail as well."""
    z = Z.to(cuda)
    M, N, K = (3 if not cols else 70), len(Z), 64
    x = torch.zeros((M, K), dtype=dtype, device=cuda)
    with plan(cols, splits):
        if packed:
            got = ops.bit_linear(x, torch.zeros((N, 4), dtype=torch.int32, device=cuda), None, z, name, out_dtype=out)
        else:
            got = ops.linear(x, torch.zeros((N, K), dtype=dtype, device=cuda), z, name, out_dtype=out)
    assert torch.equal(got, got[:1].expand_as(got))
    want, off = steps(z, name, short=out != FP32)
    top = torch.finfo(out).max
    far = want.abs() > top                             # (fp16: rounds to infinity)
    assert torch.equal(got[0].double()[far], torch.sign(want[far]) * math.inf)
    least = {FP32: 2.0 ** -126, BF16: 2.0 ** -126, FP16: 2.0 ** -25}[out]           # below the normal numbers: half a step, or none are made
    tol = want.abs() * (off + (0 if out == FP32 else torch.finfo(out).eps / 2 * (1 + off))) + least
    bad = ((got[0].double() - want).abs() > tol) & ~far
    assert not bad.any(), list(zip(z[bad][:5].tolist(), got[0][bad][:5].tolist(), want[bad][:5].tolist()))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("cols,splits", [(0, 0), (48, 1), (32, 4)])
@pytest.mark.parametrize("out", [BF16, FP32])
def test_infinities_and_nan_in_front_of_activations(cuda, packed, cols, splits, out):
    """As the formulas give them: -inf * 0 is NaN."""
    z = torch.tensor([-math.inf, math.inf, math.nan], device=cuda)
    M, K = (3 if not cols else 70), 64
    x = torch.zeros((M, K), dtype=BF16, device=cuda)
    for name, low in (("none", -math.inf), ("relu", 0.0), ("gelu", math.nan), ("gelu_tanh", math.nan), ("silu", math.nan)):
        with plan(cols, splits):
            if packed:
                got = ops.bit_linear(x, torch.zeros((3, 4), dtype=torch.int32, device=cuda), None, z, name, out_dtype=out)
            else:
                got = ops.linear(x, torch.zeros((3, K), dtype=BF16, device=cuda), z, name, out_dtype=out)
        want = torch.tensor([low, math.inf, math.nan], device=cuda).to(out).expand(M, 3)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), name
