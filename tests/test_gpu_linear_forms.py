"""Every form of the real-valued products under forced plans: 16-bit results with residuals, infinities and NaN in front of activations.

The forms: few rows on warp-level MMAs; a CTA per tile, K over a cluster, pairs of SMs on tcgen05, each with an epilogue for 16-bit results
(turned through shared memory) and one for fp32 results, the cluster's its own for both."""
import contextlib
import math

import pytest
import torch

from tcbnn_b200 import ops

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
