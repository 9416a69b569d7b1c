"""Products of real-valued rows (ops.linear, ops.bit_linear) against the formula in 64 bits.

Structure is tested on whole numbers: |x| <= 4, |w| <= 4 (or +-1), K <= 16384, so that every partial sum is a whole number
below 2^24, exact in fp32 in any order.  Bias and residual are whole numbers too; what remains is the one rounding of the
result, which torch makes alike (to nearest even), so that outputs are compared for equality.

Activations: erff, tanhf, expf and the division are a few units in the last place off (2^-24 each), and 1 + erf, 1 + tanh cancel,
so the absolute error is at most |z| 2^-21; the rounding to 16 bits adds eps / 2 of the result."""
import math
import os
import subprocess
import sys

import pytest
import torch

import util
from tcbnn_b200 import lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def whole(g, shape, most, dtype, cuda):
    return torch.randint(-most, most + 1, shape, generator=g).to(dtype).to(cuda)


def gen(*seed):
    g = torch.Generator()
    g.manual_seed(sum(s * 7919 ** i for i, s in enumerate(seed)) % (1 << 60))
    return g


def signs(g, N, K, cuda):
    """(packed words with anything behind element K, +-1 values)"""
    ld = ops.step128_words(K)
    words = torch.randint(-2 ** 31, 2 ** 31, (N, ld), generator=g).to(torch.int32)
    k = torch.arange(K)
    pm = ((words[:, k // 32] >> (31 - k % 32)) & 1).double() * 2 - 1
    return words.to(cuda), pm.to(cuda)


def activation(z, name):
    return {"none": z, "relu": z.clamp(min=0), "silu": z * torch.sigmoid(z), "gelu": z * 0.5 * torch.special.erfc(-z / math.sqrt(2)),
            "gelu_tanh": 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))}[name]


def case(bits, M, N, K, dtype, cuda, seed=0):
    """x, weight, scale (powers of two), bias and the sums in 64 bits."""
    g = gen(M, N, K, int(bits), seed)
    x = whole(g, (M, K), 4, dtype, cuda)
    if bits:
        w, w64 = signs(g, N, K, cuda)
        scale = torch.tensor([0.5, 1.0, 2.0])[torch.randint(0, 3, (N,), generator=g)].to(cuda)
        return x, w, scale, x.double() @ w64.t() * scale.double()
    w = whole(g, (N, K), 4, dtype, cuda)
    return x, w, None, x.double() @ w.double().t()


def product(bits, x, w, scale, *args, **kw):
    return ops.bit_linear(x, w, scale, *args, **kw) if bits else ops.linear(x, w, *args, **kw)


SHAPES = [(1, 1, 1), (1, 3, 7), (1, 128, 16), (1, 4096, 4096), (2, 130, 70), (3, 64, 8), (5, 1000, 2049), (8, 4096, 136), (15, 250, 512),
          (16, 129, 64), (17, 300, 1025), (31, 77, 3000), (33, 1, 65), (64, 512, 576), (65, 2000, 128), (100, 10, 9000), (129, 257, 130),
          (192, 128, 4100), (193, 1000, 333), (255, 256, 257), (300, 1024, 4096), (513, 640, 200), (777, 4096, 1216), (1000, 384, 96),
          (8, 64, 16384), (12, 4096, 4097), (33, 515, 259), (64, 1000, 1001), (120, 16, 31), (2049, 1111, 1000), (4096, 2048, 512), (1, 20000, 24), (2, 64, 16384), (40, 8192, 16384)]


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_whole_numbers_come_out_exactly(cuda, bits, M, N, K):
    dtype = BF16 if (M + N + K) % 2 else FP16
    x, w, scale, sums = case(bits, M, N, K, dtype, cuda)
    g = gen(M, N, K)
    bias = whole(g, (N,), 100, FP32, cuda)
    assert torch.equal(product(bits, x, w, scale, out_dtype=FP32).double(), sums)
    # (below 2^15 / 2^5: nothing that fp16 cannot hold)
    small = (sums.abs() < 30000).all()
    if dtype == BF16 or small:
        res = whole(g, (M, N), 100, dtype, cuda)
        want = (sums + bias.double()).clamp(min=0) + res.double()
        assert want.abs().max() < 2 ** 24
        assert torch.equal(product(bits, x, w, scale, bias, "relu", res), want.float().to(dtype))
    res = whole(g, (M, N), 1000, FP32, cuda)
    got = product(bits, x, w, scale, bias.to(dtype), "none", res, out_dtype=FP32)
    assert torch.equal(got.double(), sums + bias.double() + res.double())


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("cols,splits", [(16, 1), (48, 1), (144, 1), (192, 1), (208, 1), (256, 1), (16, 2), (96, 2), (32, 4), (240, 4), (16, 8), (128, 8), (256, 8),
                                         (32, -2), (96, -2), (192, -2), (224, -2), (256, -2)])
@pytest.mark.parametrize("M,N,K", [(1, 128, 64), (300, 700, 1000), (530, 1300, 520), (40, 129, 8200), (2000, 5000, 72), (5000, 1500, 640)])
def test_every_plan(cuda, bits, cols, splits, M, N, K):
    """Forced tiles: one and several per CTA, more splits than there is K for, pairs with half of their outputs or tokens missing."""
    x, w, scale, sums = case(bits, M, N, K, BF16, cuda)
    bias, res = whole(gen(M), (N,), 50, FP32, cuda), whole(gen(N), (M, N), 50, FP32, cuda)
    ops.set_linear_plan(cols, splits)
    if bits and (splits == -2 or (splits > 1 and cols > 128)):           # (no such kernel)
        try:
            with pytest.raises(lib.TcbnnError):
                product(bits, x, w, scale)
        finally:
            ops.set_linear_plan()
        return
    try:
        got = product(bits, x, w, scale, bias, "relu", res, out_dtype=FP32)
        assert ops.linear_status() == 0
    finally:
        ops.set_linear_plan()
    assert torch.equal(got.double(), (sums + bias.double()).clamp(min=0) + res.double())


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (FP16, FP16), (BF16, FP32), (FP16, FP32)])
def test_activations(cuda, bits, name, dtype, out):
    M, N, K = 37, 200, 64
    x, w, scale, sums = case(bits, M, N, K, dtype, cuda)
    x, sums = x / 16, sums / 16                        # |z| up to about 10, exact
    bias = whole(gen(5), (N,), 3, FP32, cuda) / 8
    z = sums + bias.double()
    want = activation(z, name)
    got = product(bits, x, w, scale, bias, name, out_dtype=out).double()
    half_step = 0 if out == FP32 else torch.finfo(out).eps / 2
    # (the smallest steps of fp16 are 2^-24: results near 0 round to those)
    tol = z.abs() * 2.0 ** -21 + want.abs() * (half_step * (1 + 2.0 ** -10)) + (2.0 ** -24 if out == FP16 else 1e-30)
    assert ((got - want).abs() <= tol).all()
    far = torch.tensor([-math.inf, -300.0, -100.0, 100.0, 300.0], device=cuda)     # at the ends: 0 or z, never NaN
    if not bits:
        one = torch.ones((1, 1), dtype=dtype, device=cuda)
        y = ops.linear(one, torch.zeros((5, 1), dtype=dtype, device=cuda), far, name, out_dtype=FP32)[0]
        assert torch.equal(y[1:3].abs(), torch.zeros(2, device=cuda)) and torch.equal(y[3:], far[3:])


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 512, 8192), (16, 1000, 4096), (200, 384, 2048), (1024, 512, 4096)])
def test_real_values(cuda, bits, M, N, K):
    """Error of a sum of K products in fp32, each addition off by at most 2^-23 (truncated) of the partial sum: with
    partial sums like a random walk's, sqrt(K) 2^-23 of the norm sqrt(sum x^2 w^2) times sqrt(K) additions; ten times that."""
    g = torch.Generator(device=cuda)
    g.manual_seed(M + N)
    x = torch.randn((M, K), device=cuda, generator=g).to(BF16)
    if bits:
        w, w64 = signs(gen(N, K), N, K, cuda)
        scale = torch.rand((N,), device=cuda, generator=g) + 0.5
        w64 = w64 * scale.double()[:, None]
    else:
        w, scale = torch.randn((N, K), device=cuda, generator=g).to(BF16), None
        w64 = w.double()
    got = product(bits, x, w, scale, out_dtype=FP32).double()
    want = x.double() @ w64.t()
    norm = ((x.double() ** 2) @ (w64 ** 2).t()).sqrt()
    assert ((got - want).abs() <= 10 * math.sqrt(K) * 2.0 ** -23 * norm).all()


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,N,K,pad", [(1, 130, 100, 3), (7, 200, 333, 5), (130, 257, 129, 7), (40, 300, 128, 8), (260, 128, 512, 1)])
def test_rows_apart_and_what_lies_between_them(cuda, bits, dtype, M, N, K, pad):
    """Inputs with NaN between their rows, results between marks; every combination of operands that start on odd elements."""
    x0, w0, scale, sums = case(bits, M, N, K, dtype, cuda)
    for shift in (0, 1, 8):
        buf = torch.full((M, K + pad + shift), math.nan, dtype=dtype, device=cuda)
        x = buf[:, shift:shift + K]
        x.copy_(x0)
        w = w0
        if not bits:
            wbuf = torch.full((N, K + pad + shift), math.nan, dtype=dtype, device=cuda)
            w = wbuf[:, shift:shift + K]
            w.copy_(w0)
        obuf = torch.full((M, N + pad + shift), -77.0, dtype=FP32, device=cuda)
        out = obuf[:, shift:shift + N]
        assert product(bits, x, w, scale, out=out) is out
        assert torch.equal(out.double(), sums)
        mask = torch.ones_like(obuf, dtype=torch.bool)
        mask[:, shift:shift + N] = False
        assert (obuf[mask] == -77.0).all()
        # the residual stream updated in place
        rbuf = torch.full((M, N + pad + shift), 5.0, dtype=FP32, device=cuda)
        r = rbuf[:, shift:shift + N]
        product(bits, x, w, scale, residual=r, out=r)
        assert torch.equal(r.double(), sums + 5)
        assert (rbuf[mask] == 5.0).all()


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,N,K", [(3, 100, 64), (50, 264, 96), (300, 513, 128), (700, 1024, 72)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 8), (3, 0), (7, 1), (6, 2)])
def test_results_and_residuals_of_16_bits_anywhere(cuda, bits, dtype, M, N, K, pad, shift):
    """Blocks of columns of wider buffers, x next to its result in one of them; what lies around them stays."""
    x0, w, scale, _ = case(bits, M, N, K, dtype, cuda)
    x0 = x0.clamp(-1, 1)
    want = product(bits, x0, w, scale, out_dtype=FP32)                   # (whole numbers, exact: tested above)
    buf = torch.full((M, K + N + pad + shift), 3.0, dtype=dtype, device=cuda)
    x, out = buf[:, :K], buf[:, K + shift:K + shift + N]
    x.copy_(x0)
    res = torch.full((M, N + pad + shift), 2.0, dtype=dtype, device=cuda)
    r = res[:, shift:shift + N]
    product(bits, x, w, scale, residual=r, out=out)
    assert torch.equal(out, (want + 2).to(dtype))
    assert torch.equal(x, x0) and (buf[:, K:K + shift] == 3).all() and (buf[:, K + shift + N:] == 3).all()
    product(bits, x, w, scale, residual=r, out=r)
    assert torch.equal(r, (want + 2).to(dtype)) and (res[:, :shift] == 2).all() and (res[:, shift + N:] == 2).all()


@pytest.mark.parametrize("M,N,K", [(16, 70, 100), (100, 300, 100), (60, 1000, 100), (60, 300, 1000), (33, 2000, 100), (128, 300, 1000), (24, 2000, 2049),
                                   (16, 2100, 2049), (60, 2000, 100), (32, 2000, 1000), (33, 4000, 100), (33, 2000, 2049), (100, 1000, 333), (60, 4000, 333),
                                   (24, 5000, 2049), (5, 5000, 1000), (24, 8192, 1001), (9, 3001, 127), (47, 600, 129), (1, 40, 100000)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_few_rows_of_packed_weights(cuda, M, N, K, dtype, pad):
    """Every split of few rows: 8 to 32 of them to a block, 16 to 64 outputs, warps without a piece of K, rows on 16 bytes or not."""
    x, w, scale, sums = case(True, M, N, K, dtype, cuda)
    wide = torch.full((M, (K + 7) // 8 * 8 + pad), math.nan, dtype=dtype, device=cuda)
    wide[:, :K] = x
    bias = whole(gen(M, N), (N,), 50, FP32, cuda)
    got = ops.bit_linear(wide[:, :K], w, scale, bias, "relu", out_dtype=FP32)
    assert torch.equal(got.double(), (sums + bias.double()).clamp(min=0))


@pytest.mark.parametrize("bits", [False, True])
def test_results_of_more_than_two_to_the_31(cuda, bits):
    M, N, K = 66000, 33000, 40
    x, w, scale, _ = case(bits, M, N, K, BF16, cuda)
    out = product(bits, x, w, scale)
    assert out.numel() > 1 << 31
    rows = torch.tensor([0, 1, 32767, 65074, 65075, 65999], device=cuda)
    w64 = w.double()
    if bits:
        w64 = torch.stack([(w[:, k // 32] >> (31 - k % 32) & 1).double() * 2 - 1 for k in range(K)], 1) * scale.double()[:, None]
    assert torch.equal(out[rows], (x[rows].double() @ w64.t()).to(BF16))


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("M,N,K", [(3, 50, 77), (500, 600, 333)])
def test_workspaces(cuda, bits, M, N, K):
    """A workspace of one's own, for operands that need one; too small ones and none are refused by the library."""
    x, w, scale, sums = case(bits, M, N, K, BF16, cuda)
    ws = ops.linear_workspace(x, w)
    assert (ws is None) == (M == 3)                    # (few rows are read where they lie)
    assert torch.equal(product(bits, x, w, scale, out_dtype=FP32, workspace=ws).double(), sums)
    aligned = torch.zeros((M, 80 if K == 77 else 336), dtype=BF16, device=cuda)
    assert ops.linear_workspace(aligned, w if bits else aligned) is None
    if ws is not None:
        with pytest.raises(lib.TcbnnError):
            product(bits, x, w, scale, workspace=ws[:-256])


@pytest.mark.parametrize("bits", [False, True])
def test_infinities_and_nan_stay_in_their_rows_and_outputs(cuda, bits):
    M, N, K = 70, 300, 200
    x, w, scale, sums = case(bits, M, N, K, BF16, cuda)
    x = x.clone()
    x[3, 7], x[11, 199], x[69, 0] = math.inf, math.nan, -math.inf
    got = product(bits, x, w, scale, out_dtype=FP32).double()
    keep = [i for i in range(M) if i not in (3, 11, 69)]
    assert torch.equal(got[keep], sums[keep])
    assert got[11].isnan().all() and not got[3].isfinite().any() and not got[69].isfinite().any()
    if not bits:
        w = w.clone()
        w[299, 0] = math.nan
        got = ops.linear(x, w, out_dtype=FP32).double()
        assert torch.equal(got[keep][:, :299], sums[keep][:, :299]) and got[:, 299].isnan().all()


@pytest.mark.parametrize("bits", [False, True])
def test_no_rows(cuda, bits):
    x, w, scale, _ = case(bits, 1, 5, 9, BF16, cuda)
    assert product(bits, x[:0], w, scale).shape == (0, 5)


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("K", [72, 75])
def test_rows_over_four_gigabytes_apart(cuda, bits, K):
    """Offsets that pass 32 bits, in elements and in bytes."""
    far = (1 << 31) + 24
    x0, w, scale, sums = case(bits, 2, 40, K, BF16, cuda)
    big = torch.empty((far + K + 64,), dtype=BF16, device=cuda)
    x = big.as_strided((2, K), (far, 1))
    x.copy_(x0)
    assert torch.equal(product(bits, x, w, scale, out_dtype=FP32).double(), sums)
    out = big.as_strided((2, 40), (far, 1), 96)
    res = product(bits, x0, w, scale, out_dtype=BF16)
    product(bits, x0, w, scale, out=out)
    assert torch.equal(out, res)


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 1024, 2048), (90, 500, 333), (600, 512, 1024)])
def test_on_other_streams_and_in_graphs(cuda, bits, M, N, K):
    x, w, scale, sums = case(bits, M, N, K, BF16, cuda)
    want = sums.float()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(12):                                # calls that run at the same time
        with torch.cuda.stream(streams[i % 3]):
            outs.append(product(bits, x, w, scale, out_dtype=FP32))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    # two graphs, replayed at the same time with new inputs
    graphs = []
    for i in range(2):
        xi, oi = x.clone(), torch.empty_like(want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            product(bits, xi, w, scale, out=oi)
            product(bits, xi, w, scale, residual=oi, out=oi)
        graphs.append((g, xi, oi))
    graphs[1][1].mul_(0.5)
    torch.cuda.synchronize()
    for i, (g, _, _) in enumerate(graphs * 3):
        with torch.cuda.stream(streams[i % 2]):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][2], 2 * want) and torch.equal(graphs[1][2], want)
    assert ops.linear_status() == 0


@pytest.mark.parametrize("bits", [False, True])
def test_a_chain_of_dependent_calls(cuda, bits):
    """Each call reads what the one in front wrote, weights among it."""
    M, K = 24, 512
    g = gen(9)
    x = whole(g, (M, K), 1, BF16, cuda)
    want, have = x.double(), x
    for i in range(6):
        if bits:
            w, w64 = signs(g, K, K, cuda)
        else:
            w = torch.zeros((K, K), dtype=BF16, device=cuda)
            w[torch.arange(K), torch.randperm(K, generator=g).to(cuda)] = 2.0          # a permutation, doubled, just written
            w64 = w.double()
        want = (want @ w64.t()).clamp(min=0)
        want = want / (2.0 ** 10 if bits else 2)
        scale = torch.full((K,), 2.0 ** -10, device=cuda) if bits else None
        have = product(bits, have, w, scale, None, "relu") if bits else product(bits, have, w * 0.5, scale, None, "relu")
        if bits:
            want = want.float().to(BF16).double()
            # sums of rounded values: not whole numbers any more; an fp32 sum of 512 terms is within 512 2^-23 of sum |x|
            tol = have.double().abs() * 2.0 ** -8 + 512 * 2.0 ** -23 * 2.0 ** -10 * 512
            assert ((have.double() - want).abs() <= tol).all()
            want = have.double()
        else:
            assert torch.equal(have.double(), want)


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured: what is configured on first use is no obstacle."""
    program = """
import torch
from tcbnn_b200 import ops
x, w = torch.ones((%d, 100), dtype=torch.bfloat16, device="cuda"), torch.ones((70, 100), dtype=torch.bfloat16, device="cuda")
bits = torch.full((70, 4), -1, dtype=torch.int32, device="cuda")
logits = torch.ones((3, 5000), device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a, b, c = ops.linear(x, w), ops.bit_linear(x, bits), ops.log_probs(logits, None, 4)
g.replay()
torch.cuda.synchronize()
assert (a == 100).all() and (b == 100).all() and c[2].tolist() == [[0, 1, 2, 3]] * 3
print("fine")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for rows in (2, 400):
        r = subprocess.run([sys.executable, "-c", program % rows], cwd=root, capture_output=True, text=True, timeout=300)
        assert r.stdout.strip() == "fine", r.stderr[-2000:]


def test_results_are_the_same_every_time(cuda):
    for bits in (False, True):
        for M, N, K in [(1, 4096, 4096), (33, 1000, 3333), (500, 512, 2048)]:
            g = torch.Generator(device=cuda)
            g.manual_seed(3)
            x = torch.randn((M, K), device=cuda, generator=g).to(BF16)
            w = signs(gen(1), N, K, cuda)[0] if bits else torch.randn((N, K), device=cuda, generator=g).to(BF16)
            first = product(bits, x, w, None, out_dtype=FP32)
            for _ in range(4):
                assert torch.equal(product(bits, x, w, None, out_dtype=FP32), first)


def test_binary_weights_are_those_of_the_packers(cuda):
    """ops.pack_fc_weight's rows, and agreement with the bit GEMM where the inputs are signs too."""
    g = util.rng(11)
    W = torch.from_numpy(util.rand_pm1(g, (200, 64))).to(cuda)           # [K][N]
    X = torch.from_numpy(util.rand_pm1(g, (50, 200))).to(cuda)
    packed = ops.pack_fc_weight(W)
    got = ops.bit_linear(X.to(BF16), packed, out_dtype=FP32)
    assert torch.equal(got, X @ W)
    assert torch.equal(got.to(torch.int32), ops.bgemm(ops.pack_rows(X), packed, 200))


def test_refusals_with_tensors(cuda):
    x, w = torch.zeros((4, 32), dtype=BF16, device=cuda), torch.zeros((8, 32), dtype=BF16, device=cuda)
    bits = torch.zeros((8, 4), dtype=torch.int32, device=cuda)
    bad = [lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w[:, :31]),
           lambda: ops.linear(x, w, activation="tanh"), lambda: ops.linear(x, w, bias=torch.zeros(7, device=cuda)),
           lambda: ops.linear(x, w, bias=torch.zeros(8)), lambda: ops.linear(x, w, out_dtype=torch.float16),
           lambda: ops.linear(x, w, residual=torch.zeros((4, 8), device=cuda)), lambda: ops.linear(x.t(), w[:, :4]),
           lambda: ops.linear(x, w, out=torch.zeros((4, 9), dtype=BF16, device=cuda)), lambda: ops.linear(x.cpu(), w),
           lambda: ops.linear(x[:1].expand(4, 32), w), lambda: ops.linear(x, w, out=x[:, :8]), lambda: ops.linear(x[0], w),
           lambda: ops.bit_linear(x, bits[:, 1:]), lambda: ops.bit_linear(x, w),
           lambda: ops.bit_linear(x, bits, scale=torch.ones(8, dtype=BF16, device=cuda)),
           lambda: ops.bit_linear(torch.zeros((4, 129), dtype=BF16, device=cuda), bits)]
    for call in bad:
        with pytest.raises(lib.TcbnnError):
            call()
    buf = torch.zeros((4, 8 + 4), dtype=BF16, device=cuda)
    assert torch.equal(ops.bit_linear(x + 1, bits[:, :3]), torch.full((4, 8), -32.0, dtype=BF16, device=cuda))      # (words enough)
    with pytest.raises(lib.TcbnnError):
        ops.linear(x, w, residual=buf[:, 4:], out=buf[:, :8])
