"""ops.log_probs and Network.score against the definitions in 64 bits.

Tolerances: with d = (x - max) / T, a term e^d is off by 2^-22 (the exponential) and by the rounding of its argument, 2^-23 |d|;
sums run over at most V / 32 + 64 terms one after another, 2^-24 each; logarithm and differences add a few 2^-24 of the result.
E = sum p |d| (in 64 bits) is what the arguments' roundings weigh on average."""
import math

import pytest
import torch

from tcbnn_b200 import lib, models, ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(logits, T):
    """(log probabilities [M][V], entropy [M], E [M]) in 64 bits, rows without any token as documented."""
    z = logits.double()
    m = z.amax(1, keepdim=True)
    d = torch.where(m == -math.inf, -math.inf, (z - m) / T)
    S = torch.exp(d).sum(1, keepdim=True)
    logp = torch.where(S == 0, -math.inf, d - torch.log(S))
    p = torch.where(S == 0, 0.0, torch.exp(d) / S)
    pd = torch.where(p > 0, p * d, 0.0).sum(1)
    entropy = torch.where(S[:, 0] == 0, 0.0, torch.log(S[:, 0]) - pd)
    return logp, entropy, pd.abs()


def order(logits, top):
    """Ids in falling order, equal ones in rising order of tokens, -1 behind the last that is not ruled out."""
    v, i = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    return torch.where(v == -math.inf, -1, i)[:, :top]


def check(logits, targets, top, T=1.0, answer=None):
    M, V = logits.shape
    logp, entropy, ids, top_logp = answer or ops.log_probs(logits, targets, top, T)
    all_logp, want_h, E = definition(logits, T)
    steps = (V / 32 + 64) * 2.0 ** -24
    off_s = steps + 2.0 ** -21 + E * 2.0 ** -22
    assert ((entropy.double() - want_h).abs() <= (1 + E) * off_s + want_h.abs() * 2.0 ** -21).all()

    def near(got, want, off):
        # (the largest logit and the lowest are 2 x 3.4e38 apart in fp32 and bf16: past what fp32 holds, -inf when rounded)
        want = torch.where(want < -torch.finfo(torch.float32).max, -math.inf, want)
        ends = ~want.isfinite()
        assert torch.equal(got.double()[ends], want[ends])
        assert ((got.double() - want)[~ends].abs() <= off.expand_as(want)[~ends] + want[~ends].abs() * 2.0 ** -21).all()
    if targets is None:
        assert logp is None
    else:
        given = targets >= 0
        want = all_logp.gather(1, targets.long().clamp(min=0)[:, None])[:, 0]
        near(logp[given], want[given], off_s[given])
        assert (logp[~given] == 0).all()
    assert ids.shape == top_logp.shape == (M, top) and ids.dtype == torch.int64
    want_ids = order(logits, top)
    assert torch.equal(ids, want_ids)
    if top:
        want = torch.where(want_ids < 0, -math.inf, all_logp.gather(1, want_ids.clamp(min=0)))
        near(top_logp, want, off_s[:, None])


def rows(M, V, dtype, cuda, seed, sd=2.5):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return torch.randn((M, V), device=cuda, generator=g).mul_(sd).to(dtype), torch.randint(0, V, (M,), device=cuda, generator=g)


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 5, 5), (7, 10, 3), (2, 31, 31), (5, 33, 32), (300, 100, 5), (64, 1000, 5), (9, 1023, 32), (33, 1025, 1),
          (4, 4095, 20), (6, 4097, 0), (1, 8192, 8), (10, 20001, 32), (700, 2000, 10), (1, 131072, 20), (3, 131073, 32), (40, 50257, 7),
          (200, 32000, 1), (1500, 129, 0), (2, 524289, 32), (1, 1000003, 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,top", SHAPES)
def test_scores(cuda, dtype, M, V, top):
    x, y = rows(M, V, dtype, cuda, M + V)
    check(x, y, top, T=1.0 if V % 2 else 0.7)
    if M > 2:
        y[::3] = -1
    check(x, y.to(torch.int32), top, T=1.7)
    check(x, None, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [10, 100, 1000, 5000, 40000, 150001])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "two values", "one allowed", "few allowed", "lowest", "lowest and few",
                                  "last block", "peaked", "zeros of both signs", "huge"])
def test_orders_ties_and_masks(cuda, dtype, V, kind):
    M, top = 3, min(32, V)
    x, y = rows(M, V, dtype, cuda, V)
    n = torch.arange(V, device=cuda)
    lowest = torch.finfo(dtype).min
    if kind in ("rising", "falling"):
        x = (n.float() if kind == "rising" else -n.float()).mul(16.0 / V).to(dtype).repeat(M, 1)
    elif kind == "equal":
        x = torch.full_like(x, 1.5)
    elif kind == "two values":
        x = torch.where(x > 0, 3.0, -3.0).to(dtype)
    elif kind in ("one allowed", "few allowed"):
        keep = torch.zeros((M, V), dtype=torch.bool, device=cuda)
        for m in range(M):
            keep[m, ::max(1, V // (1 if kind == "one allowed" else 7))] = True
            if kind == "one allowed":
                keep[m] = False
                keep[m, (V - 1) * m // (M - 1)] = True
        x = x.masked_fill(~keep, -math.inf)
    elif kind == "lowest":
        x = torch.full_like(x, lowest)
    elif kind == "lowest and few":
        x = torch.where(n % max(1, V // 5) == 0, x, torch.full_like(x, lowest))
    elif kind == "last block":
        x[:, :-(V // 8 + 1)] = -math.inf
    elif kind == "peaked":
        x[:, V // 2] = 60.0
    elif kind == "zeros of both signs":
        x = torch.where(n % 3 == 0, -0.0, 0.0).to(dtype).repeat(M, 1)
    else:
        x = torch.where(x > 0, torch.finfo(dtype).max, lowest).to(dtype)
    check(x, y, top)


@pytest.mark.parametrize("warps,ctas", [(1, 1), (2, 1), (4, 1), (8, 1), (8, 2), (8, 4), (8, 8)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,top", [(3, 1, 1), (5, 9, 9), (9, 300, 32), (4, 2050, 5), (3, 30011, 32), (2, 100001, 20)])
def test_every_way_to_share_a_row(cuda, warps, ctas, dtype, M, V, top):
    """Random rows, one with more ties than any list holds, rising ones, masked ones; forced plans."""
    x, y = rows(M, V, dtype, cuda, V + M)
    n = torch.arange(V, device=cuda)
    x[0] = 0.5
    x[1] = (n.float() * (16.0 / V)).to(dtype)
    x[-1, n % 5 != 2] = -math.inf
    ops.set_log_probs_plan(warps, ctas)
    try:
        answer = ops.log_probs(x, y, top)
    finally:
        ops.set_log_probs_plan()
    check(x, y, top, answer=answer)


@pytest.mark.parametrize("value", [-1e4, -1e9, -1e20, -3e38])
@pytest.mark.parametrize("warps,ctas", [(1, 1), (8, 1), (8, 4)])
def test_masks_of_finite_values(cuda, value, warps, ctas):
    """Masks by large negative numbers, in front of, between and behind what is allowed; and nothing else at all."""
    V = 40000
    for dtype in (torch.float32, torch.bfloat16) + ((torch.float16,) if value == -1e4 else ()):
        x, y = rows(4, V, dtype, cuda, 3)
        x[0, :30000], x[1, 10000:], x[2, ::2] = value, value, value
        x[3] = value
        ops.set_log_probs_plan(warps, ctas)
        try:
            for T in (1.0, 0.01, 50.0):
                check(x, y, 9, T, answer=ops.log_probs(x, y, 9, T))
        finally:
            ops.set_log_probs_plan()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 40, 3000, 70001])
def test_rows_that_rule_out_everything(cuda, dtype, V):
    x, y = rows(5, V, dtype, cuda, V)
    x[1], x[4] = -math.inf, -math.inf
    top = min(V, 6)
    check(x, y, top)
    logp, entropy, ids, top_logp = ops.log_probs(x, y, top)
    for m in (1, 4):
        assert logp[m] == -math.inf and entropy[m] == 0 and (ids[m] == -1).all() and (top_logp[m] == -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 70001])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("masked", [False, True])
def test_nan_and_infinity_stay_in_their_row(cuda, dtype, V, value, masked):
    M, top = 6, 5
    x, y = rows(M, V, dtype, cuda, V)
    if masked:
        x[:, V // 3:] = -math.inf
    x[2, V // 4], y[2], y[3] = value, 0, -1
    x[3, 0] = value
    keep = [0, 1, 4, 5]
    logp, entropy, ids, top_logp = ops.log_probs(x, y, top)
    assert logp[2].isnan() and logp[3] == 0 and entropy[2:4].isnan().all() and top_logp[2:4].isnan().all()
    clean = x.clone()
    clean[2, V // 4] = clean[3, 0] = -math.inf if math.isnan(value) else math.inf
    if math.isnan(value):                              # NaN is no alternative, +inf the first
        assert torch.equal(ids, order(clean, top))
    else:
        assert torch.equal(ids, order(clean, top)) and ids[2, 0] == V // 4 and ids[3, 0] == 0
    # (not bit for bit what the rows alone give: a thread's share depends on where a row starts modulo 16 bytes, and with it
    # the order of the sums)
    check(x[keep], y[keep], top, answer=(logp[keep], entropy[keep], ids[keep], top_logp[keep]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,pad,shift", [(5, 3, 1), (1000, 24, 0), (1001, 1, 3), (50001, 47, 0), (50001, 0, 0), (33333, 5, 7)])
def test_rows_apart(cuda, dtype, V, pad, shift):
    """Rows that start anywhere, between NaN."""
    M = 9
    buf = torch.full((M, shift + V + pad), math.nan, dtype=dtype, device=cuda)
    x, y = rows(M, V, dtype, cuda, V)
    view = buf[:, shift:shift + V]
    view.copy_(x)
    check(view, y, min(V, 9))


def test_logits_over_four_gigabytes_apart(cuda):
    V, far = 3001, (1 << 32) // 2 + 72
    big = torch.empty((far + V,), dtype=torch.bfloat16, device=cuda)
    x = big.as_strided((2, V), (far, 1))
    src, y = rows(2, V, torch.bfloat16, cuda, 1)
    x.copy_(src)
    check(x, y, 4)


def test_targets_outside_the_vocabulary(cuda):
    x, y = rows(4, 100, torch.float32, cuda, 1)
    y[1], y[2] = 100, 1 << 40
    logp = ops.log_probs(x, y)[0]
    assert logp[1].isnan() and logp[2].isnan() and logp[[0, 3]].isfinite().all()


def test_extreme_temperatures(cuda):
    x, y = rows(4, 777, torch.float32, cuda, 2)
    logp, entropy, ids, top = ops.log_probs(x, y, 3, 1e-30)
    assert torch.equal(top[:, 0], torch.zeros(4, device=cuda)) and (entropy == 0).all() and (top[:, 1:] < -1e20).all()
    assert torch.equal(ids, order(x, 3))
    logp, entropy, ids, top = ops.log_probs(x, y, 3, 1e30)
    assert torch.equal(ids, order(x, 3)) and ((entropy.double() - math.log(777)).abs() < 1e-5).all()


def test_no_rows_and_no_outputs(cuda):
    x = torch.empty((0, 10), device=cuda)
    logp, entropy, ids, top = ops.log_probs(x, torch.empty((0,), dtype=torch.int64, device=cuda), 3)
    assert logp.shape == entropy.shape == (0,) and ids.shape == top.shape == (0, 3)


def test_the_same_every_time_on_streams_and_in_graphs(cuda):
    for M, V, dtype in [(2, 100000, torch.bfloat16), (500, 1000, torch.float32), (300, 30000, torch.float16)]:
        x, y = rows(M, V, dtype, cuda, M)
        want = ops.log_probs(x, y, 12)
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got = []
        for i in range(9):
            with torch.cuda.stream(streams[i % 3]):
                got.append(ops.log_probs(x, y, 12))
        torch.cuda.synchronize()
        for r in got:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
        xs = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.log_probs(xs, y, 12)
        for flip in (False, True):
            xs.copy_(x.flip(1) if flip else x)
            g.replay()
            w = ops.log_probs(xs, y, 12)
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_refusals_with_tensors(cuda):
    x, y = rows(4, 50, torch.float32, cuda, 2)
    bad = [lambda: ops.log_probs(x.double(), y), lambda: ops.log_probs(x, y[:3]), lambda: ops.log_probs(x, y.float()), lambda: ops.log_probs(x.cpu(), y),
           lambda: ops.log_probs(x, y.cpu()), lambda: ops.log_probs(x, y, 33), lambda: ops.log_probs(x, y, -1), lambda: ops.log_probs(x[:, :5], y, 6),
           lambda: ops.log_probs(x, y, 3, 0.0), lambda: ops.log_probs(x, y, 3, math.nan), lambda: ops.log_probs(x, y, 3, -1.0),
           lambda: ops.log_probs(x.t(), None), lambda: ops.log_probs(x[0], None), lambda: ops.log_probs(x[:1].expand(4, 50), y)]
    for call in bad:
        with pytest.raises(lib.TcbnnError):
            call()


def test_network_score(cuda):
    """A network's answers scored: the live images' logits, and a real-valued head in front of the same scores."""
    spec = models.mlp_spec(70, features=100, hidden=128)
    net = models.Network(spec, models.synthetic_weights(spec, 1), models.synthetic_input(spec, 2))
    labels = torch.arange(70, device=cuda) % 10
    logits = net.forward()
    want = ops.log_probs(logits, labels, 5)
    assert all(torch.equal(a, b) for a, b in zip(net.score(labels, top=5), want))
    net.set_batch(33)
    net.forward()
    got = net.score(labels[:33], top=5, temperature=2.0)
    assert got[0].shape == (33,)
    check(net.forward()[:33], labels[:33], 5, 2.0)


@pytest.mark.parametrize("M,V", [(1, 5003), (77, 5003), (300, 1000)])
def test_head_and_scores_together(cuda, M, V):
    """A binary hidden layer, a real-valued head and the scores of its fp32 logits, as one graph."""
    g = torch.Generator(device=cuda)
    g.manual_seed(M)
    K = 512
    x = torch.randn((M, K), device=cuda, generator=g).to(torch.bfloat16)
    bits = torch.randint(-2 ** 31, 2 ** 31, (K, K // 32), device=cuda, generator=g).to(torch.int32)
    scale = torch.full((K,), K ** -0.5, device=cuda)
    head = torch.randn((V, K), device=cuda, generator=g).mul_(3 * K ** -0.5).to(torch.bfloat16)
    y = torch.randint(0, V, (M,), device=cuda, generator=g)

    def step():
        h = ops.bit_linear(x, bits, scale, None, "gelu", x)
        logits = ops.linear(h, head, out_dtype=torch.float32)
        return logits, ops.log_probs(logits, y, 10)
    logits, first = step()
    check(logits, y, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits2, second = step()
    graph.replay()
    assert torch.equal(logits, logits2) and all(torch.equal(a, b) for a, b in zip(first, second))
