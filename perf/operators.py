"""The operators of language-model heads and projections that stand beside the bit GEMM family, as work to be
timed: ops.linear, ops.bit_linear and ops.log_probs.

A case is a dict of plain values; "op" picks the operator:

  linear      y = act(x W^T + b) + r,             x [M][K] and W [N][K] in 16 bits
  bit_linear  y = act(s * (x W^T) + b) + r,       W [N] rows of packed signs (bit 31 - k % 32 of word k / 32 is
                                                  element k, set = +1), s one scale per output
  log_probs   log probabilities of given tokens, entropy and the `top` likeliest alternatives of [M][V] logits

All data is synthetic.  `own` picks between the plain forms below and the framework's calls.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases -----------------------------------------------------------------------------------

def _product(op, M, N, K, dtype="bf16", out="same", bias=True, act="none", residual=False, pad=0):
    """pad: elements behind each row of x (x is a block of columns of a wider buffer)."""
    return dict(op=op, M=M, N=N, K=K, dtype=dtype, out=out, bias=bias, act=act, residual=residual, pad=pad)


def _scores(M, V, dtype, top, temperature=1.0, pad=0, masked=0.0):
    """pad: logits behind each row (a vocabulary padded to a round number); masked: share of the tokens that a
    grammar rules out, their logits -inf."""
    return dict(op="log_probs", M=M, V=V, dtype=dtype, top=top, temperature=temperature, pad=pad, masked=masked)


def listed():
    return [
        # one token through a 4096-wide projection that adds to its residual stream: the weight's way from memory
        dict(_product("linear", 1, 4096, 4096, bias=False, residual=True), name="linear_1x4096x4096"),
        # a batch of 16 requests through the first FC layer of AlexNet, held in real values
        dict(_product("linear", 16, 4096, 9216, dtype="fp16", act="relu"), name="linear_16x4096x9216_relu"),
        # classifier head on a ragged batch: odd features, fp32 logits
        dict(_product("linear", 333, 1000, 2049, out="fp32"), name="linear_333x1000x2049_fp32"),
        # a prompt through a wide hidden layer: tensor cores throughout
        dict(_product("linear", 4096, 16384, 4096, act="gelu"), name="linear_4096x16384x4096_gelu"),
        # the same layers with binary weights: one token, ...
        dict(_product("bit_linear", 1, 4096, 4096, bias=False, residual=True), name="bit_1x4096x4096"),
        # ... a few requests through wide layers
        dict(_product("bit_linear", 24, 8192, 8192, act="silu"), name="bit_24x8192x8192_silu"),
        # ... a ragged batch, its input a block of columns of a wider buffer
        dict(_product("bit_linear", 1001, 5000, 2049, dtype="fp16", residual=True, pad=31), name="bit_1001x5000x2049"),
        # ... and the prompt
        dict(_product("bit_linear", 4096, 16384, 4096, act="gelu_tanh"), name="bit_4096x16384x4096_gelu_tanh"),
        # eight images' class scores with the five likeliest, from an output layer's fp32 logits
        dict(_scores(8, 1000, "fp32", 5), name="scores_8x1000"),
        # one decoding step of one request
        dict(_scores(1, 131072, "bf16", 20, temperature=0.7), name="scores_1x131072"),
        # one decoding step of 48 requests under a grammar
        dict(_scores(48, 100003, "fp32", 10, masked=0.9), name="scores_48x100003_masked"),
        # scoring a prompt: every position's token against the vocabulary, padded rows
        dict(_scores(4096, 50001, "bf16", 8, pad=47), name="scores_4096x50001"),
    ]


def _log(rng, lo, hi, whole=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / whole)) * whole))


def draw(rng):
    while True:
        if rng.random() < 0.62:
            whole = rng.choice([1, 1, 8, 64])
            c = _product(rng.choice(["linear", "bit_linear"]), _log(rng, 1, 4096), _log(rng, 64, 16384, whole), _log(rng, 64, 16384, whole),
                         rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["same", "same", "fp32"]), rng.random() < 0.6,
                         rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]), rng.random() < 0.4,
                         rng.choice([0, 0, 0, 64, rng.randint(1, 40)]))
        else:
            c = _scores(_log(rng, 1, 8192), _log(rng, 10, 200000), rng.choice(["bf16", "fp16", "fp32"]), rng.choice([0, 1, 5, rng.randint(2, 32)]),
                        rng.choice([1.0, 1.0, 0.7, 1.3]), rng.choice([0, 0, rng.randint(1, 63)]), rng.choice([0.0, 0.0, 0.5, 0.95]))
            c["top"] = min(c["top"], c["V"])
        w = work(c)
        if w["flops"] <= 5.4e11 and w["bytes"] <= 4.0e8:
            return c


# ---- inputs ----------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    t, M = TYPES[case["dtype"]], case["M"]
    if case["op"] == "log_probs":
        V, pitch = case["V"], case["V"] + case["pad"]
        logits = torch.empty((M, pitch), dtype=t, device="cuda")
        logits.normal_(0.0, 2.5, generator=g)
        targets = torch.randint(0, V, (M,), device="cuda", generator=g)
        if case["masked"]:
            out = torch.rand((M, pitch), device="cuda", generator=g) < case["masked"]
            out.scatter_(1, targets[:, None], False)          # the token that was taken was allowed
            logits.masked_fill_(out, -math.inf)
        if M > 8:
            targets[torch.rand((M,), device="cuda", generator=g) < 0.05] = -1       # positions without a token
        return dict(case=case, logits=logits[:, :V], targets=targets)
    N, K = case["N"], case["K"]
    y = t if case["out"] == "same" else TYPES[case["out"]]
    s = dict(case=case, out=y, x=rand(M, K + case["pad"]).to(t)[:, :K], bias=rand(N) * 0.5 if case["bias"] else None,
             residual=rand(M, N).to(y) if case["residual"] else None)
    if case["op"] == "linear":
        s["weight"] = torch.empty((N, K), dtype=t, device="cuda").normal_(0.0, K ** -0.5, generator=g)
        s["bias"] = s["bias"].to(t) if case["bias"] else None
    else:
        ld = (K + 127) // 128 * 4
        bits = torch.randint(-2 ** 31, 2 ** 31, (N, ld), dtype=torch.int64, device="cuda", generator=g)
        word = torch.arange(ld, device="cuda")
        left = (K - 32 * word).clamp(0, 32)
        s["bits"] = (bits & -(1 << (32 - left))).to(torch.int32)       # bits behind the last element are 0
        s["scale"] = (0.5 + torch.rand((N,), device="cuda", generator=g)) * K ** -0.5
    return s


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        from tcbnn_b200 import ops
        if case["op"] == "log_probs":
            return ops.log_probs(state["logits"], state["targets"], top=case["top"], temperature=case["temperature"])
        if case["op"] == "linear":
            return ops.linear(state["x"], state["weight"], state["bias"], case["act"], state["residual"], out_dtype=state["out"])
        return ops.bit_linear(state["x"], state["bits"], state["scale"], state["bias"], case["act"], state["residual"], out_dtype=state["out"])
    return _plain_scores(state) if case["op"] == "log_probs" else _plain_product(state)


def _activation(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _signs(bits, K):
    """Packed signs as fp32 +-1 [N][K]."""
    shift = torch.arange(31, -1, -1, dtype=torch.int32, device=bits.device)
    return ((bits[:, :, None] >> shift) & 1).reshape(bits.shape[0], -1)[:, :K].float() * 2 - 1


def _plain_product(state):
    case = state["case"]
    if case["op"] == "linear":
        z = state["x"].float() @ state["weight"].float().t()
    else:
        z = (state["x"].float() @ _signs(state["bits"], case["K"]).t()) * state["scale"]
    if state["bias"] is not None:
        z = z + state["bias"].float()
    z = _activation(z, case["act"])
    if state["residual"] is not None:
        z = z + state["residual"].float()
    return z.to(state["out"])


def _plain_scores(state):
    """logp [M], entropy [M], top_ids [M][top], top_logp [M][top]."""
    case, x, target = state["case"], state["logits"].float(), state["targets"]
    d = (x - x.amax(1, keepdim=True)) / case["temperature"]
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    lse = torch.log(S)
    entropy = lse[:, 0] - torch.where(e > 0, e * d, 0.0).sum(1) / S[:, 0]
    logp = torch.where(target >= 0, (d.gather(1, target.clamp(min=0)[:, None]) - lse)[:, 0], 0.0)
    # in falling order of the logits, equal ones in rising order of their tokens; ruled out ones are none
    best = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top"]]
    top = d.gather(1, best) - lse
    return logp, entropy, torch.where(top > -math.inf, best, -1), top


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    size = lambda t: 4 if t == "fp32" else 2  # noqa: E731
    M = case["M"]
    if case["op"] == "log_probs":
        return {"bytes": M * case["V"] * size(case["dtype"]) + 8 * M + 8 * M + 12 * M * case["top"], "flops": 6 * M * case["V"]}
    N, K = case["N"], case["K"]
    out = 2 if case["out"] == "same" else size(case["out"])
    one = case["op"] == "linear"
    weight = 2 * N * K if one else N * K // 8 + 4 * N
    return {"bytes": 2 * M * K + weight + (M * N * out) * (2 if case["residual"] else 1) + (N * (2 if one else 4) if case["bias"] else 0),
            "flops": 2 * M * N * K}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _gelu64(z, tanh):
    if not tanh:
        return z * 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "log_probs":
        rows = []
        for first in range(0, case["M"], 256):
            z = s["logits"][first:first + 256].double() / case["temperature"]
            t = s["targets"][first:first + 256]
            logp = torch.log_softmax(z, dim=1)
            taken = torch.gather(logp, 1, torch.where(t < 0, 0, t).unsqueeze(1)).squeeze(1)
            rows.append((taken.masked_fill(t < 0, 0.0), torch.special.entr(logp.exp()).sum(1), torch.topk(logp, case["top"], dim=1)[0]))
        logp, entropy, top = (torch.cat(r) for r in zip(*rows))
        return logp, entropy, None, top
    x = s["x"].double()
    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", x, s["weight"].double())
    else:
        k = torch.arange(case["K"], device=x.device)
        w = torch.where((s["bits"][:, k // 32].long() >> (31 - k % 32)) % 2 == 1, 1.0, -1.0).double()
        z = torch.einsum("mk,nk->mn", x, w) * s["scale"].double()
    if s["bias"] is not None:
        z += s["bias"].double()
    act = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: _gelu64(v, False),
           "gelu_tanh": lambda v: _gelu64(v, True)}[case["act"]]
    z = act(z)
    return z if s["residual"] is None else z + s["residual"].double()
