"""CPU-only: what the entry points of the real-valued products and of the scores refuse, before any device is asked."""
import pytest

from tcbnn_b200 import lib

X, W, B, R, O = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000        # addresses that nothing reads


def product(name="tcbnn_linear", scale=None, **kw):
    a = dict(x=X, W=W, bias=B, residual=R, out=O, M=4, N=64, K=128, ldx=128, ldw=4 if "bit" in name else 128, ldr=64, ldo=64,
             type=lib.BF16, out_type=lib.BF16, bias_type=lib.FP32, activation=1, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    args = list(a.values())
    if "bit" in name:
        args.insert(2, scale)
    rc = getattr(lib.load(), name)(*args)
    return rc, lib.load().tcbnn_last_error().decode()


BAD = [(dict(N=0), "N and K"), (dict(K=0), "N and K"), (dict(M=-1), "M >= 0"), (dict(M=(1 << 30) + 1), "2^30"),
       (dict(N=(1 << 30) + 1, ldo=1 << 31, ldr=1 << 31), "2^30"), (dict(K=(1 << 24) + 1, ldx=1 << 25), "2^24"), (dict(ldo=(1 << 40) + 8), "2^40"),
       (dict(type=lib.FP32), "fp16 or bf16"), (dict(type=7), "fp16 or bf16"),
       (dict(out_type=lib.FP16), "x's type or fp32"), (dict(bias_type=lib.FP16), "x's type or fp32"), (dict(activation=5), "activation"),
       (dict(activation=-1), "activation"), (dict(x=None), "null"), (dict(W=None), "null"), (dict(out=None), "null"), (dict(ldx=127), "closer"),
       (dict(ldo=63), "closer"), (dict(ldr=63), "closer"), (dict(x=X + 1), "aligned"), (dict(out=O + 1), "aligned"), (dict(residual=R + 1), "aligned"),
       (dict(bias=B + 2), "aligned"), (dict(out=X + 512), "overlaps x"), (dict(out=W), "overlaps x"), (dict(out=B - 64), "overlaps the bias"),
       (dict(residual=O + 64), "residual overlaps"), (dict(residual=O, ldr=72), "residual overlaps")]


@pytest.mark.parametrize("name", ["tcbnn_linear", "tcbnn_bit_linear"])
@pytest.mark.parametrize("kw,says", BAD)
def test_products_refuse(name, kw, says):
    rc, text = product(name, **kw)
    assert rc != 0 and says in text, text


def test_dense_and_packed_weights_refuse():
    assert "closer" in product(ldw=127)[1]
    assert "aligned" in product(W=W + 1)[1]
    for kw in (dict(ldw=3), dict(ldw=5), dict(ldw=4, K=129, ldx=129)):
        rc, text = product("tcbnn_bit_linear", **kw)
        assert rc != 0 and "multiple of 4" in text
    assert "16-byte" in product("tcbnn_bit_linear", W=W + 4)[1]
    assert "scale" in product("tcbnn_bit_linear", scale=B + 2)[1]
    assert "overlaps the scale" in product("tcbnn_bit_linear", scale=O + 16)[1]


def test_no_rows_is_no_call():
    for name in ("tcbnn_linear", "tcbnn_bit_linear"):
        assert product(name, M=0, x=None, out=None)[0] == 0


def test_columns_side_by_side_do_not_overlap():
    """x and out as blocks of columns of one buffer pass the checks: refused for another reason further on."""
    rc, text = product(x=X, out=X + 256, ldx=192, ldo=192, W=None)
    assert rc != 0 and "null" in text
    rc, text = product(x=X, out=X + 254, ldx=192, ldo=192)
    assert rc != 0 and "overlaps x" in text


def scores(**kw):
    a = dict(logits=X, type=lib.FP32, M=4, V=100, ld=100, targets=W, target_bytes=8, temperature=1.0, top=5, logp=B, entropy=R, ids=O, top_logp=O + 4096, stream=None)
    a.update(kw)
    rc = lib.load().tcbnn_log_probs(*a.values())
    return rc, lib.load().tcbnn_last_error().decode()


@pytest.mark.parametrize("kw,says", [
    (dict(M=-1), "M >= 0"), (dict(V=0), "V >= 1"), (dict(V=(1 << 30) + 1, ld=1 << 31), "2^30"), (dict(ld=(1 << 40) + 1), "2^40"), (dict(type=3), "fp32, fp16 or bf16"), (dict(ld=99), "closer"), (dict(target_bytes=2), "int32 or int64"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(top=33), "top"), (dict(top=-1), "top"), (dict(top=6, V=5, ld=5), "top"), (dict(logits=None), "null"),
    (dict(ids=None), "null"), (dict(top_logp=None), "null"), (dict(logp=None), "null"), (dict(logits=X + 2), "aligned"), (dict(targets=W + 4), "aligned"),
    (dict(ids=O + 4), "aligned"), (dict(entropy=R + 1), "aligned")])
def test_scores_refuse(kw, says):
    rc, text = scores(**kw)
    assert rc != 0 and says in text, text


def test_no_rows_of_scores():
    assert scores(M=0, logits=None)[0] == 0
