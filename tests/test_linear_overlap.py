"""CPU-only: a workspace is written while operands are read and results stored, so it may share no memory with them."""
import pytest

from tcbnn_b200 import lib

X, W, B, R, O, S = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000, 0x60000000        # addresses that nothing reads
M, N, K = 500, 600, 333
ROWS = 336 * 2                                         # bytes of a copied row


def product(ws, packed, x=X, w=W, ws_bytes=1 << 24):
    args = [x, w] + ([S] if packed else []) + [B, R, O, M, N, K, K, 12 if packed else K, N, N, lib.BF16, lib.BF16, lib.FP32, 0, ws, ws_bytes, None]
    rc = getattr(lib.load(), "tcbnn_bit_linear" if packed else "tcbnn_linear")(*args)
    assert rc != 0                                     # (there is no device, if nothing else)
    return lib.load().tcbnn_last_error().decode()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("at", [X, W, B, R, O, S])
@pytest.mark.parametrize("off", [0, -256, 256])
def test_workspaces_over_operands_are_refused(packed, at, off):
    if at == S and not packed:
        pytest.skip("no scale")
    assert "workspace overlaps" in product(at + off, packed), (hex(at), off)


@pytest.mark.parametrize("packed", [False, True])
def test_workspaces_apart_from_operands_pass(packed):
    used = sum((rows * ROWS + 255) // 256 * 256 for rows in ((M,) if packed else (M, N)))
    assert lib.load().tcbnn_linear_workspace_bytes(X, None if packed else W, M, N, K, K, K) == used
    for ws in (0x70000000, O - used, O + M * N * 2 + 256 - M * N * 2 % 256):
        assert "workspace overlaps" not in product(ws, packed), hex(ws)
    # (what is given beyond what is used may be anything, all of it where nothing is copied)
    assert "workspace overlaps" not in product(O - used, packed, ws_bytes=1 << 30)


def scores(**kw):
    a = dict(logits=X, type=lib.FP32, M=4, V=100, ld=128, targets=W, target_bytes=8, temperature=1.0, top=5, logp=B, entropy=R, ids=O, top_logp=S, stream=None)
    a.update(kw)
    rc = lib.load().tcbnn_log_probs(*a.values())
    assert rc != 0                                     # (there is no device, if nothing else)
    return lib.load().tcbnn_last_error().decode()


@pytest.mark.parametrize("kw", [dict(logp=X), dict(entropy=X + 396), dict(ids=X + 512), dict(top_logp=X + 3 * 512 + 396), dict(logp=W + 16), dict(entropy=W),
                                dict(ids=W + 24), dict(top_logp=W), dict(entropy=B + 12), dict(ids=B), dict(top_logp=B - 76), dict(ids=R + 8), dict(top_logp=R),
                                dict(top_logp=O + 156)])
def test_scores_over_logits_targets_or_one_another_are_refused(kw):
    assert "overlap" in scores(**kw)


@pytest.mark.parametrize("kw", [dict(), dict(logp=X + 400), dict(entropy=B + 16), dict(top_logp=O + 160), dict(targets=None, logp=X), dict(entropy=None), dict(top=0, ids=X, top_logp=X),
                                dict(targets=W, entropy=W + 32)])
def test_scores_side_by_side_pass(kw):
    assert "overlap" not in scores(**kw)
