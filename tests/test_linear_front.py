"""CPU-only: what ops.linear, ops.bit_linear and ops.log_probs hand to the library, with tensors that have no memory and a library that
only takes notes."""
import pytest
import torch

from tcbnn_b200 import lib, ops

BF16 = torch.bfloat16
BIG = 1 << 32                                          # an int of the C interface keeps the rest of what is added to it


@pytest.fixture
def calls(monkeypatch):
    made = []

    def bound(name):
        def f(*args):
            made.append((name, args))
            return 0
        return f
    monkeypatch.setattr(ops, "_current_device", lambda: -1)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(lib, "bound", bound)
    return made


def meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_calls_within_the_range_go_through(calls):
    ops.linear(meta(4, 8), meta(5, 8))
    ops.bit_linear(meta(4, 8), meta(5, 4, dtype=torch.int32))
    ops.log_probs(meta(4, 8), None, 2)
    assert [name for name, _ in calls] == ["tcbnn_linear", "tcbnn_bit_linear", "tcbnn_log_probs"]


@pytest.mark.parametrize("call", [
    lambda: ops.linear(meta(BIG + 4, 8), meta(5, 8)), lambda: ops.linear(meta(4, 8), meta(BIG + 5, 8)),
    lambda: ops.linear(meta(4, BIG + 8), meta(5, BIG + 8)), lambda: ops.linear(meta((1 << 31) + 4, 8), meta(5, 8)),
    lambda: ops.bit_linear(meta(BIG + 4, 8), meta(5, 4, dtype=torch.int32)), lambda: ops.bit_linear(meta(4, 8), meta(BIG + 5, 4, dtype=torch.int32)),
    lambda: ops.bit_linear(meta(4, BIG + 8), meta(5, BIG // 32 + 4, dtype=torch.int32)),
    lambda: ops.linear_workspace(meta(BIG + 4, 8), meta(5, 8)), lambda: ops.linear_workspace(meta(4, 8), meta(BIG + 5, 8)),
    lambda: ops.log_probs(meta(BIG + 4, 8), None, 2), lambda: ops.log_probs(meta(4, BIG + 8), None, 2)])
def test_sizes_that_no_int_holds_are_refused(calls, call):
    with pytest.raises(lib.TcbnnError, match="2\\^31"):
        call()
    assert not calls


@pytest.mark.parametrize("workspace", [torch.empty((1,), dtype=torch.uint8, device="meta").expand(1 << 20),
                                       torch.empty((1 << 20, 2), dtype=torch.uint8, device="meta")[:, 0],
                                       torch.empty((2, 1 << 20), dtype=torch.uint8, device="meta").as_strided((2, 1 << 20), (1, 1))])
def test_workspaces_that_do_not_lie_together_are_refused(calls, workspace):
    """Their number of elements says nothing about how much memory follows their address."""
    with pytest.raises(lib.TcbnnError, match="contiguous"):
        ops.linear(meta(400, 7), meta(500, 7), workspace=workspace)
    with pytest.raises(lib.TcbnnError, match="contiguous"):
        ops.bit_linear(meta(400, 7), meta(500, 4, dtype=torch.int32), workspace=workspace)
    assert not calls
