"""Refusals of the short convolution, the selective scan and beam search's operators that need no GPU: wrong tensors at the Python entries, wrong
arguments at the C ones (nothing is launched, pointers are never followed)."""
import ctypes

import pytest
import torch

P = 4096  # never dereferenced


def conv_args(**over):
    from functs_b200 import _lib
    a = _lib.CausalConvArgs(dtype=2, batch=2, tokens=3, channels=8, width=4, num_slots=2, x=P, weight=P, bias=P, out=P, state_in=P, state_out=P)
    for name, value in over.items():
        setattr(a, name, value)
    return a


def scan_args(**over):
    from functs_b200 import _lib
    a = _lib.SelectiveScanArgs(dtype=2, batch=2, tokens=3, channels=8, groups=2, states=16, num_slots=2, x=P, dt=P, z=P, B=P, C=P, out=P, A=P, D=P,
                               dt_bias=P, state_in=P, state_out=P)
    for name, value in over.items():
        setattr(a, name, value)
    return a


def conv(a):
    from functs_b200 import _lib
    return _lib.lib.functs_b200_causal_conv(None if a is None else ctypes.byref(a), None), _lib.last_error()


def scan(a):
    from functs_b200 import _lib
    return _lib.lib.functs_b200_selective_scan(None if a is None else ctypes.byref(a), None, None), _lib.last_error()


@pytest.mark.parametrize("over,match", [
    ({"dtype": 3}, "dtype"), ({"batch": -1}, "batch"), ({"batch": 65536}, "batch"), ({"tokens": -1}, "tokens"), ({"channels": 0}, "channels"),
    ({"width": 1}, "width"), ({"width": 9}, "width"), ({"num_slots": 3}, "as many states"), ({"num_slots": -1, "slots": P}, "negative"),
    ({"weight": None}, "null pointer"), ({"state_out": None}, "null pointer"), ({"x": None}, "null pointer"), ({"out": None}, "null pointer"),
] + [({n: P + 1}, "boundary") for n in ("x", "weight", "bias", "out", "state_in", "state_out")] + [({n: P + 2}, "boundary") for n in ("slots", "lengths", "status")])
def test_causal_conv_arguments(over, match):
    rc, why = conv(conv_args(**over))
    assert rc == -1 and match in why


@pytest.mark.parametrize("over,match", [
    ({"dtype": -1}, "dtype"), ({"batch": -1}, "batch"), ({"tokens": -1}, "tokens"), ({"channels": 0}, "channels"), ({"groups": 3}, "multiple"),
    ({"groups": 0}, "multiple"), ({"states": 0}, "states"), ({"states": 65}, "states"), ({"num_slots": 3}, "as many states"),
    ({"num_slots": -1, "slots": P}, "negative"), ({"A": None}, "null pointer"), ({"state_out": None}, "null pointer"),
] + [({n: None}, "null pointer") for n in ("x", "dt", "B", "C", "out")] + [({n: P + 1}, "boundary") for n in ("x", "dt", "z", "B", "C", "out")]
    + [({n: P + 2}, "boundary") for n in ("A", "D", "dt_bias", "state_in", "state_out", "slots", "lengths", "status")])
def test_selective_scan_arguments(over, match):
    rc, why = scan(scan_args(**over))
    assert rc == -1 and match in why


def test_of_nothing():
    assert conv(conv_args(batch=0, num_slots=0))[0] == 0 and conv(None)[0] == -1
    assert scan(scan_args(batch=0, num_slots=0))[0] == 0 and scan(None)[0] == -1


def select(**over):
    from functs_b200 import _lib
    a = dict(logits=P, dtype=1, group_stride=40, beam_stride=10, scores=P, ended=P, end_token=2, groups=2, beams=4, vocab=10, top=8, out=P, parents=P,
             tokens=P, scratch=P, stream=None)
    a.update(over)
    return _lib.lib.functs_b200_beam_select(*a.values()), _lib.last_error()


@pytest.mark.parametrize("over,match", [
    ({"dtype": 3}, "dtype"), ({"groups": -1}, "groups"), ({"beams": 0}, "beams"), ({"beams": 65}, "beams"), ({"vocab": 0}, "vocab"), ({"top": 0}, "top"),
    ({"top": 65, "vocab": 100}, "top"), ({"top": 41}, "top"), ({"end_token": 10}, "end_token"), ({"end_token": -1}, "end_token"),
] + [({n: None}, "null pointer") for n in ("logits", "scores", "out", "parents", "tokens", "scratch")] + [({"logits": P + 1}, "boundary")]
    + [({n: P + 2}, "boundary") for n in ("scores", "out")] + [({n: P + 4}, "boundary") for n in ("parents", "tokens", "scratch")])
def test_beam_select_arguments(over, match):
    rc, why = select(**over)
    assert rc == -1 and match in why


def test_beam_select_of_nothing():
    from functs_b200 import _lib
    assert select(groups=0)[0] == 0
    assert _lib.lib.functs_b200_beam_select_scratch_bytes(0, 4, 4) == 0
    assert _lib.lib.functs_b200_beam_select_scratch_bytes(3, 4, 8) >= 3 * 4 * 8 * 8


def reorder(pools=((P, 64),), **over):
    from functs_b200 import _lib
    table = (_lib.StatePool * max(1, len(pools)))(*[_lib.StatePool(*p) for p in pools])
    a = dict(pools=table, count=len(pools), num_slots=9, parents=P, slots=P, new_slots=P, groups=2, beams=4, status=P, stream=None)
    a.update(over)
    return _lib.lib.functs_b200_beam_reorder(*a.values()), _lib.last_error()


@pytest.mark.parametrize("over,match", [
    ({"groups": -1}, "groups"), ({"beams": 0}, "beams"), ({"beams": 65}, "beams"), ({"count": -1}, "negative"), ({"num_slots": -1}, "negative"),
    ({"pools": None}, "null pointer"), ({"parents": None}, "null pointer"), ({"slots": None}, "null pointer"), ({"new_slots": None}, "null pointer"),
    ({"parents": P + 4}, "boundary"), ({"slots": P + 2}, "boundary"), ({"new_slots": P + 2}, "boundary"), ({"status": P + 2}, "boundary"),
])
def test_beam_reorder_arguments(over, match):
    if over.get("pools", 0) is None:
        from functs_b200 import _lib
        rc = _lib.lib.functs_b200_beam_reorder(None, 1, 9, P, P, P, 2, 4, P, None)
        why = _lib.last_error()
    else:
        rc, why = reorder(**over)
    assert rc == -1 and match in why


def test_beam_reorder_pools():
    assert reorder(groups=0)[0] == 0
    for pools, match in ((((None, 64),), "null pointer"), (((P, -1),), "row_bytes"), (((P, 2 ** 40 + 1),), "row_bytes"), (((P, 2 ** 39),) * 3, "too large")):
        rc, why = reorder(pools=pools, groups=1 << 20)
        assert rc == -1 and match in why


def test_there_is_no_cpu_path():
    from functs_b200 import ops
    x = torch.zeros(2, 3, 4)
    bc = torch.zeros(2, 3, 1, 5)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv(x, torch.zeros(4, 3))
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv_step(x[:, 0], torch.zeros(4, 3), torch.zeros(2, 2, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan(x, x, torch.zeros(4, 5), bc, bc)
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan_step(x[:, 0], x[:, 0], torch.zeros(4, 5), bc[:, 0], bc[:, 0], torch.zeros(2, 4, 5))
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(x, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_reorder([x], torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32))


@pytest.mark.parametrize("groups,beams", [((1 << 14) + 1, 64), ((1 << 20) // 3 + 1, 3), (1 << 20, 2)])
def test_beam_reorder_of_too_many_beams(groups, beams):
    """Every slot is compared with all that stand before it: a table has 2^20 beams at most."""
    rc, why = reorder(groups=groups, beams=beams)
    assert rc == -1 and "too large" in why
