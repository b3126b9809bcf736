"""Refusals of the sequence operators that need no GPU: wrong tensors at the Python entries, wrong arguments at the C ones (nothing is
launched, pointers are never followed)."""
import ctypes

import pytest
import torch


def args(**over):
    from functs_b200 import _lib
    p = 4096
    a = _lib.LinearAttentionArgs(dtype=2, batch=2, tokens=3, heads=4, kv_heads=2, dk=16, dv=16, num_slots=2, q=p, k=p, v=p, out=p, log_decay=p,
                                 state_in=p, state_out=p, scale=1.0)
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("over,match", [
    ({"dtype": 3}, "dtype"), ({"dtype": -1}, "dtype"), ({"batch": -1}, "negative"), ({"tokens": -1}, "negative"), ({"heads": 0}, "multiple"),
    ({"kv_heads": 3}, "multiple"), ({"kv_heads": 0}, "multiple"), ({"dk": 0}, "dk"), ({"dk": 129}, "dk"), ({"dv": 129}, "dv"),
    ({"num_slots": 3}, "as many states"), ({"num_slots": -1, "slots": 4096}, "negative"), ({"log_decay": None}, "null pointer"),
    ({"state_out": None}, "null pointer"), ({"q": None}, "null pointer"), ({"v": None}, "null pointer"), ({"out": None}, "null pointer"),
])
def test_linear_attention_arguments(over, match):
    from functs_b200 import _lib
    assert _lib.lib.functs_b200_linear_attention(ctypes.byref(args(**over)), None, None) == -1
    assert match in _lib.last_error()


def test_linear_attention_of_nothing():
    from functs_b200 import _lib
    assert _lib.lib.functs_b200_linear_attention(ctypes.byref(args(batch=0, num_slots=0)), None, None) == 0
    assert _lib.lib.functs_b200_linear_attention(None, None, None) == -1


@pytest.mark.parametrize("at,value,match", [
    (1, 3, "dtype"), (4, -1, "rows"), (5, 0, "vocab"), (6, -1, "top"), (6, 65, "top"), (6, 11, "top"), (0, None, "null pointer"), (3, None, "null pointer"),
    (7, None, "null pointer"), (8, None, "null pointer"), (9, None, "null pointer"), (10, None, "null pointer"), (0, 4097, "boundary"),
])
def test_token_logprobs_arguments(at, value, match):
    from functs_b200 import _lib
    p = 4096
    a = [p, 2, 10, p, 1, 10, 5, p, p, p, p, None, None]
    a[at] = value
    if match == "top" and value == 65:
        a[5] = 100
    assert _lib.lib.functs_b200_token_logprobs(*a) == -1
    assert match in _lib.last_error()


def test_token_logprobs_of_nothing():
    from functs_b200 import _lib
    assert _lib.lib.functs_b200_token_logprobs(None, 0, 10, None, 0, 10, 5, None, None, None, None, None, None) == 0


def test_there_is_no_cpu_path():
    from functs_b200 import ops
    x = torch.zeros(1, 2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_attention(x, x, x, torch.zeros(3))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_attention_step(x[0], x[0], x[0], torch.zeros(3), torch.zeros(2, 3, 4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))


def test_decaying_state_program_reaches_its_kernel():
    """The imperative loop (a state that decays, outputs assigned by step) is one functor bound to the attention kernels."""
    from functs_b200 import jit, patterns
    f = jit.build(patterns.DecayAttentionSeq(torch.rand(4, 1, 1)))
    assert jit.functor_regions(f.graph) == ["decay_attention_seq"]
    assert "prim::Loop" not in {n.kind() for n in f.graph.nodes()}


class OtherUpdate(torch.nn.Module):
    """The same loop with the state's halves added the other way round: another program."""

    def __init__(self, decay: torch.Tensor):
        super().__init__()
        self.decay = decay

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        outs = torch.zeros(q.size(0), q.size(1), q.size(2), v.size(3), dtype=q.dtype, device=q.device)
        s = torch.zeros(q.size(1), q.size(2), q.size(3), v.size(3), dtype=q.dtype, device=q.device)
        for t in range(q.size(0)):
            s = s * self.decay - k[t].unsqueeze(3) * v[t].unsqueeze(2)
            outs[t] = torch.matmul(q[t].unsqueeze(2), s).squeeze(2)
        return outs, s


def test_another_update_does_not_match():
    from functs_b200 import jit
    f = jit.build(OtherUpdate(torch.rand(4, 1, 1)))
    assert "decay_attention_seq" not in jit.functor_regions(f.graph)


@pytest.mark.parametrize("dtype,over", [(2, {n: 4097}) for n in ("q", "k", "v", "out")] + [(0, {n: 4098}) for n in ("q", "k", "v", "out")] +
                         [(1, {n: 4098}) for n in ("log_decay", "state_in", "state_out", "slots", "lengths", "status")])
def test_linear_attention_pointers_off_their_boundary(dtype, over):
    from functs_b200 import _lib
    assert _lib.lib.functs_b200_linear_attention(ctypes.byref(args(dtype=dtype, **over)), None, None) == -1
    assert "boundary" in _lib.last_error()


@pytest.mark.parametrize("at,value", [(3, 4100), (7, 4098), (8, 4098), (9, 4098), (10, 4100), (11, 4098)])
def test_token_logprobs_pointers_off_their_boundary(at, value):
    from functs_b200 import _lib
    a = [4096, 2, 10, 4096, 1, 10, 5, 4096, 4096, 4096, 4096, None, None]
    a[at] = value
    assert _lib.lib.functs_b200_token_logprobs(*a) == -1
    assert "boundary" in _lib.last_error()
