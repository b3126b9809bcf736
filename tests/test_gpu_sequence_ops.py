"""Attention with a decaying state and log probabilities of tokens, against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(cuda_device):
    import functs_b200
    return functs_b200.ops


# ---- attention with a decaying state: the definition --------------------------------------------------------------------


def recurrence(q, k, v, log_decay, scale, state, lengths):
    """The definition, token by token in 64 bits, and the same with every factor's magnitude (what rounding errors are relative to)."""
    b, t, h, _ = q.shape
    share = torch.arange(h, device=q.device) // (h // k.size(2))
    decay = torch.exp(log_decay.double())[None, :, None, None]
    s = torch.zeros(b, h, q.size(3), v.size(3), dtype=torch.float64, device=q.device) if state is None else state.double()
    m = s.abs()
    out = torch.zeros(b, t, h, v.size(3), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(t):
        live = (i < lengths)[:, None, None, None]
        qi, ki, vi = (torch.where(live[..., 0], x, 0.0) for x in (q[:, i].double(), k[:, i].double()[:, share], v[:, i].double()[:, share]))
        step = ki[..., None] * vi[..., None, :]
        s = torch.where(live, decay * s + step, s)
        m = torch.where(live, decay * m + step.abs(), m)
        out[:, i] = (qi[..., None, :] @ s)[..., 0, :] * scale * live[..., 0]
        mag[:, i] = (qi.abs()[..., None, :] @ m)[..., 0, :] * abs(scale) * live[..., 0]
    return out, s, mag, m


def check_attention(got_out, got_state, want, dtype, tokens, dk):
    """Errors are bounded relative to the sum of the magnitudes of the terms.  In 32 bits every token adds at most four roundings of 2^-24
    to what is carried (the product with the decay, the sum, and two units of the decay itself), the dot product dk.  Beside that, 16-bit
    types may hold the states and the weights of a chunk as two parts of eight bits each for the product that makes `out` (2^-17 per
    factor, two factors), and `out` is rounded once (half a step)."""
    out, state, mag, m = want
    carried = (4 * tokens + dk + 8) * 2.0 ** -24
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tol = half * out.abs() + (carried + (0.0 if dtype == F32 else 2.0 ** -15)) * mag + (torch.finfo(dtype).tiny if dtype != F32 else 0.0)
    err = (got_out.double() - out).abs()
    assert bool((err <= tol).all()), f"out: error {float((err - tol).max()):.3g} over its bound"
    assert bool(((got_state.double() - state).abs() <= carried * m).all()), "state outside its bound"
    # and together: far inside the bounds above
    off = float((got_state.double() - state).norm()) / max(float(state.norm()), 1e-30)
    assert off <= 1e-6, f"state: {off:.3g} off"
    if dtype == F32:
        off = float(err.norm()) / max(float(out.norm()), 1e-30)
        assert off <= 1e-6, f"out: {off:.3g} off"


def make(b, t, h, hk, dk, dv, dtype, layout="batch", seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "fused":
        x = torch.randn(b, t, h * dk + hk * (dk + dv), generator=g, device="cuda").to(dtype)
        q, k, v = x.split([h * dk, hk * dk, hk * dv], dim=-1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hk, dv))
    qkv = [torch.randn(b, t, n, d, generator=g, device="cuda").to(dtype) for n, d in ((h, dk), (hk, dk), (hk, dv))]
    if layout == "time":  # [T, B, ...] in memory
        qkv = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in qkv]
    if layout == "heads":  # [B, H, T, ...] in memory
        qkv = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in qkv]
    if layout == "odd":  # rows that no vector load fits
        qkv = [torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in qkv]
    return qkv


def decays(h, seed=1):
    return -torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=F32) / h)


SHAPES = [
    # b, t, h, hk, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 1, 3, 1, 128, 128), (3, 2, 4, 2, 17, 33), (1, 7, 2, 2, 64, 64), (2, 63, 2, 2, 128, 128), (2, 64, 2, 1, 128, 64),
    (1, 65, 3, 3, 64, 128), (3, 129, 4, 2, 80, 48), (1, 200, 2, 2, 37, 5), (1, 700, 3, 3, 128, 128), (2, 333, 2, 2, 64, 64), (2, 130, 1, 1, 96, 112), (1, 1500, 3, 1, 128, 128), (2, 2113, 1, 1, 64, 40),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prompt(ops, shape, dtype):
    b, t, h, hk, dk, dv = shape
    q, k, v = make(*shape, dtype)
    full = torch.full((b,), t, device="cuda")
    out, state = ops.linear_attention(q, k, v, decays(h), scale=dk ** -0.5)
    assert out.dtype == dtype and out.shape == (b, t, h, dv) and state.dtype == F32 and state.shape == (b, h, dk, dv)
    check_attention(out, state, recurrence(q, k, v, decays(h), dk ** -0.5, None, full), dtype, t, dk)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["fused", "time", "heads", "odd"])
@pytest.mark.parametrize("shape", [(3, 150, 4, 2, 64, 64), (2, 70, 6, 3, 128, 128), (5, 9, 4, 4, 40, 72), (4, 1300, 2, 1, 128, 64)], ids=str)
def test_prompt_lengths_pool_and_layouts(ops, shape, layout, dtype):
    """Sequences of uneven lengths (none, one, all tokens) that go on from states in any order; rows behind them are not read."""
    b, t, h, hk, dk, dv = shape
    q, k, v = make(*shape, dtype, layout)
    lengths = torch.tensor([t, 0, 1, t // 2, 3][:b], device="cuda", dtype=torch.int32)
    pool = torch.randn(b + 4, h, dk, dv, device="cuda")
    slots = torch.randperm(b + 4, device="cuda")[:b].to(torch.int32)
    start, before = pool[slots.long()].clone(), pool.clone()
    want = recurrence(q, k, v, decays(h), 0.3, start, lengths)
    for i in range(b):
        for x in (q, k, v):
            x[i, int(lengths[i]):] = math.nan
    out, state = ops.linear_attention(q, k, v, decays(h), scale=0.3, state=pool, slots=slots, lengths=lengths)
    assert state.data_ptr() == pool.data_ptr()
    check_attention(out, pool[slots.long()], want, dtype, t, dk)
    for i in range(b):
        assert bool((out[i, int(lengths[i]):] == 0).all())
    others = torch.ones(b + 4, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert torch.equal(pool[others], before[others])
    assert torch.equal(pool[slots[1].long()], start[1])  # (no tokens: the state as it was)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 512, 16, 8, 64, 64), (1, 513, 16, 16, 128, 128), (2, 256, 4, 4, 128, 128), (3, 320, 5, 5, 100, 36), (1, 1024, 16, 2, 64, 128)],
                         ids=str)
def test_prompts_in_parts_of_one_or_two_chunks(ops, shape, dtype):
    """Long prompts of few heads are cut into parts, some of one chunk: lengths that end in one, at its end, and before most of them."""
    b, t, h, hk, dk, dv = shape
    q, k, v = make(*shape, dtype)
    for first in (t, 64, 65, 1, t - 1):
        lengths = torch.tensor([first, 0, 200][:b], device="cuda", dtype=torch.int32)
        pool = torch.randn(b + 1, h, dk, dv, device="cuda")
        slots = torch.arange(b, 0, -1, device="cuda", dtype=torch.int32)
        want = recurrence(q, k, v, decays(h), 0.2, pool[slots.long()].clone(), lengths)
        before = pool[0].clone()
        out, _ = ops.linear_attention(q, k, v, decays(h), scale=0.2, state=pool, slots=slots, lengths=lengths)
        check_attention(out, pool[slots.long()], want, dtype, t, dk)
        assert torch.equal(pool[0], before)
        for i in range(b):
            assert bool((out[i, int(lengths[i]):] == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 16, 16, 128, 128), (33, 12, 4, 72, 40), (7, 4, 2, 128, 17), (70, 8, 8, 64, 64)], ids=str)
def test_step(ops, shape, dtype):
    b, h, hk, dk, dv = shape
    q, k, v = (x[:, 0] for x in make(b, 1, h, hk, dk, dv, dtype, "fused"))
    pool = torch.randn(2 * b + 1, h, dk, dv, device="cuda")
    slots = torch.randperm(2 * b + 1, device="cuda")[:b].to(torch.int32)
    want = recurrence(q[:, None], k[:, None], v[:, None], decays(h), 0.5, pool[slots.long()], torch.ones(b, device="cuda"))
    before = pool.clone()
    out = ops.linear_attention_step(q, k, v, decays(h), pool, scale=0.5, slots=slots)
    check_attention(out[:, None], pool[slots.long()], want, dtype, 1, dk)
    others = torch.ones(2 * b + 1, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(73, 1, 1, 128, 128), (74, 1, 1, 128, 128), (1, 1, 1, 128, 32), (1, 2, 1, 128, 36), (3, 2, 2, 33, 124), (2, 3, 1, 3, 4),
                                   (5, 2, 2, 64, 64), (5, 2, 2, 65, 64), (40, 2, 1, 128, 127), (74, 1, 1, 127, 65), (5, 2, 2, 65, 39), (7, 3, 1, 128, 31),
                                   (5, 4, 2, 64, 33), (3, 1, 1, 1, 1), (2, 2, 2, 20, 7)], ids=str)
def test_step_of_whole_states_and_of_tiles(ops, shape, dtype):
    """Sizes on either side of those where a block takes a whole state; some slots name no sequence."""
    b, h, hk, dk, dv = shape
    q, k, v = (x[:, 0] for x in make(b, 1, h, hk, dk, dv, dtype, "fused"))
    pool = torch.randn(b + 2, h, dk, dv, device="cuda")
    slots = torch.randperm(b + 2, device="cuda")[:b].to(torch.int32)
    slots[1::3] = -1
    live = slots >= 0
    before = pool.clone()
    want = recurrence(q[:, None], k[:, None], v[:, None], decays(h), 0.5, pool[slots.clamp(min=0).long()], torch.ones(b, device="cuda"))
    out = ops.linear_attention_step(q, k, v, decays(h), pool, scale=0.5, slots=slots)
    check_attention(out[live][:, None], pool[slots[live].long()], tuple(x[live] for x in want), dtype, 1, dk)
    assert bool((out[~live] == 0).all())
    others = torch.ones(b + 2, dtype=torch.bool, device="cuda")
    others[slots[live].long()] = False
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_slots_that_are_none_out_of_range_or_named_twice(ops, tokens):
    import functs_b200
    b, h, d = 6, 2, 64
    q, k, v = make(b, tokens, h, h, d, d, BF16)
    pool = torch.randn(4, h, d, d, device="cuda")
    start = pool.clone()
    slots = torch.tensor([2, -1, 4, 2, 0, -7], device="cuda", dtype=torch.int32)
    status = ops.new_status("cuda")
    out, _ = ops.linear_attention(q, k, v, decays(h), state=pool, slots=slots, status=status)
    live = torch.tensor([0, 4], device="cuda")
    want = recurrence(q[live], k[live], v[live], decays(h), 1.0, start[[2, 0]], torch.full((2,), tokens, device="cuda"))
    check_attention(out[live], pool[[2, 0]], want, BF16, tokens, d)
    assert bool((out[[1, 2, 3, 5]] == 0).all()) and torch.equal(pool[[1, 3]], start[[1, 3]])
    assert int(status) == 4 | 8
    with pytest.raises(functs_b200.FunctsB200Error, match="out of range; an index was named twice"):
        ops.raise_on_status(status, "linear_attention")
    ok = ops.new_status("cuda")
    ops.linear_attention(q, k, v, decays(h), state=pool, slots=torch.tensor([3, -1, 1, 0, -1, 2], device="cuda", dtype=torch.int32), status=ok)
    assert int(ok) == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [5, 150])
def test_values_that_are_not_finite(ops, tokens, dtype):
    """They reach the outputs from their token on, in their own channels or rows, and nothing before them."""
    b, h, d, at = 1, 2, 64, tokens - 3
    for which in range(3):
        qkv = [x.clone() for x in make(b, tokens, h, h, d, d, dtype)]
        clean, clean_state = ops.linear_attention(*qkv, decays(h))
        qkv[which][0, at, 0, 7] = (math.nan, math.inf, -math.inf)[which]
        out, state = ops.linear_attention(*qkv, decays(h))
        assert torch.equal(out[:, :at], clean[:, :at]) and torch.equal(out[:, :, 1], clean[:, :, 1])
        bad = ~torch.isfinite(out[0, at:, 0])
        if which == 0:  # a query: its own row alone
            assert bool(bad[0].all()) and torch.equal(out[:, at + 1:], clean[:, at + 1:]) and torch.equal(state, clean_state)
        elif which == 1:  # a key: a row of the state, so every channel from here on
            assert bool(bad.all()) and bool((~torch.isfinite(state[0, 0, 7])).all())
        else:  # a value: its channel from here on
            assert bool(bad[:, 7].all()) and not bool(bad[:, :7].any()) and not bool(bad[:, 8:].any())
            assert bool((~torch.isfinite(state[0, 0, :, 7])).all()) and bool(torch.isfinite(state[0, 0, :, :7]).all())


@pytest.mark.parametrize("tokens", [3, 100])
def test_decays_at_their_ends(ops, tokens):
    """No decay, one that forgets at once (-inf), and one whose powers leave the range of fp32."""
    g = torch.tensor([0.0, -math.inf, -1e4, -60.0], device="cuda")
    q, k, v = make(2, tokens, 4, 4, 64, 64, BF16)
    state = torch.randn(2, 4, 64, 64, device="cuda")
    want = recurrence(q, k, v, g, 1.0, state, torch.full((2,), tokens, device="cuda"))
    out, state = ops.linear_attention(q, k, v, g, state=state)
    check_attention(out, state, want, BF16, tokens, 64)


def test_no_tokens_and_no_sequences(ops):
    q, k, v = make(2, 0, 2, 2, 16, 16, F32)
    state = torch.randn(2, 2, 16, 16, device="cuda")
    before = state.clone()
    out, _ = ops.linear_attention(q, k, v, decays(2), state=state)
    assert out.shape == (2, 0, 2, 16) and torch.equal(state, before)
    assert float(ops.linear_attention(q, k, v, decays(2))[1].abs().sum()) == 0.0
    q, k, v = make(0, 5, 2, 2, 16, 16, F32)
    out, state = ops.linear_attention(q, k, v, decays(2))
    assert out.shape == (0, 5, 2, 16) and state.shape == (0, 2, 16, 16)


@pytest.mark.parametrize("tokens", [4, 140])
def test_output_given_as_a_part_of_a_larger_one(ops, tokens):
    q, k, v = make(2, tokens, 3, 3, 64, 40, BF16)
    room = torch.full((2, tokens + 2, 5, 48), 7.0, device="cuda", dtype=BF16)
    part = room[:, 1:-1, 1:4, 3:43]
    out, _ = ops.linear_attention(q, k, v, decays(3), out=part)
    assert out.data_ptr() == part.data_ptr() and torch.equal(part, ops.linear_attention(q, k, v, decays(3))[0])
    room[:, 1:-1, 1:4, 3:43] = 7.0
    assert bool((room == 7).all())


def test_large_pool(ops):
    """States behind the 2^31st element."""
    h, d = 16, 128
    n = 2 ** 31 // (h * d * d) + 2
    pool = torch.empty(n, h, d, d, device="cuda")
    for tokens in (1, 90):
        q, k, v = make(1, tokens, h, h, d, d, BF16)
        pool[n - 1] = 1.0
        pool[0] = 2.0
        slots = torch.tensor([n - 1], device="cuda", dtype=torch.int32)
        want = recurrence(q, k, v, decays(h), 0.1, pool[n - 1:], torch.full((1,), tokens, device="cuda"))
        out, _ = ops.linear_attention(q, k, v, decays(h), scale=0.1, state=pool, slots=slots)
        check_attention(out, pool[n - 1:], want, BF16, tokens, d)
        assert bool((pool[0] == 2).all())


def test_attention_refuses(ops):
    q, k, v = make(2, 3, 4, 2, 16, 16, F32)
    g, state = decays(4), torch.zeros(2, 4, 16, 16, device="cuda")
    i32 = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    call = ops.linear_attention
    for error, match, f in [
        (ValueError, "CUDA tensor", lambda: call(q.cpu(), k, v, g)),
        (ValueError, "CUDA tensor", lambda: call(q, k.cpu(), v, g)),
        (TypeError, "q must be torch.float32", lambda: call(q.double(), k.double(), v.double(), g)),
        (TypeError, "k must be", lambda: call(q, k.half(), v, g)),
        (TypeError, "log_decay must be", lambda: call(q, k, v, g.half())),
        (ValueError, "log_decay must be of sizes", lambda: call(q, k, v, g[:2])),
        (ValueError, "multiple of the key", lambda: call(q[:, :, :3], k, v, g[:3])),
        (ValueError, "fit one another", lambda: call(q, k[:, :2], v, g)),
        (ValueError, "fit one another", lambda: call(q, k[..., :8], v, g)),
        (ValueError, "1 to 128 channels", lambda: call(*[torch.zeros(1, 1, 1, 129, device="cuda")] * 3, g[:1])),
        (ValueError, "state must be a contiguous", lambda: call(q, k, v, g, state=state[..., :8])),
        (ValueError, "without slots", lambda: call(q, k, v, g, state=state[:1])),
        (ValueError, "give one", lambda: call(q, k, v, g, slots=i32(0, 1))),
        (TypeError, "slots must be", lambda: call(q, k, v, g, state=state, slots=torch.tensor([0, 1], device="cuda"))),
        (ValueError, "slots must be of sizes", lambda: call(q, k, v, g, state=state, slots=i32(0))),
        (ValueError, "lengths must be of sizes", lambda: call(q, k, v, g, lengths=i32(0, 1, 2))),
        (ValueError, "out must not share", lambda: call(q, k, v, g, out=q)),
        (ValueError, "overlap itself", lambda: call(q, k, v, g, out=torch.zeros(1, 1, 4, 16, device="cuda").expand(2, 3, 4, 16))),
        (ValueError, "status must be", lambda: call(q, k, v, g, status=torch.zeros(1, device="cuda"))),
        (NotImplementedError, "gradient", lambda: call(q.clone().requires_grad_(), k, v, g)),
        (ValueError, r"\[B, heads, channels\]", lambda: ops.linear_attention_step(q, k, v, g, state)),
    ]:
        with pytest.raises(error, match=match):
            f()
    with torch.no_grad():
        call(q.clone().requires_grad_(), k, v, g)


def test_prompt_then_tokens_is_the_whole_prompt(ops):
    """A prompt, then single tokens from the pool it left (captured into a graph and replayed, with a second one that shares nothing), and
    the log probabilities of what they answer: the same as one prompt of all tokens."""
    b, t, n, h, d, vocab = 3, 100, 6, 4, 64, 1000
    q, k, v = make(b, t + n, h, h, d, d, BF16, "fused")
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    w = torch.randn(h * d, vocab, device="cuda", dtype=BF16) * 0.3
    whole, end = ops.linear_attention(q, k, v, decays(h), scale=d ** -0.5)
    pool = torch.zeros(5, h, d, d, device="cuda")
    ops.linear_attention(q[:, :t], k[:, :t], v[:, :t], decays(h), scale=d ** -0.5, state=pool, slots=slots)
    one = [torch.empty(b, x.size(2), x.size(3), device="cuda", dtype=BF16) for x in (q, k, v)]
    ids = torch.zeros(b, dtype=torch.int64, device="cuda")
    g = decays(h)

    def step(pool):
        o = ops.linear_attention_step(*one, g, pool, scale=d ** -0.5, slots=slots)
        return (o,) + tuple(ops.token_logprobs(o.flatten(1) @ w, ids, top=3))

    spare = pool.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for p in (pool, spare):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got = step(p)
        graphs.append(got)
    for i in range(n):
        for x, y in zip(one, (q, k, v)):
            x.copy_(y[:, t + i])
        ids.copy_((whole[:, t + i].flatten(1) @ w).argmax(1))
        graphs[0].replay()
        graphs[2].replay()
        for got in (graphs[1], graphs[3]):
            o, lp, entropy, top_lp, top_ids = got
            # one more rounding of what the prompt carried: two halves of a step apart at most, beside what is carried
            assert float((o.double() - whole[:, t + i].double()).norm()) <= 2 * 2.0 ** -8 * float(whole[:, t + i].double().norm())
            want = torch.log_softmax((o.flatten(1) @ w).double(), 1)
            assert torch.allclose(lp.double(), want.gather(1, ids[:, None])[:, 0], atol=1e-4)
            assert torch.equal(top_ids, torch.sort((o.flatten(1) @ w).float(), dim=1, descending=True, stable=True)[1][:, :3])
    for p in (pool, spare):
        assert float((p[slots.long()] - end).norm()) <= 2e-6 * float(end.norm())


def test_two_streams_at_once(ops):
    """Calls on two streams do not touch one another."""
    cases = [make(2, 300, 4, 4, 128, 128, BF16, seed=s) for s in (1, 2)]
    want = [ops.linear_attention(*c, decays(4)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(ops.linear_attention(*c, decays(4)))
        torch.cuda.synchronize()
        for (o, s), (wo, ws) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(s, ws)


# ---- log probabilities -----------------------------------------------------------------------------------------------


def check_logprobs(ops, logits, tokens, top):
    """A sum of V powers: each within 2^-22 of its value and, for its exponent, |d| 2^-24 (d within 2^8 of the maximum, beyond that
    it is nothing), at most V / 64 additions in one thread and 32 more above.  The logarithm turns that into an absolute error."""
    rows, vocab = logits.shape
    x = logits.double()
    want_ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    lp, entropy, top_lp, top_ids = ops.token_logprobs(logits, tokens, top=top)
    assert lp.dtype == entropy.dtype == top_lp.dtype == F32 and top_ids.dtype == torch.int64 and top_ids.shape == (rows, top)
    assert torch.equal(top_ids, want_ids)
    p = torch.log_softmax(x, dim=1)
    eps = 2.0 ** -22 + (vocab / 64 + 32 + 2 ** 8) * 2.0 ** -24
    tol = lambda want: eps + 2.0 ** -24 * want.abs()  # noqa: E731
    want = p.gather(1, tokens[:, None])[:, 0]
    fine = torch.isfinite(want)
    assert torch.equal(lp[~fine].double(), want[~fine])
    assert bool(((lp.double() - want).abs() <= tol(want))[fine].all())
    want = p.gather(1, want_ids)
    fine = torch.isfinite(want)
    assert torch.equal(top_lp[~fine].double(), want[~fine])
    assert bool(((top_lp.double() - want).abs() <= tol(want))[fine].all())
    want = -torch.where(p > -math.inf, p.exp() * p, 0.0).sum(1)
    # two sums of that kind, one of them of terms |d| e^d
    assert bool(((entropy.double() - want).abs() <= 2 * eps * (1 + want) + 2.0 ** -24 * want).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 3, 3), (3, 64, 64), (2, 100, 50), (5, 369, 5), (1, 32000, 5), (2, 32001, 64), (40, 4097, 7),
                                            (300, 5003, 20), (3, 262144, 20), (200, 1000, 0)])
def test_logprobs(ops, rows, vocab, top, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    check_logprobs(ops, logits, torch.randint(0, vocab, (rows,), generator=g, device="cuda"), top)


@pytest.mark.parametrize("top", [0, 1, 64])
@pytest.mark.parametrize("rows,vecs", [(1, 8191), (1, 8192), (37, 8193), (38, 8192), (74, 8200), (75, 8192), (3, 16385), (148, 600)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_of_rows_around_those_that_are_shared(ops, rows, vecs, top, dtype):
    """Rows as long as those that several blocks share, a little shorter and longer, on every boundary (the row before them is longer)."""
    vocab = vecs * 16 // dtype.itemsize
    g = torch.Generator(device="cuda").manual_seed(vecs)
    for less in (0, 3):
        x = (torch.randn(rows, vocab + 1, generator=g, device="cuda") * 3).to(dtype)[:, :vocab - less]
        check_logprobs(ops, x, torch.randint(0, vocab - less, (rows,), generator=g, device="cuda"), top)


@pytest.mark.parametrize("kind", ["constant", "one part", "last part", "few finite", "none but one"])
@pytest.mark.parametrize("rows", [2, 60])
def test_logprobs_of_shared_rows_that_are_hard_to_select_from(ops, kind, rows):
    vocab, top = 70003, 64
    at = torch.arange(vocab, device="cuda")
    x = torch.randn(rows, vocab, device="cuda")
    if kind == "constant":
        x = torch.full((rows, vocab), 1.25, device="cuda")
    elif kind == "one part":  # all alternatives lie in one of the parts
        x = torch.where((at > 18000) & (at < 18100), x + 50, x)
    elif kind == "last part":
        x = torch.where(at >= vocab - 64, x + 50, x)
    elif kind == "few finite":  # fewer than asked for, in two parts
        x[:, 5:vocab - 5] = -math.inf
    elif kind == "none but one":
        x = torch.full((rows, vocab), -math.inf, device="cuda")
        x[:, 69999] = -4.0
    check_logprobs(ops, x.to(BF16).contiguous(), torch.randint(0, vocab, (rows,), device="cuda"), top)


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["constant", "two values", "rising", "falling", "few finite", "one finite", "few threads", "shifted", "huge range", "zeros"])
def test_logprobs_of_rows_that_are_hard_to_select_from(ops, kind, dtype, rows):
    vocab, top = 40000, 20
    at = torch.arange(vocab, device="cuda", dtype=F32)
    x = torch.randn(rows, vocab, device="cuda")
    if kind == "constant":
        x = torch.full((rows, vocab), -3.5, device="cuda")
    elif kind == "two values":
        x = torch.where(x > 1.5, 1.0, 0.25)
    elif kind == "rising":
        x = (at / 1000).repeat(rows, 1)
    elif kind == "falling":
        x = (-at / 1000).repeat(rows, 1)
    elif kind == "few finite":
        x[:, 7:] = -math.inf
    elif kind == "one finite":
        x = torch.full((rows, vocab), -math.inf, device="cuda")
        x[:, 31234] = 2.0
    elif kind == "few threads":  # the large values all sit where a handful of threads read
        x = torch.where((at // 4) % 128 < 4, x.abs() + 10, x)
    elif kind == "shifted":
        x = x * 5 + 1000
    elif kind == "huge range":
        x = x * 1e4
    elif kind == "zeros":  # of both signs: equal, the lowest ids first
        x = torch.where(x > 0, 0.0, -0.0)
    check_logprobs(ops, x.to(dtype).contiguous(), torch.randint(0, vocab, (rows,), device="cuda"), top)


@pytest.mark.parametrize("vocab", [50, 9000])
def test_logprobs_of_rows_without_a_distribution(ops, vocab):
    x = torch.randn(6, vocab, device="cuda")
    x[0] = -math.inf
    x[1, 17] = math.nan
    x[2, 23] = math.inf
    x[3, 40] = -math.nan
    tokens = torch.tensor([3, 4, 23, 40, 5, 49], device="cuda")
    lp, entropy, top_lp, top_ids = ops.token_logprobs(x, tokens, top=4)
    assert float(lp[0]) == -math.inf and float(entropy[0]) == 0.0 and bool((top_lp[0] == -math.inf).all()) and top_ids[0].tolist() == [0, 1, 2, 3]
    for r, first in ((1, 17), (2, 23), (3, 40)):
        assert math.isnan(float(lp[r])) and math.isnan(float(entropy[r])) and bool(torch.isnan(top_lp[r]).all()) and int(top_ids[r, 0]) == first
    check_logprobs(ops, x[4:], tokens[4:], 4)


@pytest.mark.parametrize("vocab,rows", [(50, 9), (1000, 40), (9001, 3), (70001, 2), (140000, 60)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["all lowest", "few left", "one left at the lowest", "two masks", "masked and -inf", "highest", "steps"])
def test_logprobs_of_logits_masked_with_large_values(ops, kind, dtype, vocab, rows):
    """Masks of the type's lowest value and of other large ones: rows that they leave something of, and nothing; and the same far above 0."""
    lowest, highest = torch.finfo(dtype).min, torch.finfo(dtype).max
    for value in (-1e9, -1e10, -3.3e20, -1e30, lowest):
        value = max(value, lowest)
        x = torch.randn(rows, vocab, device="cuda") * 3
        if kind == "all lowest":
            x[:] = value
        elif kind == "few left":
            x[:, 3:-3] = value
        elif kind == "one left at the lowest":  # the row's largest is itself a large negative number
            x[:] = lowest
            x[:, vocab // 2] = value / 2
        elif kind == "two masks":
            x[:] = value
            x[:, ::7] = lowest
        elif kind == "masked and -inf":
            x[:] = -math.inf
            x[:, 5::11] = value
        elif kind == "highest":
            x[:, 1::5] = -value  # (and none far below 0: their log probabilities would not be numbers of 32 bits)
        elif kind == "steps":  # neighbours of 2^28, 16 and 32 apart in fp32
            x[:] = -(2.0 ** 28)
            x[:, 1::3] = -(2.0 ** 28) - 32
            x[:, 2::3] = -(2.0 ** 28) + 16
            if value == lowest:
                x = -x
        x = x.clamp(lowest, highest) if kind != "masked and -inf" else x
        check_logprobs(ops, x.to(dtype).contiguous(), torch.randint(0, vocab, (rows,), device="cuda"), min(20, vocab))


def test_logprobs_tokens_that_are_none_or_out_of_range(ops):
    x = torch.randn(4, 100, device="cuda")
    status = ops.new_status("cuda")
    lp, entropy, _, _ = ops.token_logprobs(x, torch.tensor([-1, 100, 5, -100], device="cuda"), status=status)
    assert float(lp[0]) == 0.0 == float(lp[3]) and math.isnan(float(lp[1])) and int(status) == 4
    assert bool((entropy > 0).all())
    ok = ops.new_status("cuda")
    ops.token_logprobs(x, torch.tensor([-1, 99, 5, 0], device="cuda"), status=ok)
    assert int(ok) == 0


def test_logprobs_rows_in_a_larger_tensor(ops):
    """Rows apart, off every 16-byte boundary, and behind the 2^31st element."""
    for dtype in (F32, F16, BF16):
        big = torch.randn(7, 1033, device="cuda").to(dtype)
        for first in range(9):
            check_logprobs(ops, big[:, first:first + 1001], torch.arange(7, device="cuda"), 9)
    store = torch.empty(2 ** 31 + 5000, device="cuda", dtype=BF16)
    x = store.as_strided((2, 3000), (2 ** 31, 1), 11)
    x.copy_(torch.randn(2, 3000, device="cuda"))
    check_logprobs(ops, x, torch.tensor([5, 2999], device="cuda"), 5)


def test_logprobs_refuses(ops):
    x, t = torch.randn(3, 50, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int64)
    for error, match, f in [
        (ValueError, "CUDA tensor", lambda: ops.token_logprobs(x.cpu(), t)),
        (ValueError, "CUDA tensor", lambda: ops.token_logprobs(x, t.cpu())),
        (TypeError, "logits must be torch.float32", lambda: ops.token_logprobs(x.double(), t)),
        (TypeError, "tokens must be", lambda: ops.token_logprobs(x, t.int())),
        (ValueError, "rows, vocab", lambda: ops.token_logprobs(x[0], t)),
        (ValueError, "rows, vocab", lambda: ops.token_logprobs(x[:, :0], t)),
        (ValueError, "tokens must be of sizes", lambda: ops.token_logprobs(x, t[:2])),
        (ValueError, "top must be", lambda: ops.token_logprobs(x, t, top=51)),
        (ValueError, "top must be", lambda: ops.token_logprobs(x, t, top=-1)),
        (ValueError, "top must be", lambda: ops.token_logprobs(torch.randn(3, 500, device="cuda"), t, top=65)),
        (NotImplementedError, "gradient", lambda: ops.token_logprobs(x.clone().requires_grad_(), t)),
    ]:
        with pytest.raises(error, match=match):
            f()
    lp, entropy, top_lp, top_ids = ops.token_logprobs(x[:0], t[:0], top=2)
    assert lp.shape == (0,) and top_ids.shape == (0, 2)


@pytest.mark.parametrize("vocab", [200, 1000])
@pytest.mark.parametrize("kind", ["constant", "two values", "few finite", "zeros", "rising"])
def test_logprobs_of_short_rows(ops, kind, vocab):
    x = torch.randn(37, vocab, device="cuda")
    if kind == "constant":
        x = torch.full((37, vocab), 2.0, device="cuda")
    elif kind == "two values":
        x = torch.where(x > 1.5, 1.0, 0.25)
    elif kind == "few finite":
        x[:, 3:] = -math.inf
    elif kind == "zeros":
        x = torch.where(x > 0, 0.0, -0.0)
    elif kind == "rising":
        x = torch.arange(vocab, device="cuda", dtype=F32).repeat(37, 1)
    for dtype in (F32, F16, BF16):
        for top in (0, 1, 20, 64):
            check_logprobs(ops, x.to(dtype).contiguous(), torch.randint(0, vocab, (37,), device="cuda"), top)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,dv,front", [(100, 100, 0), (60, 36, 0), (64, 64, 4), (64, 64, 2), (128, 128, 1)])
def test_prompt_rows_on_other_boundaries(ops, dk, dv, front, dtype):
    """Rows on boundaries of 8, 4 and 2 bytes take other loads than those of 16."""
    b, t, h = 2, 150, 2
    x = torch.randn(b, t, h, 2 * dk + dv + 8, device="cuda").to(dtype)
    q, k, v = x[..., front:front + dk], x[..., front + dk:front + 2 * dk], x[..., front + 2 * dk:front + 2 * dk + dv]
    out, state = ops.linear_attention(q, k, v, decays(h), scale=dk ** -0.5)
    check_attention(out, state, recurrence(q, k, v, decays(h), dk ** -0.5, None, torch.full((b,), t, device="cuda")), dtype, t, dk)


@pytest.mark.parametrize("dk,dv", [(8, 16), (16, 8), (24, 40), (8, 128)])
def test_prompt_heads_narrower_than_a_tile(ops, dk, dv):
    """Boxes that reach past the channels, sequences and heads of the tensor; batches and heads of one."""
    for b, h in ((1, 1), (2, 3)):
        q, k, v = make(b, 100, h, h, dk, dv, BF16)
        out, state = ops.linear_attention(q, k, v, decays(h))
        check_attention(out, state, recurrence(q, k, v, decays(h), 1.0, None, torch.full((b,), 100, device="cuda")), BF16, 100, dk)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompt_of_shared_and_expanded_tensors(ops, dtype):
    """Keys and values of one sequence for all (stride 0), queries that share memory with them."""
    b, t, h, d = 3, 130, 2, 64
    x = torch.randn(1, t, h, d, device="cuda").to(dtype)
    q = k = v = x.expand(b, t, h, d)
    out, state = ops.linear_attention(q, k, v, decays(h), scale=0.1)
    check_attention(out, state, recurrence(q, k, v, decays(h), 0.1, None, torch.full((b,), t, device="cuda")), dtype, t, d)
    assert torch.equal(out[0], out[2])


def test_many_sequences_of_which_few_have_tokens(ops):
    b, t, h, d = 300, 70, 2, 64
    q, k, v = make(b, t, h, h, d, d, BF16)
    lengths = torch.zeros(b, device="cuda", dtype=torch.int32)
    lengths[[3, 299]] = torch.tensor([70, 5], device="cuda", dtype=torch.int32)
    out, state = ops.linear_attention(q, k, v, decays(h), lengths=lengths)
    for i in (3, 299):
        n = int(lengths[i])
        want = recurrence(q[i:i + 1], k[i:i + 1], v[i:i + 1], decays(h), 1.0, None, lengths[i:i + 1])
        check_attention(out[i:i + 1], state[i:i + 1], want, BF16, n, d)
    others = lengths == 0
    assert bool((out[others] == 0).all()) and bool((state[others] == 0).all())


def test_first_call_in_a_capture(cuda_device):
    """A process whose first prompt is captured into a graph."""
    import subprocess
    import sys
    code = """
import torch
from functs_b200 import ops
q, k, v = (torch.randn(1, 200, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3))
g = torch.tensor([-0.1, -0.5], device="cuda")
x, ids = torch.randn(2, 5000, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, state = ops.linear_attention(q, k, v, g)
    lp = ops.token_logprobs(x, ids, top=3)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
want = ops.linear_attention(q, k, v, g)
assert torch.equal(out, want[0]) and torch.equal(state, want[1])
assert all(torch.equal(a, b) for a, b in zip(lp, ops.token_logprobs(x, ids, top=3)))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("steps,batch,heads,dk,dv", [(1, 1, 1, 4, 4), (20, 2, 3, 16, 24), (300, 2, 4, 64, 64), (0, 2, 2, 8, 8)])
def test_decaying_state_program_through_the_graph(ops, steps, batch, heads, dk, dv):
    """The imperative program, built, against its own loop in 64 bits; time-major tensors, one functor, no interpreted run."""
    from functs_b200 import jit, launch_count, patterns
    decay = (1 - torch.exp2(-torch.arange(heads, dtype=F32) - 1)).reshape(heads, 1, 1)
    decay[0] = 0.0 if heads == 3 else decay[0]
    program = patterns.DecayAttentionSeq(decay)
    fn = jit.build(program)
    assert jit.functor_regions(fn.graph) == ["decay_attention_seq"]
    q, k, v = (torch.randn(steps, batch, heads, d, device="cuda") for d in (dk, dk, dv))
    before = jit.interpreted_functor_runs()
    outs, s = fn(q, k, v)
    launches = launch_count()
    outs, s = fn(q, k, v)
    assert jit.interpreted_functor_runs() == before and launch_count() - launches <= 3
    want, want_s = patterns.DecayAttentionSeq(decay.double())(*(x.double().cpu() for x in (q, k, v)))
    mag, mag_s = patterns.DecayAttentionSeq(decay.double())(*(x.double().cpu().abs() for x in (q, k, v)))
    # (as above; the decay goes through its logarithm, which costs it another 2^-24 per token)
    tol = (5 * steps + dk + 8) * 2.0 ** -24
    assert outs.shape == want.shape and bool(((outs.cpu().double() - want).abs() <= tol * mag).all())
    assert bool(((s.cpu().double() - want_s).abs() <= tol * mag_s).all())


def test_decaying_state_program_that_does_not_fit_the_kernels(ops):
    """Other types, wide heads and decays above one run as before there was a kernel: step by step."""
    from functs_b200 import jit, patterns
    for decay, dtype, d in ((0.5, torch.float64, 16), (0.5, F32, 144), (1.5, F32, 16)):
        decay = torch.full((2, 1, 1), decay, device="cuda", dtype=dtype if dtype == torch.float64 else F32)
        fn = jit.build(patterns.DecayAttentionSeq(decay))
        q, k, v = (torch.randn(5, 1, 2, d, device="cuda", dtype=dtype) for _ in range(3))
        before = jit.interpreted_functor_runs()
        outs, s = fn(q, k, v)
        assert jit.interpreted_functor_runs() > before
        want, want_s = patterns.DecayAttentionSeq(decay)(q, k, v)
        assert torch.allclose(outs, want) and torch.allclose(s, want_s)


@pytest.mark.parametrize("b,t,d", [(40, 131, 128), (6, 190, 128), (1, 3 * 64 + 5, 64), (30, 5 * 64 + 33, 64)])
def test_prompt_whose_last_chunk_is_partial_and_whose_queries_arrive_late(ops, b, t, d):
    """Three chunks and more, the last one partial: V is at hand, Q and K are not (every token's row in a page of its own, out of the cache),
    and what lies behind the sequences is NaN."""
    h = 4
    far = 2 ** 14 // h
    room = [torch.full((b, t + 40, h, far // (4 if i else 1)), math.nan, device="cuda", dtype=BF16) for i in range(2)]
    q, k = (x[:, :, :, 8:8 + d] for x in room)
    v = torch.full((b, t + 40, h, d), math.nan, device="cuda", dtype=BF16)
    for x in (q, k, v):
        x[:, :t] = torch.randn(b, t, h, d, device="cuda").to(BF16)
    lengths = torch.full((b,), t, device="cuda", dtype=torch.int32)
    want = recurrence(q[:, :t], k[:, :t], v[:, :t], decays(h), 0.1, None, lengths)
    flush = torch.empty(2 ** 28, device="cuda", dtype=torch.uint8)
    first = None
    for i in range(12):
        flush.fill_(i)
        v.sum()
        out, state = ops.linear_attention(q, k, v, decays(h), scale=0.1, lengths=lengths)
        if first is None:
            first = out, state
            check_attention(out[:, :t], state, want, BF16, t, d)
        assert torch.equal(out, first[0]) and torch.equal(state, first[1])
        assert bool((out[:, t:] == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,d", [(1, 64), (5, 64), (150, 64), (200, 128), (2048, 64)])
def test_decay_that_is_not_a_number(ops, tokens, d, dtype):
    """A NaN in one head's decay: that head's outputs and states are NaN however many tokens there are, other heads are as without it, and a
    sequence without tokens keeps its state."""
    b, h = 2, 3
    q, k, v = make(b, tokens, h, h, d, d, dtype)
    g = decays(h)
    bad = g.clone()
    bad[1] = math.nan
    for lengths in (None, torch.tensor([tokens, 0], device="cuda", dtype=torch.int32)):
        for start in (None, torch.randn(b, h, d, d, device="cuda")):
            clean, clean_state = ops.linear_attention(q, k, v, g, state=None if start is None else start.clone(), lengths=lengths)
            out, state = ops.linear_attention(q, k, v, bad, state=None if start is None else start.clone(), lengths=lengths)
            live = b if lengths is None else 1
            assert bool(torch.isnan(out[:live, :, 1]).all()) and bool(torch.isnan(state[:live, 1]).all())
            assert torch.equal(out[:, :, ::2], clean[:, :, ::2]) and torch.equal(state[:, ::2], clean_state[:, ::2])
            assert torch.equal(out[live:], clean[live:]) and torch.equal(state[live:], clean_state[live:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t", [8192, 4000])
def test_slow_decays_over_many_parts(ops, t, dtype):
    """A state that outlives a long prompt, which is cut into parts.  Its tokens add next to nothing, so that the error is the decay's: of
    every token's or part's factor at most half a step if it is rounded apart from the others (random, so sqrt(128) * 2^-24 = 6.7e-7 for
    128 factors), and 2^-25 * 128 = 3.8e-6 if it is the same every time."""
    h, d = 2, 64
    g = torch.tensor([-1.59e-7, -1e-4], device="cuda")
    for g in (g, torch.tensor([0.0, -1e-5], device="cuda"), torch.tensor([-2.3e-6, -3.7e-4], device="cuda")):
        q, k, v = make(1, t, h, h, d, d, dtype)
        k, v = k * 2.0 ** -10, v * 2.0 ** -10
        start = torch.randn(1, h, d, d, device="cuda") * 100
        state = start.clone()
        want = recurrence(q, k, v, g, 0.1, start, torch.full((1,), t, device="cuda"))
        out, _ = ops.linear_attention(q, k, v, g, scale=0.1, state=state)
        check_attention(out, state, want, dtype, t, d)
        for i in range(h):
            assert float((state[:, i].double() - want[1][:, i]).norm()) <= 1e-6 * float(want[1][:, i].norm())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,t,h,d", [(2, 60, 2, 64), (2, 200, 2, 128), (1, 2048, 2, 64)])
def test_waits_that_run_out(ops, b, t, h, d, dtype):
    """With the state never announced the waits for it run out: the kernel ends all the same, with no product and no copy under way, says so to
    the caller's status word, or else to the next call once, and the one after that is as ever."""
    import functs_b200
    from functs_b200 import _lib
    q, k, v = make(b, t, h, h, d, d, dtype)
    want = ops.linear_attention(q, k, v, decays(h))
    status = ops.new_status("cuda")
    drop = lambda on: _lib.check(_lib.lib.functs_b200_debug_set(b"linattn_drop_state", on), "debug_set")  # noqa: E731
    for given in (status, None):
        drop(1)
        try:
            ops.linear_attention(q, k, v, decays(h), status=given)
        finally:
            drop(0)
        torch.cuda.synchronize()
        if given is not None:
            with pytest.raises(functs_b200.FunctsB200Error, match="wait ran out"):
                ops.raise_on_status(status, "linear_attention")
        else:
            with pytest.raises(RuntimeError, match="wait ran out in an earlier call"):
                ops.linear_attention(q, k, v, decays(h))
        for _ in range(2):
            got = ops.linear_attention(q, k, v, decays(h))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_a_wait_that_ran_out_is_told_on_its_own_device(ops):
    from functs_b200 import _lib
    q, k, v = make(1, 200, 2, 2, 64, 64, BF16)
    drop = lambda on: _lib.check(_lib.lib.functs_b200_debug_set(b"linattn_drop_state", on), "debug_set")  # noqa: E731
    drop(1)
    try:
        ops.linear_attention(q, k, v, decays(2))
    finally:
        drop(0)
    torch.cuda.synchronize()
    ops.linear_attention(*(x.to("cuda:1") for x in (q, k, v, decays(2))))
    with pytest.raises(RuntimeError, match="wait ran out in an earlier call on cuda:0"):
        ops.linear_attention(q, k, v, decays(2))


def test_inputs_that_carry_a_tangent(ops):
    """Forward derivatives are refused, not lost; a built program runs step by step, so that the state keeps them (the immutable assignment of
    `outs` has never had any)."""
    import torch.autograd.forward_ad as fwd
    from functs_b200 import jit, patterns
    q, k, v = make(1, 70, 2, 2, 16, 16, F32)
    g, state = decays(2), torch.zeros(1, 2, 16, 16, device="cuda")
    x, ids = torch.randn(2, 2000, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int64)
    decay = torch.full((2, 1, 1), 0.5, device="cuda")
    program = patterns.DecayAttentionSeq(decay)
    fn = jit.build(program)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: ops.linear_attention(dual(q), k, v, g), lambda: ops.linear_attention(q, dual(k), v, g),
                  lambda: ops.linear_attention(q, k, dual(v), g), lambda: ops.linear_attention(q, k, v, dual(g)),
                  lambda: ops.linear_attention(q, k, v, g, state=dual(state)),
                  lambda: ops.linear_attention_step(dual(q[:, 0]), k[:, 0], v[:, 0], g, state), lambda: ops.token_logprobs(dual(x), ids)):
            with pytest.raises(NotImplementedError, match="tangent"):
                f()
        before = jit.interpreted_functor_runs()
        q, k, v = q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1)
        outs, s = fn(q, dual(k), v)
        assert jit.interpreted_functor_runs() > before
        want = fwd.unpack_dual(program(q, dual(k), v)[1]).tangent
        got = fwd.unpack_dual(s).tangent
        assert got is not None and torch.allclose(got, want, atol=1e-4)
    with pytest.raises(NotImplementedError, match="transform"):
        torch.func.vmap(lambda y: ops.token_logprobs(y, ids)[0])(x[None])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,d", [(1, 64), (6, 64), (150, 128), (2048, 64)])
def test_decays_above_zero(ops, tokens, d, dtype):
    """States that grow: the same formula, and the same bounds."""
    g = torch.tensor([2.0 ** -9, 0.02 if tokens < 1000 else 0.004], device="cuda")
    q, k, v = make(2, tokens, 2, 2, d, d, dtype)
    q = q * 2.0 ** -8  # (that the outputs stay within fp16)
    start = torch.randn(2, 2, d, d, device="cuda")
    want = recurrence(q, k, v, g, 0.1, start, torch.full((2,), tokens, device="cuda"))
    out, state = ops.linear_attention(q, k, v, g, scale=0.1, state=start)
    check_attention(out, state, want, dtype, tokens, d)


@pytest.mark.parametrize("tokens", [1, 5, 150])
def test_tensors_that_are_slices_of_one_buffer(ops, tokens):
    """out and state may lie in one workspace with the inputs, beside them; where they share an element with anything that is read, or out one
    with itself, the call is refused."""
    b, h, d = 2, 2, 16
    n, states = b * tokens * h * d, b * h * d * d
    room = torch.zeros(4 * n + states + 64, device="cuda")
    q, k, v, out = (room[i * n:(i + 1) * n].view(b, tokens, h, d) for i in range(4))
    state = room[4 * n:4 * n + states].view(b, h, d, d)
    rest = room[4 * n + states:]
    g, slots, lengths, status = rest[:2], rest[2:4].view(torch.int32), rest[4:6].view(torch.int32), rest[6:7].view(torch.int32)
    for x in (q, k, v):
        x.normal_()
    g.copy_(decays(h))
    slots.copy_(torch.tensor([1, 0]))
    lengths.fill_(tokens)
    want = ops.linear_attention(q.clone(), k.clone(), v.clone(), decays(h), state=state.clone(), slots=slots.clone())
    got = ops.linear_attention(q, k, v, g, state=state, slots=slots, lengths=lengths, out=out, status=status)
    assert torch.equal(got[0], want[0]) and torch.equal(state, want[1]) and int(status) == 0
    whole = torch.zeros(n + 64, device="cuda")
    front, behind = whole[:n].view(b, tokens, h, d), whole[n - 2:n]
    with pytest.raises(ValueError, match="out must not share memory with the inputs"):
        ops.linear_attention(q, k, v, behind, out=front)
    for name in ("slots", "lengths"):
        given = {"slots": slots, "lengths": lengths, name: behind.view(torch.int32)}
        with pytest.raises(ValueError, match="out must not share memory with the inputs"):
            ops.linear_attention(q, k, v, g, state=state, out=front, **given)
        given[name] = state.view(-1)[:2].view(torch.int32)
        with pytest.raises(ValueError, match="state must not share memory with the inputs"):
            ops.linear_attention(q, k, v, g, state=state, **given)
    with pytest.raises(ValueError, match="out must not share memory with the state"):
        both = torch.zeros(n + states, device="cuda")
        ops.linear_attention(q, k, v, g, state=both[:states].view(b, h, d, d), out=both[states - 1:states - 1 + n].view(b, tokens, h, d))
    if tokens > 1:
        with pytest.raises(ValueError, match="overlap itself"):
            ops.linear_attention(q, k, v, g, out=torch.zeros(2 * n, device="cuda").as_strided((b, tokens, h, d), (tokens * h * d - 1, h * d, d, 1)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", [1, 100])
def test_views_that_negate(ops, tokens):
    """A tensor whose values are the negatives of its memory's (as the imaginary part of a conjugate is)."""
    q, k, v = make(2, tokens, 2, 2, 16, 16, F32)
    g, state = decays(2), torch.zeros(2, 2, 16, 16, device="cuda")
    neg = torch._neg_view
    want = ops.linear_attention(-q, -k, v, g)
    got = ops.linear_attention(neg(q), neg(k), v, neg(-g))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = torch.complex(torch.randn(3, 3000, device="cuda"), torch.randn(3, 3000, device="cuda"))
    ids = torch.tensor([5, 1, 2999], device="cuda")
    for view in (x.conj().imag, neg(x.real.contiguous())):
        assert view.is_neg()
        for a, b in zip(ops.token_logprobs(view, neg(-ids), top=3), ops.token_logprobs(view.clone().resolve_neg(), ids, top=3)):
            assert torch.equal(a, b)
    with pytest.raises(ValueError, match="state must not be a negated view"):
        ops.linear_attention(q, k, v, g, state=neg(state))
    with pytest.raises(ValueError, match="out must not be a negated view"):
        ops.linear_attention(q, k, v, g, out=neg(torch.zeros_like(q)))


def test_tensors_that_autograd_has_saved_and_a_call_writes(ops):
    """A backward pass through a state or an output that a later call wrote over is refused by autograd, as behind any in-place operator."""
    q, k, v = make(1, 3, 2, 2, 16, 16, F32)
    w = torch.ones(1, device="cuda", requires_grad=True)
    for tokens in (3, 1):
        for which in ("state", "out"):
            state, out = torch.ones(1, 2, 16, 16, device="cuda"), torch.ones(1, 3, 2, 16, device="cuda")
            loss = (w * (state if which == "state" else out)).sum()
            if tokens == 1:
                ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decays(2), state, out=out[:, 0])
            else:
                ops.linear_attention(q, k, v, decays(2), state=state, out=out)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():
        state = torch.zeros(1, 2, 16, 16, device="cuda")
    ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decays(2), state)
    with torch.inference_mode():
        ops.linear_attention(q, k, v, decays(2), state=state)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(5, 200), (7, 1000), (3, 5003), (40, 32000), (2, 131072), (200, 32001)])
def test_logprobs_of_confident_rows(ops, rows, vocab, dtype):
    """One logit far above the others, wherever it lies, as a model's answers mostly are.  Against its power, which is 1, the others sum to
    `rest`.  On its way into a sum of 1 and more an addend is rounded by half a step, 2^-24, and by no more than itself (leaving it out is
    one of the two neighbours): 17 times at most (3 in a vector's tree, 4 between vectors, 5 and 4 in the warp and the block, 1 for the
    logarithm's result), together by no more than `rest`.  Every power is off by less than 2^-20 of itself (its exponent, below 2^7, is
    rounded by 2^-24 of itself twice, the power by 2^-22).  The entropy has that error of ln s, the same relative to its other part, which is
    divided by s, and its own terms off by 2^-20 too.  That part's sum passes by the largest element's exponent against its rounded
    reference, r <= 2^-24 |m| log2 e, which is added and taken off again: 32 roundings between, each of half of 2^-23 r at most."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for gap in (3.0, 10.0, 16.0, 17.5, 20.0, 25.0, 30.0, 48.0):
        for base in (0.0, -30.0, 50.0):
            x = (torch.randn(rows, vocab, generator=g, device="cuda") + base).to(dtype)
            at = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
            at[0], at[-1] = vocab - 1, 0
            x[torch.arange(rows, device="cuda"), at] = base + gap + 4
            lp, entropy, top_lp, top_ids = ops.token_logprobs(x, at, top=2)
            assert torch.equal(top_ids[:, 0], at) and torch.equal(top_lp[:, 0], lp)
            assert bool((lp <= 0).all()) and bool((top_lp <= 0).all()) and bool((entropy >= 0).all())
            p = torch.log_softmax(x.double(), dim=1)
            want = p.gather(1, at[:, None])[:, 0]
            others = p.scatter(1, at[:, None], -math.inf)
            rest = torch.exp(torch.logsumexp(others, dim=1) - want)
            want = -torch.log1p(rest)  # (log_softmax itself is off by 2^-53 of the logits)
            tol = torch.minimum(rest, torch.full_like(rest, 17 * 2.0 ** -24)) + 2.0 ** -20 * rest + 2.0 ** -24 * want.abs()
            assert bool(((lp.double() - want).abs() <= tol).all()), (gap, base, float((lp.double() - want).abs().max()))
            h = -want * torch.exp(want) - (torch.exp(others) * others.clamp(min=-1e300)).sum(1)
            r = 2.0 ** -24 * x.double().abs().amax(1) * 1.4427
            assert bool(((entropy.double() - h).abs() <= tol * (1 + h) + 2.0 ** -20 * h + 32 * 2.0 ** -24 * r).all()), (gap, base, float((entropy.double() - h).abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [64, 1000, 9001, 140000])
def test_logprobs_are_not_above_zero_nor_entropies_below(ops, vocab, dtype):
    rows = 64
    r = torch.arange(rows, device="cuda")
    for kind in range(6):
        x = torch.randn(rows, vocab, device="cuda")
        if kind == 1:
            x[r, torch.randint(0, vocab, (rows,), device="cuda")] += torch.linspace(0, 90, rows, device="cuda")
        elif kind == 2:  # two that share the row
            x[r, torch.randint(0, vocab, (rows,), device="cuda")] = 30.0
            x[r, torch.randint(0, vocab, (rows,), device="cuda")] = 30.0
        elif kind == 3:  # rising, so that every element is the largest so far
            x = torch.arange(vocab, device="cuda", dtype=F32)[None] * torch.linspace(0.001, 3, rows, device="cuda")[:, None]
        elif kind == 4:  # one of many is left
            x[:] = -math.inf
            x[r, torch.randint(0, vocab, (rows,), device="cuda")] = torch.linspace(-200, 200, rows, device="cuda")
        elif kind == 5:
            x = x * 1e5
        x = x.to(dtype)
        lp, entropy, top_lp, _ = ops.token_logprobs(x, torch.randint(0, vocab, (rows,), device="cuda"), top=8)
        assert bool((lp <= 0).all()) and bool((top_lp <= 0).all()) and bool((entropy >= 0).all())
        if kind == 4:
            assert bool((entropy == 0).all()) and bool((top_lp[:, 0] == 0).all())
        check_logprobs(ops, x, torch.randint(0, vocab, (rows,), device="cuda"), 8)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_outputs_of_states_that_cancel(ops, dtype, d):
    """Two rows of the state that differ by 2^-10 of themselves, one taken from the other.  A value in [1, 2) as two parts of 8 bits: the first
    leaves 2^-8 at most, which lies in a binade whose half step is 2^-17.  So that is what a product with a query of one part is off by; of
    two (fp16) the product of the second parts, 2^-8 of each, is left out too.  Beside that fp32 sums of a few terms, 2^-21, and half a step
    of the output."""
    tokens, h = 130, 4
    q, k, v = (torch.zeros(2, tokens, h, d, device="cuda", dtype=dtype) for _ in range(3))
    q[..., 3], q[..., 7] = 1 + 2.0 ** -7, -1 - 2.0 ** -7
    if dtype == F16:
        q[..., 3], q[..., 7] = 1 + 2.0 ** -9 + 2.0 ** -10, -1 - 2.0 ** -9 - 2.0 ** -10
    state = torch.zeros(2, h, d, d, device="cuda")
    state[:, :, 3] = torch.randn(2, h, d, device="cuda")
    state[:, :, 7] = state[:, :, 3] * (1 + 2.0 ** -10 * torch.rand(2, h, d, device="cuda"))
    a, b = (q[:, 0, 0, 3].double()[:, None, None] * state[:, :, i].double() for i in (3, 7))
    out, _ = ops.linear_attention(q, k, v, torch.zeros(h, device="cuda"), state=state.clone())
    want = (a - b)[:, None]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + ((3 if dtype == F16 else 1) * 2.0 ** -17 + 2.0 ** -21) * (a.abs() + b.abs())[:, None] + torch.finfo(dtype).tiny
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("b", [2, 127, 128, 129, 1100])
def test_uneven_sequences_in_any_order(ops, b):
    """Batches on either side of those whose sequences are taken longest first."""
    t, h, d = 140, 2, 32
    q, k, v = make(b, t, h, h, d, d, BF16)
    lengths = torch.randint(0, t + 1, (b,), device="cuda", dtype=torch.int32)
    lengths[::5] = 70  # (and equal ones)
    out, state = ops.linear_attention(q, k, v, decays(h), lengths=lengths)
    check_attention(out, state, recurrence(q, k, v, decays(h), 1.0, None, lengths), BF16, t, d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [200, 1000, 3001, 40003, 140007])
def test_logprobs_of_rows_with_values_that_are_not_finite(ops, vocab, dtype):
    """A NaN of either sign or an infinity wherever it lies: in vectors, in front of and behind them, in every block's part."""
    places = [0, 1, 5, vocab // 7, vocab // 3, vocab // 2 + 1, vocab - 9, vocab - 2, vocab - 1]
    for value in (math.nan, -math.nan, math.inf):
        x = torch.randn(len(places) + 1, vocab + 1, device="cuda").to(dtype)[:, :vocab]  # (rows on every boundary)
        for r, at in enumerate(places):
            x[r, at] = value
        ids = torch.tensor(places + [3], device="cuda")
        for top in (0, 3):
            lp, entropy, top_lp, top_ids = ops.token_logprobs(x, ids, top=top)
            assert bool(torch.isnan(lp[:-1]).all()) and bool(torch.isnan(entropy[:-1]).all()) and bool(torch.isnan(top_lp[:-1]).all())
            assert bool(torch.isfinite(lp[-1])) and bool(torch.isfinite(entropy[-1]))
            if top:
                assert torch.equal(top_ids[:-1, 0], ids[:-1])
        check_logprobs(ops, x[-1:], ids[-1:], 3)
