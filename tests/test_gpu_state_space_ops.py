"""The short convolution and the selective scan, over prompts and single tokens, against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24  # one rounding in 32 bits


@pytest.fixture(scope="module")
def ops(cuda_device):
    import functs_b200
    return functs_b200.ops


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows(shape, widths, dtype, layout, gen):
    """Tensors shape + [width]: of their own, parts of one projection, time-major, or rows that no vector load fits."""
    if layout == "fused":
        return torch.randn(*shape, sum(widths), generator=gen, device="cuda").to(dtype).split(list(widths), dim=-1)
    got = [torch.randn(*shape, w, generator=gen, device="cuda").to(dtype) for w in widths]
    if layout == "time" and len(shape) == 2:
        return [x.transpose(0, 1).contiguous().transpose(0, 1) for x in got]
    if layout == "odd":
        return [torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in got]
    return got


def silu_off(y, off):
    """What an error `off` of y and its own make of y / (1 + exp(-y)): its slope is 1.1 at most; an exponential of a rounded argument is off by
    (|y| + 3) roundings, four more follow, and y^2 exp(-|y|) is 0.55 at most."""
    out = y * torch.sigmoid(y)
    return out, 1.1 * off + U * (8 * out.abs() + 0.6)


# ---- short convolution --------------------------------------------------------------------------------------------------


def conv_reference(x, weight, bias, silu, state, lengths):
    """-> out, its bound in 32 bits, the new state (exact: inputs are kept as they are)."""
    b, t, c = x.shape
    w = weight.size(1)
    line = torch.cat([torch.zeros(b, w - 1, c, dtype=x.dtype, device=x.device) if state is None else state, x], dim=1)
    d = line.double()
    y = torch.zeros(b, t, c, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    for j in range(w):
        y = y + weight[:, j].double() * d[:, j: j + t]
        mag = mag + (weight[:, j].double() * d[:, j: j + t]).abs()
    off = (w + 2) * U * mag
    if silu:
        y, off = silu_off(y, off)
    there = (torch.arange(t, device=x.device)[None] < lengths[:, None])[..., None]
    last = lengths[:, None].long() + torch.arange(w - 1, device=x.device)
    return torch.where(there, y, 0.0), torch.where(there, off, 0.0), line.gather(1, last[..., None].expand(-1, -1, c))


def check(got, want, off, dtype):
    """One rounding to the output's type on top of the bound in 32 bits."""
    tol = half_step(dtype) * (want.abs() + off) + off + torch.finfo(dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"error {float((err - tol).max()):.3g} over its bound"


CONV = [(1, 1, 1, 2), (2, 1, 8, 4), (1, 2, 5, 4), (3, 3, 64, 4), (1, 7, 33, 8), (2, 65, 130, 4), (3, 130, 1001, 4), (2, 200, 96, 3), (1, 513, 16, 5), (4, 40, 264, 6),
        (2, 33, 40, 7), (1, 1000, 2048, 4)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", CONV, ids=str)
def test_conv(ops, shape, dtype):
    b, t, c, w = shape
    gen = torch.Generator(device="cuda").manual_seed(b * 1000 + t)
    x, = rows((b, t), (c,), dtype, "batch", gen)
    weight, bias = torch.randn(c, w, generator=gen, device="cuda").to(dtype), torch.randn(c, generator=gen, device="cuda").to(dtype)
    full = torch.full((b,), t, device="cuda")
    for silu, use_bias in ((True, True), (False, False)):
        out, state = ops.causal_conv(x, weight, bias if use_bias else None, silu=silu)
        assert out.dtype == dtype and out.shape == x.shape and state.dtype == dtype and state.shape == (b, w - 1, c)
        want, off, final = conv_reference(x, weight, bias if use_bias else None, silu, None, full)
        check(out, want, off, dtype)
        assert torch.equal(state, final)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["fused", "time", "odd"])
@pytest.mark.parametrize("width", [2, 4, 8])
def test_conv_lengths_pool_and_layouts(ops, width, layout, dtype):
    """Sequences of uneven lengths (none, fewer than the state has, all) that go on from states in any order; rows behind them are not read."""
    b, t, c = 7, 90, 72
    gen = torch.Generator(device="cuda").manual_seed(width)
    x, _ = rows((b, t), (c, c), dtype, layout, gen)
    weight, bias = torch.randn(c, width, generator=gen, device="cuda").to(dtype), torch.randn(c, generator=gen, device="cuda").to(dtype)
    lengths = torch.tensor([t, 0, 1, 2, 5, 64, 200], device="cuda", dtype=torch.int32)
    taken = lengths.clamp(0, t)
    pool = torch.randn(b + 3, width - 1, c, generator=gen, device="cuda").to(dtype)
    slots = torch.randperm(b + 3, generator=gen, device="cuda")[:b].to(torch.int32)
    before = pool.clone()
    want, off, final = conv_reference(x, weight, bias, True, before[slots.long()], taken)
    for i in range(b):
        x[i, int(taken[i]):] = math.nan
    out, state = ops.causal_conv(x, weight, bias, silu=True, state=pool, slots=slots, lengths=lengths)
    assert state.data_ptr() == pool.data_ptr()
    check(out, want, off, dtype)
    expect = before.clone()
    expect[slots.long()] = final
    assert torch.equal(pool, expect)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 4), (5, 33, 2), (70, 264, 4), (192, 1000, 8)], ids=str)
def test_conv_step_is_a_prompt_of_one_token(ops, shape, dtype):
    b, c, w = shape
    gen = torch.Generator(device="cuda").manual_seed(c)
    x, _ = rows((b,), (c, c), dtype, "fused", gen)
    weight, bias = torch.randn(c, w, generator=gen, device="cuda").to(dtype), torch.randn(c, generator=gen, device="cuda").to(dtype)
    pool = torch.randn(2 * b, w - 1, c, generator=gen, device="cuda").to(dtype)
    slots = torch.randperm(2 * b, generator=gen, device="cuda")[:b].to(torch.int32)
    before = pool.clone()
    out = ops.causal_conv_step(x, weight, pool, bias, silu=True, slots=slots)
    want, off, final = conv_reference(x[:, None], weight, bias, True, before[slots.long()], torch.ones(b, device="cuda"))
    check(out[:, None], want, off, dtype)
    before[slots.long()] = final
    assert torch.equal(pool, before)


def test_conv_of_values_that_are_not_finite(ops):
    """A NaN or an infinity reaches the width's tokens behind it, of its channel alone, whatever the weights."""
    x = torch.zeros(1, 20, 16, device="cuda", dtype=BF16)
    weight = torch.zeros(16, 4, device="cuda", dtype=BF16)
    weight[:, 3] = 1.0
    x[0, 5, 3], x[0, 7, 9] = math.nan, math.inf
    out, state = ops.causal_conv(x, weight)
    bad = ~torch.isfinite(out[0])
    want = torch.zeros(20, 16, dtype=torch.bool, device="cuda")
    want[5:9, 3] = want[7:11, 9] = True
    assert torch.equal(bad, want) and bool((out[0][~want] == 0).all())


# ---- selective scan: the definition ----------------------------------------------------------------------------------------


def recurrence(x, dt, A, B, C, D, z, bias, softplus, state, lengths):
    """The definition, token by token in 64 bits, with a bound of what 32 bits make of it: out, its bound, state, its bound.

    A decay is an exponential of a rounded argument: off by 2^-22 and by |d A| roundings (its own two, and those of d); d is off by `grain`: its sum
    with the bias, and, with softplus, an exponential and a logarithm of three roundings each.  A token adds two roundings of what is carried and three of
    what it adds."""
    b, t, c = x.shape
    n, g = A.size(1), B.size(2)
    share = torch.arange(c, device=x.device) // (c // g)
    h = torch.zeros(b, c, n, dtype=torch.float64, device=x.device) if state is None else state.double()
    off = torch.zeros_like(h)
    out = torch.zeros(b, t, c, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    a64 = A.double()
    for i in range(t):
        live = (i < lengths)[:, None]
        xi, v, bi, ci = (torch.where(live if q.dim() == 2 else live[..., None], q, 0.0) for q in
                         (x[:, i].double(), dt[:, i].double(), B[:, i].double()[:, share], C[:, i].double()[:, share]))
        if bias is not None:
            v = v + bias.double()
        d = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
        grain = (2 + v.abs() + (8 if softplus else 0)) * U if softplus else U * torch.ones_like(v)
        da = (d[..., None] * a64).clamp(max=80.0)
        decay = torch.exp(da)
        add = (d * xi)[..., None] * bi
        new = decay * h + add
        new_off = decay * off + (decay * h).abs() * (4 * U + 2 * U + da.abs() * (2 * U + grain[..., None])) + add.abs() * (grain[..., None] + 3 * U) + new.abs() * U
        h = torch.where(live[..., None], new, h)
        off = torch.where(live[..., None], new_off, off)
        y = (h * ci).sum(-1)
        e = (off * ci.abs()).sum(-1) + (n + 3) * U * (h * ci).abs().sum(-1)
        if D is not None:
            y = y + D.double() * xi
            e = e + 2 * U * (D.double() * xi).abs()
        e = e + U * y.abs()
        if z is not None:
            gate, gate_off = silu_off(torch.where(live, z[:, i].double(), 0.0), 0.0)
            y, e = y * gate, e * gate.abs() + y.abs() * gate_off + U * (y * gate).abs()
        out[:, i] = torch.where(live, y, 0.0)
        bound[:, i] = torch.where(live, e, 0.0)
    return out, bound, h, off


def check_scan(got_out, got_state, want, dtype):
    out, bound, state, off = want
    check(got_out, out, bound, dtype)
    err = (got_state.double() - state).abs()
    assert bool((err <= off + torch.finfo(F32).tiny).all()), f"state: error {float((err - off).max()):.3g} over its bound"
    rel = float(err.norm()) / max(float(state.norm()), 1e-30)
    assert rel <= 1e-6, f"state: {rel:.3g} off"  # (together: far inside the bound of each)


def make(b, t, c, n, g, dtype, layout="batch", seed=1, span=0.1):
    """Steps up to `span`, rates about -1 .. -n: memories of a token up to some hundred."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (b, t)
    x, z = rows(shape, (c, c), dtype, layout, gen)
    dt, bm, cm = rows(shape, (c, g * n, g * n), dtype, layout, gen)
    bias = torch.log(torch.expm1(torch.rand(c, generator=gen, device="cuda") * span + 1e-3))
    A = -torch.arange(1, n + 1, device="cuda", dtype=F32) * torch.exp(0.2 * torch.randn(c, n, generator=gen, device="cuda"))
    D = torch.randn(c, generator=gen, device="cuda")
    return x, dt, A, bm.unflatten(-1, (g, n)), cm.unflatten(-1, (g, n)), D, z, bias


SCAN = [
    # b, t, c, n, g
    (1, 1, 1, 1, 1), (2, 1, 8, 16, 1), (1, 2, 33, 3, 3), (3, 31, 40, 4, 2), (2, 32, 64, 8, 1), (1, 33, 100, 16, 4), (2, 100, 130, 5, 1), (1, 64, 36, 32, 1),
    (1, 65, 12, 64, 2), (2, 40, 20, 33, 1), (1, 300, 256, 16, 1), (1, 1200, 48, 16, 2), (1, 2100, 17, 7, 1), (5, 150, 520, 16, 1),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SCAN, ids=str)
def test_scan(ops, shape, dtype):
    b, t, c, n, g = shape
    x, dt, A, B, C, D, z, bias = make(*shape, dtype)
    full = torch.full((b,), t, device="cuda")
    out, state = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True)
    assert out.dtype == dtype and out.shape == x.shape and state.dtype == F32 and state.shape == (b, c, n)
    check_scan(out, state, recurrence(x, dt, A, B, C, D, z, bias, True, None, full), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 70, 40, 16, 1), (1, 400, 24, 6, 2)], ids=str)
def test_scan_without_what_is_optional(ops, shape, dtype):
    """Steps as they come (some negative: a state that grows), no gate, no direct term."""
    b, t, c, n, g = shape
    x, dt, A, B, C, _, _, _ = make(*shape, dtype)
    dt = dt.abs() * 0.05 - 0.005
    out, state = ops.selective_scan(x, dt, A, B, C)
    check_scan(out, state, recurrence(x, dt, A, B, C, None, None, None, False, None, torch.full((b,), t, device="cuda")), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["fused", "time", "odd"])
@pytest.mark.parametrize("shape", [(7, 150, 72, 16, 2), (6, 40, 33, 5, 1), (3, 1100, 20, 16, 1)], ids=str)
def test_scan_lengths_pool_and_layouts(ops, shape, layout, dtype):
    """Sequences of uneven lengths (none, one, all tokens) that go on from states in any order; rows behind them are not read."""
    b, t, c, n, g = shape
    x, dt, A, B, C, D, z, bias = make(*shape, dtype, layout)
    lengths = torch.tensor([t, 0, 1, t // 2, 33, t - 1, 5000][:b], device="cuda", dtype=torch.int32)
    taken = lengths.clamp(0, t)
    pool = torch.randn(b + 3, c, n, device="cuda")
    slots = torch.randperm(b + 3, device="cuda")[:b].to(torch.int32)
    before = pool.clone()
    want = recurrence(x, dt, A, B, C, D, z, bias, True, before[slots.long()], taken)
    for i in range(b):
        for q in (x, dt, B, C, z):
            q[i, int(taken[i]):] = math.nan
    out, state = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True, state=pool, slots=slots, lengths=lengths)
    assert state.data_ptr() == pool.data_ptr()
    check_scan(out, pool[slots.long()], want, dtype)
    others = torch.ones(b + 3, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert torch.equal(pool[others], before[others])
    assert torch.equal(pool[slots[1].long()], before[slots[1].long()])  # (no tokens: the state as it was)
    for i in range(b):
        assert bool((out[i, int(taken[i]):] == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 4096, 16, 1), (33, 100, 16, 4), (7, 33, 5, 1), (70, 264, 64, 2), (130, 40, 8, 1), (9, 50, 20, 1)], ids=str)
def test_scan_step(ops, shape, dtype):
    b, c, n, g = shape
    x, dt, A, B, C, D, z, bias = make(b, 1, c, n, g, dtype, "fused")
    pool = torch.randn(2 * b + 1, c, n, device="cuda")
    slots = torch.randperm(2 * b + 1, device="cuda")[:b].to(torch.int32)
    before = pool.clone()
    want = recurrence(x, dt, A, B, C, D, z, bias, True, before[slots.long()], torch.ones(b, device="cuda"))
    out = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], pool, D=D, z=z[:, 0], dt_bias=bias, softplus=True, slots=slots)
    check_scan(out[:, None], pool[slots.long()], want, dtype)
    others = torch.ones(2 * b + 1, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert torch.equal(pool[others], before[others])
    bare = ops.selective_scan_step(x[:, 0], dt[:, 0] * 0.02, A, B[:, 0], C[:, 0], before[slots.long()].clone())
    want = recurrence(x, dt * 0.02, A, B, C, None, None, None, False, before[slots.long()], torch.ones(b, device="cuda"))
    check(bare[:, None], want[0], want[1], dtype)


@pytest.mark.parametrize("shape", [(600, 1024, 16, 1), (700, 8192, 1, 1), (65, 2052, 20, 2)], ids=str)
def test_scan_step_of_many_sequences(ops, shape):
    """Blocks that go through many sequences, some of which are none."""
    b, c, n, g = shape
    x, dt, A, B, C, D, z, bias = make(b, 1, c, n, g, BF16, "fused")
    pool = torch.randn(b + 5, c, n, device="cuda")
    slots = torch.randperm(b + 5, device="cuda")[:b].to(torch.int32)
    slots[3::7] = -1
    slots[5], slots[b - 1] = b + 5, slots[0]
    live = slots >= 0
    live[5] = live[b - 1] = False
    before = pool.clone()
    want = recurrence(x, dt, A, B, C, D, z, bias, True, before[slots.clamp(0, b + 4).long()], torch.ones(b, device="cuda"))
    status = ops.new_status("cuda")
    out = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], pool, D=D, z=z[:, 0], dt_bias=bias, softplus=True, slots=slots, status=status)
    check_scan(out[live][:, None], pool[slots[live].long()], tuple(w[live] for w in want), BF16)
    assert bool((out[~live] == 0).all()) and int(status) == 4 | 8
    others = torch.ones(b + 5, dtype=torch.bool, device="cuda")
    others[slots[live].long()] = False
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("tokens", [7, 600])
def test_more_sequences_than_are_put_in_order(ops, tokens):
    b, c, n = 40, 24, 16
    x, dt, A, B, C, D, z, bias = make(b, tokens, c, n, 1, F32)
    weight = torch.randn(c, 4, device="cuda")
    lengths = torch.randint(0, tokens + 1, (b,), generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
    out, state = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True, lengths=lengths)
    check_scan(out, state, recurrence(x, dt, A, B, C, D, z, bias, True, None, lengths), F32)
    out, state = ops.causal_conv(x, weight, lengths=lengths)
    want, off, final = conv_reference(x, weight, None, False, None, lengths)
    check(out, want, off, F32)
    assert torch.equal(state, final)


def test_states_beyond_2_31_elements(ops):
    """Slots whose states lie more than 2^31 elements into the pool."""
    c, n = 32768, 64
    pool = torch.zeros(1050, c, n, device="cuda")
    lines = torch.zeros(22000, 3, c, device="cuda", dtype=BF16)
    x, dt, A, B, C, D, z, bias = make(2, 3, c, n, 1, BF16)
    weight = torch.randn(c, 4, device="cuda").to(BF16)
    slots = torch.tensor([1049, 7], dtype=torch.int32, device="cuda")
    want, state = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True)
    out, _ = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True, state=pool, slots=slots)
    assert torch.equal(out, want) and torch.equal(pool[slots.long()], state)
    one = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], pool, slots=slots)
    same = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], state)
    # (steps as they come: some states grow until they are no numbers, in both pools alike)
    assert torch.equal(one.view(torch.int16), same.view(torch.int16)) and torch.equal(pool[slots.long()].view(torch.int32), state.view(torch.int32))
    assert not bool(pool[8].any())
    slots = torch.tensor([21999, 7], dtype=torch.int32, device="cuda")
    want, last = ops.causal_conv(x, weight)
    out, _ = ops.causal_conv(x, weight, state=lines, slots=slots)
    assert torch.equal(out, want) and torch.equal(lines[slots.long()], last)
    one, same = ops.causal_conv_step(x[:, 0], weight, lines, slots=slots), ops.causal_conv_step(x[:, 0], weight, last)
    assert torch.equal(one, same) and torch.equal(lines[slots.long()], last)


def test_long_memories(ops):
    """Decays next to 1 over thousands of tokens: what a decay is off adds up, but stays within 32 bits' measure."""
    b, t, c, n = 1, 4000, 24, 16
    x, dt, A, B, C, D, z, bias = make(b, t, c, n, 1, F32, span=0.0)
    A = A / 16
    out, state = ops.selective_scan(x, dt * 0.2, A, B, C, D=D, z=z, dt_bias=bias, softplus=True)
    want = recurrence(x, dt * 0.2, A, B, C, D, z, bias, True, None, torch.full((b,), t, device="cuda"))
    check(out, want[0], want[1], F32)
    assert bool(((state.double() - want[2]).abs() <= want[3]).all())


@pytest.mark.parametrize("tokens", [1, 40, 700])
def test_slots_that_are_none_out_of_range_or_named_twice(ops, tokens):
    import functs_b200
    b, c, n = 6, 40, 16
    x, dt, A, B, C, D, z, bias = make(b, tokens, c, n, 1, BF16)
    weight = torch.randn(c, 4, device="cuda").to(BF16)
    slots = torch.tensor([2, -1, 4, 2, 0, -7], device="cuda", dtype=torch.int32)
    live, idle = torch.tensor([0, 4], device="cuda"), torch.tensor([1, 2, 3, 5], device="cuda")
    pool, lines = torch.randn(4, c, n, device="cuda"), torch.randn(4, 3, c, device="cuda").to(BF16)
    start, before = pool.clone(), lines.clone()
    status = ops.new_status("cuda")
    out, _ = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True, state=pool, slots=slots, status=status)
    want = recurrence(x[live], dt[live], A, B[live], C[live], D, z[live], bias, True, start[[2, 0]], torch.full((2,), tokens, device="cuda"))
    check_scan(out[live], pool[[2, 0]], want, BF16)
    assert bool((out[idle] == 0).all()) and torch.equal(pool[[1, 3]], start[[1, 3]]) and int(status) == 4 | 8
    status = ops.new_status("cuda")
    out, _ = ops.causal_conv(x, weight, state=lines, slots=slots, status=status)
    want, off, final = conv_reference(x[live], weight, None, False, before[[2, 0]], torch.full((2,), tokens, device="cuda"))
    check(out[live], want, off, BF16)
    assert bool((out[idle] == 0).all()) and torch.equal(lines[[1, 3]], before[[1, 3]]) and torch.equal(lines[[2, 0]], final) and int(status) == 4 | 8
    with pytest.raises(functs_b200.FunctsB200Error, match="out of range; an index was named twice"):
        ops.raise_on_status(status, "causal_conv")
    if tokens == 1:
        status = ops.new_status("cuda")
        out = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], start, slots=slots, status=status)
        assert bool((out[idle] == 0).all()) and int(status) == 4 | 8


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", ["x", "dt", "B", "C", "z"])
def test_scan_of_values_that_are_not_finite(ops, what, dtype):
    """A NaN or an infinity leaves the tokens before it, other sequences and other channels alone."""
    b, t, c, n = 2, 130, 40, 16
    inputs = dict(zip(("x", "dt", "A", "B", "C", "D", "z", "bias"), make(b, t, c, n, 1, dtype)))

    def call():
        return ops.selective_scan(*(inputs[k] for k in ("x", "dt", "A", "B", "C", "D", "z")), dt_bias=inputs["bias"], softplus=True)

    clean, clean_state = call()
    for bad in (math.nan, math.inf, -math.inf):
        kept = inputs[what]
        inputs[what] = kept.clone()
        inputs[what][(0, 70, 0, 3) if what in ("B", "C") else (0, 70, 3)] = bad
        out, state = call()
        inputs[what] = kept
        assert torch.equal(out[:, :70], clean[:, :70]) and torch.equal(out[1], clean[1]) and torch.equal(state[1], clean_state[1])
        if what in ("x", "dt", "z"):
            others = torch.arange(c, device="cuda") != 3
            assert torch.equal(out[..., others], clean[..., others]) and torch.equal(state[:, others], clean_state[:, others])
        if what in ("x", "B") or (what == "dt" and not bad < 0):
            assert not bool(torch.isfinite(state[0, 3]).all())
        if what == "dt" and bad < 0:  # (a step of nothing)
            assert bool(torch.isfinite(state).all())
        if what in ("C", "z") or math.isnan(bad):
            assert what == "z" and bad < 0 or not bool(torch.isfinite(out[0, 70, 3]))
        if what in ("C", "z"):
            assert torch.equal(state, clean_state) and torch.equal(out[:, 71:], clean[:, 71:])


def test_nothing_to_do(ops):
    x, dt, A, B, C, D, z, bias = make(2, 3, 8, 4, 1, BF16)
    weight = torch.randn(8, 4, device="cuda").to(BF16)
    out, state = ops.selective_scan(x[:, :0], dt[:, :0], A, B[:, :0], C[:, :0], z=z[:, :0])
    assert out.shape == (2, 0, 8) and bool((state == 0).all())
    pool = torch.randn(2, 8, 4, device="cuda")
    kept = pool.clone()
    ops.selective_scan(x[:, :0], dt[:, :0], A, B[:, :0], C[:, :0], state=pool)
    assert torch.equal(pool, kept)
    out, state = ops.selective_scan(x[:0], dt[:0], A, B[:0], C[:0])
    assert out.shape == (0, 3, 8) and state.shape == (0, 8, 4)
    out, state = ops.causal_conv(x[:, :0], weight)
    assert out.shape == (2, 0, 8) and bool((state == 0).all())
    lines = torch.randn(2, 3, 8, device="cuda").to(BF16)
    kept = lines.clone()
    ops.causal_conv(x[:, :0], weight, state=lines)
    assert torch.equal(lines, kept)
    out, state = ops.causal_conv(x[:0], weight)
    assert out.shape == (0, 3, 8) and state.shape == (0, 3, 8)
    assert ops.causal_conv_step(x[:0, 0], weight, lines[:0]).shape == (0, 8)
    assert ops.selective_scan_step(x[:0, 0], dt[:0, 0], A, B[:0, 0], C[:0, 0], pool[:0]).shape == (0, 8)


def test_prompts_in_pieces_are_whole_prompts(ops):
    """A prompt in pieces, the last of single tokens, leaves the same states and outputs up to roundings."""
    b, t, c, n = 2, 150, 48, 16
    x, dt, A, B, C, D, z, bias = make(b, t, c, n, 2, F32)
    weight = torch.randn(c, 4, device="cuda")
    kw = dict(D=D, dt_bias=bias, softplus=True)
    whole, state = ops.selective_scan(x, dt, A, B, C, z=z, **kw)
    line, last = ops.causal_conv(x, weight, silu=True)
    pool, lines = torch.zeros(b, c, n, device="cuda"), torch.zeros(b, 3, c, device="cuda")
    at = 0
    for piece in (1, 2, 64, 60, 20):
        s = slice(at, at + piece)
        out, _ = ops.selective_scan(x[:, s], dt[:, s], A, B[:, s], C[:, s], z=z[:, s], state=pool, **kw)
        assert torch.allclose(out, whole[:, s], rtol=1e-4, atol=1e-5)
        out, _ = ops.causal_conv(x[:, s], weight, silu=True, state=lines)
        assert torch.equal(out, line[:, s])
        at += piece
    for i in range(at, t):
        out = ops.selective_scan_step(x[:, i], dt[:, i], A, B[:, i], C[:, i], pool, z=z[:, i], **kw)
        assert torch.allclose(out, whole[:, i], rtol=1e-4, atol=1e-5)
        assert torch.equal(ops.causal_conv_step(x[:, i], weight, lines, silu=True), line[:, i])
    assert torch.allclose(pool, state, rtol=1e-5, atol=1e-5) and torch.equal(lines, last)


def test_out_strides_streams_and_graphs(ops):
    b, t, c, n = 3, 70, 64, 16
    x, dt, A, B, C, D, z, bias = make(b, t, c, n, 1, BF16)
    weight = torch.randn(c, 4, device="cuda").to(BF16)
    kw = dict(D=D, z=z, dt_bias=bias, softplus=True)
    want, state = ops.selective_scan(x, dt, A, B, C, **kw)
    line, last = ops.causal_conv(x, weight, silu=True)
    wide = torch.full((t, b, 2 * c + 8), 7.0, device="cuda", dtype=BF16)
    first, second = wide[..., :c].transpose(0, 1), wide[..., c:2 * c].transpose(0, 1)
    ops.selective_scan(x, dt, A, B, C, out=first, **kw)
    ops.causal_conv(x, weight, silu=True, out=second)
    assert torch.equal(first, want) and torch.equal(second, line) and bool((wide[..., 2 * c:] == 7).all())
    # channels that are not adjacent, a broadcast step, another stream
    apart = x.transpose(1, 2).contiguous().transpose(1, 2)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again, _ = ops.selective_scan(apart, dt, A, B, C, **kw)
        same, _ = ops.causal_conv(apart, weight, silu=True)
    other.synchronize()
    assert torch.equal(again, want) and torch.equal(same, line)
    flat = dt[:, :, :1].expand(-1, -1, c)
    spread, _ = ops.selective_scan(x, flat, A, B[:1].expand(b, -1, -1, -1), C, **kw)
    full, _ = ops.selective_scan(x, flat.contiguous(), A, B[:1].repeat(b, 1, 1, 1), C, **kw)
    assert torch.equal(spread, full)
    # single tokens, captured: each replay goes on from where the last one ended
    pool, lines = torch.zeros(b, c, n, device="cuda"), torch.zeros(b, 3, c, device="cuda", dtype=BF16)
    xs, dts, bs, cs, zs = x[:, 0].clone(), dt[:, 0].clone(), B[:, 0].clone(), C[:, 0].clone(), z[:, 0].clone()
    got, here = torch.empty(b, c, device="cuda", dtype=BF16), torch.empty(b, c, device="cuda", dtype=BF16)

    def step():
        ops.selective_scan_step(xs, dts, A, bs, cs, pool, D=D, z=zs, dt_bias=bias, softplus=True, out=got)
        ops.causal_conv_step(xs, weight, lines, silu=True, out=here)

    step()
    pool.zero_(), lines.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(t):
        for to, at in ((xs, x), (dts, dt), (bs, B), (cs, C), (zs, z)):
            to.copy_(at[:, i])
        graph.replay()
        assert torch.equal(here, line[:, i])
    assert torch.allclose(pool, state, rtol=1e-5, atol=1e-6) and torch.equal(lines, last)
    # a captured prompt
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, fresh = ops.selective_scan(x, dt, A, B, C, **kw)
    out.zero_(), fresh.zero_()
    graph.replay()
    assert torch.equal(out, want) and torch.equal(fresh, state)


def test_refusals(ops):
    x, dt, A, B, C, D, z, bias = make(2, 5, 16, 8, 2, BF16)
    weight = torch.randn(16, 4, device="cuda").to(BF16)
    for bad, match in (((x[0], weight), "must be"), ((x, weight[:8]), "weight"), ((x, torch.cat([weight, weight, weight], 1)), "width"),
                       ((x, weight[:, :1]), "width")):
        with pytest.raises(ValueError, match=match):
            ops.causal_conv(*bad)
    with pytest.raises(TypeError, match="weight"):
        ops.causal_conv(x, weight.float())
    with pytest.raises(TypeError, match="float32"):
        ops.causal_conv(x.double(), weight.double())
    with pytest.raises(ValueError, match="give one"):
        ops.causal_conv(x, weight, slots=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="states"):
        ops.causal_conv(x, weight, state=torch.zeros(3, 3, 16, device="cuda", dtype=BF16))
    with pytest.raises(TypeError, match="state"):
        ops.causal_conv(x, weight, state=torch.zeros(2, 3, 16, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        ops.causal_conv(x, weight, weight)
    good = dict(x=x, dt=dt, A=A, B=B, C=C)
    for name, value, match in (("dt", dt[:, :3], "dt"), ("A", A[:8], "A must"), ("A", torch.zeros(16, 65, device="cuda"), "A must"), ("B", B[:, :3], "B"),
                               ("C", C[:, :, :1], "C"), ("B", torch.zeros(2, 5, 3, 8, device="cuda", dtype=BF16), "C|multiple"), ("x", x[0], "must be"),
                               ("D", D[:3], "D"), ("dt_bias", bias[:3], "dt_bias"), ("z", z[:1], "z"), ("lengths", torch.zeros(3, dtype=torch.int32, device="cuda"), "lengths"),
                               ("slots", torch.zeros(2, dtype=torch.int32, device="cuda"), "give one"), ("state", torch.zeros(2, 16, 4, device="cuda"), "state"),
                               ("state", torch.zeros(2, 8, 16, device="cuda").transpose(1, 2), "contiguous"), ("out", x, "share memory"),
                               ("out", torch.zeros(1, 5, 16, device="cuda", dtype=BF16).expand(2, -1, -1), "overlap itself"), ("out", x[:1], "out")):
        with pytest.raises(ValueError, match=match):
            ops.selective_scan(**{**good, name: value})
    for name, value in (("dt", dt.float()), ("A", A.to(BF16)), ("B", B.float()), ("state", torch.zeros(2, 16, 8, device="cuda", dtype=BF16)),
                        ("lengths", torch.zeros(2, dtype=torch.int64, device="cuda")), ("D", D.double())):
        with pytest.raises(TypeError, match=name):
            ops.selective_scan(**{**good, name: value})
    pool = torch.zeros(4, 16, 8, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        ops.selective_scan(**{**good, "A": pool[0]}, state=pool[:2])
    for name in ("x", "A"):
        leaf = good[name].clone().requires_grad_()
        with pytest.raises(NotImplementedError, match="gradient"):
            ops.selective_scan(**{**good, name: leaf})
        with torch.no_grad():
            ops.selective_scan(**{**good, name: leaf})
    with pytest.raises(NotImplementedError, match="gradient"):
        ops.causal_conv(x, weight.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="transform"):
        torch.func.vmap(lambda y: ops.causal_conv(y, weight)[0])(x[None])


def test_autograd_is_told_of_what_is_written_over(ops):
    x, dt, A, B, C, D, z, bias = make(2, 5, 16, 8, 1, F32)
    for call in (lambda s: ops.selective_scan(x, dt, A, B, C, state=s), lambda s: ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], s)):
        leaf, pool = torch.ones(2, 16, 8, device="cuda", requires_grad=True), torch.ones(2, 16, 8, device="cuda")
        y = (leaf * pool).sum()
        call(pool)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_deterministic(ops):
    x, dt, A, B, C, D, z, bias = make(3, 900, 200, 16, 1, BF16)
    first = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True)
    for _ in range(3):
        again = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---- rates that are not finite, states that grow ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,c,n", [(1, 40, 16), (5, 33, 5), (16, 40, 16), (33, 64, 8), (130, 36, 3), (1203, 48, 16)])
def test_states_that_forget_at_once(ops, t, c, n, dtype):
    """A rate of -inf, or one whose product with log2 e is: every token but the last is forgotten, at whatever token a sequence ends."""
    b = 4
    x, dt, A, B, C, D, z, bias = make(b, t, c, n, 1, dtype)
    A[::2, 0], A[1::3, n - 1] = -math.inf, -3e38
    lengths = torch.tensor([t, t // 2, 1, max(t - 3, 0)], dtype=torch.int32, device="cuda")
    start = torch.randn(b, c, n, device="cuda")
    pool = start.clone()
    out, _ = ops.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, softplus=True, state=pool, lengths=lengths)
    plain = A.clamp(min=-1e15)  # (steps are some 1e-5 at least: nothing is left either)
    check_scan(out, pool, recurrence(x, dt, plain, B, C, D, z, bias, True, start, lengths), dtype)
    pool = start.clone()
    out = ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], pool, D=D, z=z[:, 0], dt_bias=bias, softplus=True)
    want = recurrence(x[:, :1], dt[:, :1], plain, B[:, :1], C[:, :1], D, z[:, :1], bias, True, start, torch.ones(b, device="cuda"))
    check_scan(out[:, None], pool, want, dtype)


@pytest.mark.parametrize("t", [3, 17, 700])
def test_rates_without_bound_and_steps_of_either_sign(ops, t):
    """A step of 0 leaves every state as it is, and a step below 0 with a rate of +inf nothing of it; a rate that is no number reaches its own channel alone."""
    x, _, A, B, C, D, _, _ = make(2, t, 24, 16, 1, F32)
    start = torch.randn(2, 24, 16, device="cuda")
    A[:, 2], A[:, 5] = -math.inf, math.inf
    none = torch.zeros(2, t, 24, device="cuda")
    out, state = ops.selective_scan(x, none, A, B, C, D=D, state=start.clone())
    assert torch.equal(state, start) and bool(torch.isfinite(out).all())
    pool = start.clone()
    ops.selective_scan_step(x[:, 0], none[:, 0], A, B[:, 0], C[:, 0], pool)
    assert torch.equal(pool, start)
    A[:, 2] = -1.0
    back = none - 0.001
    out, state = ops.selective_scan(x, back, A, B, C, D=D, state=start.clone())
    want = recurrence(x, back, A.clamp(max=1e15), B, C, D, None, None, False, start, torch.full((2,), t, device="cuda"))
    check(out, want[0], want[1], F32)
    assert bool(((state.double() - want[2]).abs() <= want[3]).all())
    A[3, 4] = math.nan
    out, state = ops.selective_scan(x, back, A, B, C, D=D, state=start.clone())
    bad = torch.zeros(24, 16, dtype=torch.bool, device="cuda")
    bad[3, 4] = True
    assert torch.equal(torch.isnan(state), bad.expand(2, -1, -1)) and torch.equal(torch.isnan(out), bad.any(1).expand(2, t, -1))


def grows(ops, x, dt, A, B, C, D, state):
    want = recurrence(x, dt, A, B, C, D, None, None, False, state, torch.full((x.size(0),), x.size(1), device="cuda"))
    out, state = ops.selective_scan(x, dt, A, B, C, D=D, state=state)
    check(out, want[0], want[1], F32)
    assert bool(((state.double() - want[2]).abs() <= want[3]).all())


def test_states_of_0_while_others_would_grow(ops):
    """Rates above 0 whose growth over a part of a prompt passes 32 bits: nothing but zeros until late."""
    t = 4096
    x, dt, A, B, C, D, _, _ = make(1, t, 24, 16, 1, F32)
    x[:, :t - 50] = 0.0
    grows(ops, x, torch.ones_like(dt), torch.ones_like(A), B, C, D, None)


@pytest.mark.parametrize("first", [200, 290, 380, 470, 560])
def test_states_that_grow_over_a_part_of_a_prompt(ops, first):
    """Growth by e^144 within 72 tokens, of a state that starts small and stays finite."""
    x, dt, A, B, C, D, _, _ = make(1, 1500, 24, 16, 1, F32)
    dt = torch.zeros_like(dt)
    dt[:, first:first + 72] = 2.0
    grows(ops, x * 1e-28, dt, torch.ones_like(A), B, C, D, torch.full((1, 24, 16), 1e-28, device="cuda"))
