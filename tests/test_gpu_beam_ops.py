"""Beam search's selection and the reordering of states, against plain programs in 64 bits; and a search with the recurrent operators together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(cuda_device):
    import functs_b200
    return functs_b200.ops


# ---- selection --------------------------------------------------------------------------------------------------------


def select_reference(logits, scores, top, ended=None, end_token=None):
    """All candidates in 64 bits, sorted: of equal ones the lowest (parent, token) first, NaN before all."""
    v = logits.size(2)
    # (rows of whole 64 elements, so that every row is summed in the same order: rows that are the same have the same sum, to the last bit)
    x = torch.nn.functional.pad(logits.double(), (0, -v % 64), value=-math.inf)
    most = x.amax(dim=2, keepdim=True)
    empty = most == -math.inf
    apart = x - torch.where(empty, 0.0, most)  # (the difference first: beside a largest element of -3.4e38 a logarithm is lost in 64 bits too)
    lp = torch.where(empty, x, apart - torch.log(torch.exp(apart).sum(dim=2, keepdim=True)))[..., :v]
    s = scores.double()[..., None]
    total = torch.where(s == -math.inf, s, lp + s)
    if ended is not None:
        held = torch.full((v,), -math.inf, dtype=torch.float64, device=x.device)
        held[end_token] = 0.0
        total = torch.where(ended[..., None], torch.where(held == 0, s, held), total)
    nan = torch.isnan(s) | (s == math.inf) | ((s > -math.inf) & (~(most < math.inf)) & (~ended[..., None] if ended is not None else True))
    total = torch.where(nan, math.nan, total).flatten(1)
    score, place = torch.sort(torch.where(torch.isnan(total), math.inf, total), dim=1, descending=True, stable=True)
    score = torch.where(score == math.inf, math.nan, score)
    return score[:, :top], place[:, :top] // v, place[:, :top] % v


def check_select(got, want, vocab):
    """Parents and tokens are equal; a score is rounded once, and its row's logarithm is off by 2^-20 and a rounding for every sixteen of
    512 threads' elements at most."""
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    s, w = got[0].double(), want[0]
    assert torch.equal(torch.isnan(s), torch.isnan(w))
    fine = torch.isfinite(w)
    assert torch.equal(torch.isfinite(s), fine) and torch.equal(s[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)])
    off = 2.0 ** -20 + (vocab / 128 / 16 + 16) * 2.0 ** -24
    assert bool(((s - w).abs()[fine] <= 2.0 ** -24 * w.abs()[fine] + off).all())


SELECT = [
    # groups, beams, vocab, top
    (1, 1, 1, 1), (1, 1, 50, 50), (2, 3, 7, 21), (3, 2, 10, 8), (1, 64, 3, 64), (5, 4, 100, 9), (2, 12, 127, 24), (3, 5, 1000, 10), (1, 4, 1025, 64),
    (2, 8, 5003, 16), (64, 4, 4096, 8), (1, 5, 32000, 10), (2, 64, 1500, 64), (3, 3, 50001, 6), (200, 4, 9001, 4),
]


def inputs(g, k, v, dtype, seed=1, start=False, masked=False, ended=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(g, k, v, generator=gen, device="cuda") * 3
    if masked:
        logits.masked_fill_(torch.rand(g, k, v, generator=gen, device="cuda") > 0.1, -math.inf)
    scores = torch.rand(g, k, generator=gen, device="cuda") * -5
    if start:
        scores[:] = -math.inf
        scores[:, k // 2] = 0.0
    flags = torch.rand(g, k, generator=gen, device="cuda") < 0.2 if ended else None
    return logits.to(dtype), scores, flags


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SELECT, ids=str)
def test_select(ops, shape, dtype):
    g, k, v, top = shape
    for seed, start, masked, ended in ((1, False, False, False), (2, False, False, True), (3, True, False, False), (4, False, True, True)):
        logits, scores, flags = inputs(g, k, v, dtype, seed, start, masked, ended)
        end = v // 2 if ended else None
        got = ops.beam_select(logits, scores, top=top, ended=flags, end_token=end)
        assert got[0].dtype == F32 and got[1].dtype == got[2].dtype == torch.int64 and all(x.shape == (g, top) for x in got)
        check_select(got, select_reference(logits, scores, top, flags, end), v)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 3, 140003, 24), (2, 1, 70001, 9), (1, 8, 66000, 16), (1, 33, 40000, 40), (4, 4, 131072, 64)], ids=str)
def test_few_long_rows(ops, shape, dtype):
    """Rows in parts, whose lists meet."""
    g, k, v, top = shape
    for masked in (False, True):
        logits, scores, flags = inputs(g, k, v, dtype, 12, masked=masked)
        check_select(ops.beam_select(logits, scores, top=top, ended=flags, end_token=v - 1), select_reference(logits, scores, top, flags, v - 1), v)
    logits[:, 0] = -math.inf
    logits[:, 0, v - 5:] = 1.5  # (all that is left lies in the last part)
    logits[:, k // 2, 70:] = -math.inf
    flags[:] = False
    check_select(ops.beam_select(logits, scores, top=top), select_reference(logits, scores, top), v)
    flat = torch.zeros(g, k, v, device="cuda", dtype=dtype)
    check_select(ops.beam_select(flat, scores, top=top), select_reference(flat, scores, top), v)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("g,k,v", [(24, 8, 6007), (1, 8, 140003)])
def test_scores_next_to_one_another(ops, g, k, v, dtype):
    """Beams whose best continuations lie within some 2^-22 of one another: their order is that of 64 bits."""
    logits, _, _ = inputs(g, k, v, dtype, 5)
    lse = torch.logsumexp(logits.double(), dim=2)
    scores = (-20.0 - (logits.double().amax(dim=2) - lse)).float()  # (rounded: what is left of the differences)
    got = ops.beam_select(logits, scores, top=2 * k)
    want = select_reference(logits, scores, 2 * k)
    gaps = (want[0][:, :k - 1] - want[0][:, 1:k])
    assert bool((gaps < 4e-6).all()) and bool((gaps < 5e-7).any())  # (near indeed)
    check_select(got, want, v)


def test_equal_candidates(ops):
    """Beams that are the same, rows of few different values: the lowest beam and the lowest token come first."""
    logits, scores, _ = inputs(3, 6, 3001, BF16, 6)
    logits[:] = logits[:, :1]
    scores[:] = -1.0
    check_select(ops.beam_select(logits, scores, top=40), select_reference(logits, scores, 40), 3001)
    flat = torch.randint(0, 2, (2, 5, 4001), device="cuda").to(F16)
    check_select(ops.beam_select(flat, torch.zeros(2, 5, device="cuda"), top=64), select_reference(flat, torch.zeros(2, 5, device="cuda"), 64), 4001)
    same = torch.zeros(2, 4, 2000, device="cuda")
    got = ops.beam_select(same, torch.zeros(2, 4, device="cuda"), top=9)
    assert torch.equal(got[1], torch.zeros_like(got[1])) and torch.equal(got[2], torch.arange(9, device="cuda").expand(2, 9))


def test_rows_that_leave_nothing_and_values_that_are_not_finite(ops):
    g, k, v = 7, 4, 1300
    logits, scores, _ = inputs(g, k, v, F32, 7)
    ended = torch.zeros(g, k, dtype=torch.bool, device="cuda")
    logits[0, 1] = -math.inf                       # a mask that leaves nothing
    logits[1, :, :] = -math.inf                    # in every beam
    logits[2, 0, 5], logits[2, 3, 9] = math.nan, math.inf
    scores[3, 2] = math.nan
    scores[4, 0], scores[4, 1] = -math.inf, math.inf
    logits[4, 0, 3] = math.nan                     # (of a beam that is none: not looked at)
    ended[5] = True                                # nothing but beams that have ended
    logits[5, 0, 0] = math.nan
    logits[6, 0] = torch.finfo(F32).min            # a mask of the type's lowest value that leaves nothing
    logits[6, 1, 7:] = torch.finfo(F32).min
    for top in (1, 3, 20):
        check_select(ops.beam_select(logits, scores, top=top, ended=ended, end_token=11), select_reference(logits, scores, top, ended, 11), v)


def test_strides_of_logits(ops):
    """Rows any distance apart, off every vector's boundary, and logits whose tokens are not adjacent."""
    g, k, v = 3, 4, 2049
    wide, scores, _ = inputs(g, k, v + 14, BF16, 8)
    for cut in (slice(3, 3 + v), slice(8, 8 + v)):
        logits = wide[..., cut]
        check_select(ops.beam_select(logits, scores), select_reference(logits, scores, k), v)
    turned = wide[..., :v].transpose(0, 1).contiguous().transpose(0, 1)
    check_select(ops.beam_select(turned, scores), select_reference(turned, scores, k), v)
    apart = wide[..., :v].transpose(1, 2).contiguous().transpose(1, 2)
    check_select(ops.beam_select(apart, scores), select_reference(apart, scores, k), v)
    one = wide[:, :1, :v].expand(-1, k, -1)
    check_select(ops.beam_select(one, scores), select_reference(one, scores, k), v)


# ---- reordering -------------------------------------------------------------------------------------------------------


def reorder_reference(slots, parents, num_slots):
    """-> new slots, moves (to, from), faulty groups' bits; beam by beam."""
    new, moves, bits, seen = [], [], 0, set()
    for s, p in zip(slots.tolist(), parents.tolist()):
        k = len(s)
        fault = 0
        if s[0] >= 0:
            if any(not 0 <= x < num_slots for x in s) or any(not 0 <= x < k for x in p):
                fault |= 4
            for j in range(k):
                if s[j] in seen or s[j] in s[:j]:
                    fault |= 8
        seen |= set(s)
        bits |= fault
        if s[0] < 0 or fault:
            new.append(s)
            continue
        free = [s[i] for i in range(k) if i not in p]
        row = []
        for j in range(k):
            if p[j] in p[:j]:
                row.append(free.pop(0))
                moves.append((row[-1], s[p[j]]))
            else:
                row.append(s[p[j]])
        new.append(row)
    return torch.tensor(new, dtype=torch.int32), moves, bits


def check_reorder(ops, pools, slots, parents):
    num = pools[0].size(0) if pools else 2 ** 31 - 1
    new, moves, bits = reorder_reference(slots, parents, num)
    want = [p.clone() for p in pools]
    for to, at in moves:
        for w, p in zip(want, pools):
            w[to] = p[at]
    status = ops.new_status("cuda")
    got = ops.beam_reorder(pools, parents.cuda(), slots.cuda(), status=status)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), new)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)
    assert int(status) == bits


@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 2), (3, 4), (40, 5), (2, 64), (7, 33)])
def test_reorder(ops, groups, beams):
    gen = torch.Generator().manual_seed(groups * 100 + beams)
    n = groups * beams + 3
    for parents in (torch.randint(0, beams, (groups, beams), generator=gen), torch.zeros(groups, beams, dtype=torch.int64),
                    torch.arange(beams).expand(groups, beams), torch.arange(beams).flip(0).expand(groups, beams), torch.full((groups, beams), beams - 1)):
        slots = torch.randperm(n, generator=gen)[: groups * beams].to(torch.int32).view(groups, beams)
        pools = [torch.randn(n, 5, 7, device="cuda"), torch.randn(n, 33, device="cuda").to(BF16), torch.randint(0, 100, (n, 3), device="cuda").to(torch.uint8),
                 torch.randn(n, 8, 16, 40, device="cuda"), torch.randint(0, 1 << 40, (n,), device="cuda"), torch.randn(n, 0, device="cuda"),
                 torch.randn(n, 2, 8192, device="cuda").to(F16)]
        check_reorder(ops, pools, slots, parents.contiguous())


def test_reorder_of_many_pools_and_of_none(ops):
    slots, parents = torch.tensor([[3, 0, 5], [1, 2, 4]], dtype=torch.int32), torch.tensor([[2, 2, 1], [0, 0, 0]])
    check_reorder(ops, [torch.randn(6, 3 + i, device="cuda") for i in range(71)], slots, parents)
    check_reorder(ops, [], slots, parents)
    check_reorder(ops, [torch.randn(6, 0, device="cuda")], slots, parents)
    assert ops.beam_reorder([torch.randn(6, 3, device="cuda")], parents[:0].cuda(), slots[:0].cuda()).shape == (0, 3)


def test_reorder_of_pools_side_by_side_and_off_boundaries(ops):
    """Pools that are pieces of one buffer, on any boundary of their type."""
    whole = torch.randn(4 * 1000 + 64, device="cuda").to(BF16)
    slots, parents = torch.tensor([[3, 0, 1, 2]], dtype=torch.int32), torch.tensor([[1, 1, 3, 1]])
    kept = whole.clone()
    pools = [whole[1:1 + 4 * 100].view(4, 100), whole[401 + 7:401 + 7 + 4 * 31].view(4, 31), whole[1000:1000 + 4 * 64].view(4, 8, 8)]
    check_reorder(ops, pools, slots, parents)
    outside = torch.ones_like(whole, dtype=torch.bool)
    outside[1:401] = outside[408:532] = outside[1000:1256] = False
    assert torch.equal(whole[outside], kept[outside])


def test_reorder_of_groups_that_are_none_or_wrong(ops):
    import functs_b200
    pool = [torch.randn(20, 9, device="cuda")]
    fine = torch.tensor([[1, 0, 0], [0, 0, 2], [2, 2, 2], [0, 1, 1], [1, 1, 1], [0, 0, 0]])
    slots = torch.tensor([[0, 1, 2], [-1, 3, 4], [5, 6, 7], [8, 9, 10], [11, 12, 13], [14, 15, 16]], dtype=torch.int32)
    check_reorder(ops, pool, slots, fine)
    for row, col, value in ((2, 1, 20), (2, 2, -3), (3, 0, 1), (3, 2, 8), (5, 1, 4)):
        bad = slots.clone()
        bad[row, col] = value
        check_reorder(ops, pool, bad, fine)
    for value in (3, -1, 1 << 40):
        parents = fine.clone()
        parents[4, 2] = value
        check_reorder(ops, pool, slots, parents)
    status = ops.new_status("cuda")
    ops.beam_reorder(pool, parents.cuda(), slots.cuda(), status=status)
    with pytest.raises(functs_b200.FunctsB200Error, match="out of range"):
        ops.raise_on_status(status, "beam_reorder")


def test_rows_beyond_2_31_bytes(ops):
    """Offsets that pass 32 bits."""
    pool = torch.zeros(5, 700_000_000, dtype=torch.uint8, device="cuda")
    for i in range(5):
        pool[i, -1000:] = i + 1
        pool[i, :3] = 10 * i
    got = ops.beam_reorder([pool], torch.tensor([[1, 1, 1]], device="cuda"), torch.tensor([[0, 4, 3]], dtype=torch.int32, device="cuda"))
    assert got.tolist() == [[4, 0, 3]]
    assert bool((pool[[0, 3, 4], -1000:] == 5).all()) and bool((pool[[0, 3, 4], :3] == 40).all()) and bool((pool[2, -1000:] == 3).all())


# ---- refusals, streams, graphs ------------------------------------------------------------------------------------------


def test_refusals(ops):
    logits, scores, _ = inputs(2, 3, 100, BF16)
    ended = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for kw, match in ((dict(logits=logits[0]), "must be"), (dict(scores=scores[:1]), "scores"), (dict(top=0), "top"), (dict(top=65), "top"),
                      (dict(ended=ended), "go together"), (dict(end_token=3), "go together"), (dict(ended=ended, end_token=100), "end_token"),
                      (dict(ended=ended[:1], end_token=1), "ended"), (dict(logits=logits[..., :1], top=4), "top"),
                      (dict(logits=logits[:, :1].expand(-1, 65, -1), scores=scores[:, :1].expand(-1, 65)), "beams")):
        with pytest.raises(ValueError, match=match):
            ops.beam_select(**{**dict(logits=logits, scores=scores), **kw})
    for kw in (dict(logits=logits.double()), dict(scores=scores.double()), dict(ended=ended.to(torch.uint8), end_token=1)):
        with pytest.raises(TypeError):
            ops.beam_select(**{**dict(logits=logits, scores=scores), **kw})
    with pytest.raises(NotImplementedError, match="gradient"):
        ops.beam_select(logits, scores.requires_grad_())
    slots, parents = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([[0, 0]], device="cuda")
    pool = torch.zeros(4, 6, device="cuda")
    for states, match in (([pool.t()], "contiguous"), ([pool, pool], "share memory"), ([pool, pool[2:]], "as many|share"), ([torch.zeros(3, 2, device="cuda"), pool], "as many"),
                          ([torch.zeros((), device="cuda")], "pool"), ([slots.view(2, 1)], "share memory")):
        with pytest.raises(ValueError, match=match):
            ops.beam_reorder(states, parents, slots)
    with pytest.raises(ValueError, match="parents"):
        ops.beam_reorder([pool], parents[:, :1], slots)
    with pytest.raises(TypeError, match="parents"):
        ops.beam_reorder([pool], parents.int(), slots)
    with pytest.raises(TypeError, match="slots"):
        ops.beam_reorder([pool], parents, slots.long())
    with pytest.raises(NotImplementedError, match="gradient"):
        ops.beam_reorder([pool.clone().requires_grad_()], parents, slots)


def test_streams_and_graphs(ops):
    logits, scores, flags = inputs(4, 5, 3001, F16, 9)
    want = ops.beam_select(logits, scores, top=10, ended=flags, end_token=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(logits, scores, top=10, ended=flags, end_token=1)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    pool, slots = torch.randn(25, 100, device="cuda"), torch.randperm(25, device="cuda")[:20].to(torch.int32).view(4, 5)
    graph = torch.cuda.CUDAGraph()
    fixed, copy = logits.clone(), pool.clone()
    with torch.cuda.graph(graph):
        s, p, t = ops.beam_select(fixed, scores, ended=flags, end_token=1)
        new = ops.beam_reorder([copy], p, slots)
    for seed in (10, 11):
        other = inputs(4, 5, 3001, F16, seed)[0]
        fixed.copy_(other), copy.copy_(pool)
        graph.replay()
        w = ops.beam_select(other, scores, ended=flags, end_token=1)
        assert all(torch.equal(x, y) for x, y in zip((s, p, t), w))
        plain = pool.clone()
        assert torch.equal(ops.beam_reorder([plain], w[1], slots), new) and torch.equal(plain, copy)


# ---- together -----------------------------------------------------------------------------------------------------------


class Model:
    """One layer: short convolution, selective scan, attention with a decaying state; logits of a small vocabulary."""

    def __init__(self, ops, dim=32, states=8, heads=2, vocab=200):
        gen = torch.Generator(device="cuda").manual_seed(3)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.ops, self.dim, self.states, self.heads = ops, dim, states, heads
        self.embed, self.weight, self.out = r(vocab, dim), r(dim, 4) * 0.5, r(dim, vocab) * 0.6
        self.to_scan, self.to_heads = r(dim, dim + 2 * states) * 0.2, r(dim, 3 * dim) * 0.3
        self.A, self.D, self.bias = -torch.rand(dim, states, generator=gen, device="cuda") * 4 - 0.2, r(dim), r(dim) - 2
        self.decay = -torch.rand(heads, generator=gen, device="cuda")

    def pools(self, n, dtype=F32):
        z = lambda *s: torch.zeros(n, *s, dtype=dtype, device="cuda")  # noqa: E731
        return [z(3, self.dim), z(self.dim, self.states), z(self.heads, self.dim // self.heads, self.dim // self.heads)]

    def prompt(self, tokens, lengths, pools, slots):
        x, _ = self.ops.causal_conv(self.embed[tokens], self.weight, silu=True, state=pools[0], slots=slots, lengths=lengths)
        dt, b, c = (x @ self.to_scan).split([self.dim, self.states, self.states], dim=-1)
        y, _ = self.ops.selective_scan(x, dt, self.A, b[:, :, None], c[:, :, None], D=self.D, dt_bias=self.bias, softplus=True, state=pools[1], slots=slots,
                                       lengths=lengths)
        q, k, v = (y @ self.to_heads).unflatten(-1, (3 * self.heads, -1)).chunk(3, dim=2)
        o, _ = self.ops.linear_attention(q, k, v, self.decay, state=pools[2], slots=slots, lengths=lengths)
        return o.flatten(2) @ self.out

    def step(self, tokens, pools, slots):
        x = self.ops.causal_conv_step(self.embed[tokens], self.weight, pools[0], silu=True, slots=slots)
        dt, b, c = (x @ self.to_scan).split([self.dim, self.states, self.states], dim=-1)
        y = self.ops.selective_scan_step(x, dt, self.A, b[:, None], c[:, None], pools[1], D=self.D, dt_bias=self.bias, softplus=True, slots=slots)
        q, k, v = (y @ self.to_heads).unflatten(-1, (3 * self.heads, -1)).chunk(3, dim=1)
        return self.ops.linear_attention_step(q, k, v, self.decay, pools[2], slots=slots).flatten(1) @ self.out

    def exact(self, token, state):
        """One token of one sequence in 64 bits; state: the last inputs, h, S."""
        line, h, s = state
        line = torch.cat([line, self.embed[token].double()[None]])
        x = (line * self.weight.double().t()).sum(0)
        x = x * torch.sigmoid(x)
        dt, b, c = (x @ self.to_scan.double()).split([self.dim, self.states, self.states])
        d = torch.logaddexp(dt + self.bias.double(), torch.zeros_like(dt))
        h = torch.exp(d[:, None] * self.A.double()) * h + (d * x)[:, None] * b
        y = h @ c + self.D.double() * x
        q, k, v = (y @ self.to_heads.double()).unflatten(0, (3 * self.heads, -1)).chunk(3)
        s = torch.exp(self.decay.double())[:, None, None] * s + k[:, :, None] * v[:, None, :]
        return torch.einsum("hk,hkv->hv", q, s).flatten() @ self.out.double(), (line[1:], h, s)


def test_a_beam_search(ops):
    """Prompts of uneven lengths, then some tokens of beam search: states in one pool per operator, reordered as beams go on.  In 64 bits the same search
    keeps every beam's states beside it."""
    torch.backends.cuda.matmul.allow_tf32 = False
    model, groups, beams, end = Model(ops), 3, 4, 7
    prompts = torch.randint(0, 200, (groups, 9), generator=torch.Generator().manual_seed(4)).cuda()
    lengths = torch.tensor([9, 4, 1], dtype=torch.int32, device="cuda")
    pools = model.pools(groups * beams + 2)
    slots = torch.randperm(groups * beams + 2, generator=torch.Generator().manual_seed(5))[: groups * beams].to(torch.int32).cuda().view(groups, beams)
    logits = model.prompt(prompts, lengths, pools, slots[:, 0].contiguous())
    logits = logits[torch.arange(groups), lengths.long() - 1][:, None].expand(-1, beams, -1)
    scores = torch.full((groups, beams), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    ended = torch.zeros(groups, beams, dtype=torch.bool, device="cuda")
    # the same in 64 bits: per group a list of (score, ended, state, logits)
    plain = []
    for g in range(groups):
        state = tuple(p[0].double() for p in model.pools(1))
        for t in range(int(lengths[g])):
            at, state = model.exact(prompts[g, t], state)
        plain.append([(0.0 if k == 0 else -math.inf, False, state, at) for k in range(beams)])
    for step in range(6):
        scores, parents, tokens = ops.beam_select(logits, scores, ended=ended, end_token=end)
        ended = ended.gather(1, parents) | (tokens == end)
        slots = ops.beam_reorder(pools, parents, slots)
        logits = model.step(tokens.flatten(), pools, slots.flatten()).unflatten(0, (groups, beams))
        for g in range(groups):
            want = select_reference(torch.stack([b[3] for b in plain[g]])[None], torch.tensor([[b[0] for b in plain[g]]], dtype=torch.float64, device="cuda"), beams + 1,
                                    torch.tensor([[b[1] for b in plain[g]]], device="cuda"), end)
            # no two so near that 32 bits of the layers could turn them: four layers, each sums of 32 products and four more steps, 36 roundings of 2^-24
            # at most, are 8.6e-6 of a logit's terms, which are 10 in all at most
            assert float((want[0][0, :-1] - want[0][0, 1:]).min()) > 2 * 8.6e-5
            assert torch.equal(parents[g], want[1][0, :beams]) and torch.equal(tokens[g], want[2][0, :beams])
            assert torch.allclose(scores[g].double(), want[0][0, :beams], rtol=1e-4, atol=1e-4)
            new = []
            for k in range(beams):
                parent = plain[g][int(want[1][0, k])]
                at, state = model.exact(want[2][0, k], parent[2])
                new.append((float(want[0][0, k]), parent[1] or int(want[2][0, k]) == end, state, at))
                assert torch.allclose(logits[g, k].double(), at, rtol=1e-3, atol=1e-3 * float(at.abs().max()))
            plain[g] = new


# ---- logits and scores far from 0 -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("most", [2.0 ** 31, 1.2e10, -1.2e10, 1e11, 1e30, -1e30, "max", "min"])
def test_beams_that_are_alike_far_from_0(ops, most, dtype):
    """Two beams of the same score and row, whose largest logits (five of them) lie far from 0, beside lower ones and -inf; a third that is less likely than
    they are by less than log(vocabulary)."""
    v = 1300
    most = torch.tensor({"max": torch.finfo(dtype).max, "min": torch.finfo(dtype).min}.get(most, most), device="cuda").to(dtype)
    logits = torch.full((3, 4, v), -math.inf, device="cuda", dtype=dtype)
    logits[:, 1::2] = torch.randn(3, 2, v, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    logits[:, 1::2, 77] = 40.0
    logits[1, ::2] = most - most.abs() * 2.0 ** -6  # (lower by far, or, where that is none, -inf again)
    logits[2, ::2, 9::2] = most - most.abs()
    logits[:, ::2, 100:600:100] = most
    scores = torch.tensor([[-1.0, -2.0, -1.0, -5.0]], device="cuda").expand(3, -1)
    want = select_reference(logits, scores, 12)
    got = ops.beam_select(logits, scores, top=12)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    # rows far from 0 have sums of at most 11 elements a thread, each rounded, joined in 32 more
    fine = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0]), fine)
    assert bool(((got[0].double() - want[0]).abs()[fine] <= 2.0 ** -24 * want[0].abs()[fine] + (11 + 32) * 2.0 ** -24).all())


def by_logit(logits, scores, top):
    """Of candidates with equal scores in 64 bits: the lowest beam first, and of one beam the largest logit, then the lowest token."""
    total = torch.log_softmax(logits.double(), dim=2) + scores.double()[..., None]
    tokens = torch.sort(logits.double(), dim=2, descending=True, stable=True)[1]
    score, place = torch.sort(total.gather(2, tokens).flatten(1), dim=1, descending=True, stable=True)
    v = logits.size(2)
    return score[:, :top], place[:, :top] // v, tokens.flatten(1).gather(1, place[:, :top])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 140003, 8), (1, 4, 140003, 8), (2, 8, 70001, 6), (3, 5, 3001, 40), (1, 64, 300, 64)], ids=str)
def test_beams_whose_score_leaves_no_room_for_their_logits(ops, shape, dtype):
    """A beam's score so far from 0 that logits which differ make the same score in 64 bits: the order of a beam is that of its logits, whether its row is one
    part or several."""
    g, k, v, top = shape
    logits, _, _ = inputs(g, k, v, dtype, 21)
    for low in (torch.finfo(F32).min, -1e30):
        scores = torch.full((g, k), low, device="cuda")
        got, want = ops.beam_select(logits, scores, top=top), by_logit(logits, scores, top)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]) and torch.equal(got[0], want[0].float())
        if k > 1:
            scores[:, 1] = -2.0  # (one that goes on: its own come first)
            got, want = ops.beam_select(logits, scores, top=top), by_logit(logits, scores, top)
            assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


def test_scores_on_either_side_of_a_rounding_in_64_bits(ops):
    """Beams at -2^40, where a score in 64 bits is a multiple of 2^-12: one beam's lies next to the border of two such numbers, nearer than a pass over its
    logits knows it, the other's is the upper of them.  Equal they are (the lower beam first), or one is below."""
    n = torch.arange(300, 300 + 512 * 4, 4, dtype=torch.float64)
    x = torch.log(torch.expm1((n + 0.5) / 4096)).float()          # -log(1 + exp(x)) = -(n + 1/2) / 4096
    x = torch.cat([x, torch.nextafter(x, x.new_tensor(9.0)), torch.nextafter(x, x.new_tensor(-9.0))])
    logits = torch.full((x.numel(), 2, 64), -math.inf)
    logits[:, :, 3] = 0.0
    logits[:, 0, 60] = x
    logits[:, 1, 60] = torch.log(torch.expm1(n / 4096)).float().repeat(3)
    logits, scores = logits.cuda(), torch.full((x.numel(), 2), -2.0 ** 40, device="cuda")
    want = select_reference(logits, scores, 2)
    assert 0 < int((want[1][:, 0] == 1).sum()) < x.numel() and bool((want[2] == 3).all())  # (some of each)
    got = ops.beam_select(logits, scores)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 4, 140003, 8), (1, 8, 140003, 4), (2, 8, 70001, 8), (4, 4, 131072, 16), (1, 2, 66000, 32), (3, 5, 40000, 12)], ids=str)
def test_beams_of_long_rows_in_parts(ops, shape, dtype):
    """Few candidates of few long rows, which are cut into parts: masked rows, flat ones, one whose parts but the last are empty, beams that end, rows that are
    not finite in one part, and beams that lie next to one another."""
    g, k, v, top = shape
    for masked in (False, True):
        logits, scores, flags = inputs(g, k, v, dtype, 31, masked=masked)
        check_select(ops.beam_select(logits, scores, top=top, ended=flags, end_token=v - 1), select_reference(logits, scores, top, flags, v - 1), v)
    logits[:, 0] = -math.inf
    logits[:, 0, v - 5:] = 1.5
    logits[:, k - 1, 70:] = -math.inf
    check_select(ops.beam_select(logits, scores, top=top), select_reference(logits, scores, top), v)
    logits[0, k // 2, v - 2] = math.inf
    logits[g - 1, 0, v // 2] = math.nan
    check_select(ops.beam_select(logits, scores, top=top), select_reference(logits, scores, top), v)
    flat = torch.zeros(g, k, v, device="cuda", dtype=dtype)
    scores[:] = -1.0
    check_select(ops.beam_select(flat, scores, top=top), select_reference(flat, scores, top), v)
    logits, _, _ = inputs(g, k, v, dtype, 32)
    lse = torch.logsumexp(logits.double(), dim=2)
    scores = (-20.0 - (logits.double().amax(dim=2) - lse)).float()
    want = select_reference(logits, scores, top)
    assert bool((want[0][:, 0] - want[0][:, 1] < 4e-6).all())  # (near indeed)
    check_select(ops.beam_select(logits, scores, top=top), want, v)
