"""The operators of a sequence model's prompt, of its single tokens and of its answers, as cases for a timing harness.

``functs_b200.ops.linear_attention``        attention with a decaying state per head over whole prompts (beside the LSTM)
``functs_b200.ops.linear_attention_step``   the same for one token per sequence, on a pool of states
``functs_b200.ops.token_logprobs``          log probabilities of given tokens, entropies, best alternatives (beside softmax + top-k)

listed()         named cases, from the smallest call to the largest
draw(rng)        one more case of the same ranges
prepare(case, seed), run(state), work(case), exact(case, seed)

``own`` says whether run() calls the package's operators or their plain form in elementary torch operations.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
CHUNK = 64  # tokens per chunk of the plain form
MOST_ROWS = 16 * 2048 * 16 * 128 * 17 // 32  # tokens x heads x channels of the largest listed prompt (its padding left out)
MOST_STATE = 96 * 16 * 128 * 128


def listed():
    return [
        # a short question to one sequence model in the framework's own type: latency
        {"name": "prompt b1 t24 h8 d64 f32", "kind": "prompt", "dtype": "f32", "batch": 1, "tokens": 24, "heads": 8, "kv_heads": 8, "dk": 64,
         "dv": 64, "layout": "batch", "ragged": False, "pool": False},
        # a padded batch of uneven prompts that go on from earlier states; odd head sizes, three query heads per key head
        {"name": "prompt b5 t517 h6 d80x48 f16", "kind": "prompt", "dtype": "f16", "batch": 5, "tokens": 517, "heads": 6, "kv_heads": 2, "dk": 80,
         "dv": 48, "layout": "batch", "ragged": True, "pool": True},
        # a batch of sequences in the time-major layout of the LSTM, in its type
        {"name": "prompt b8 t1024 h8 d64 f32 time", "kind": "prompt", "dtype": "f32", "batch": 8, "tokens": 1024, "heads": 8, "kv_heads": 8,
         "dk": 64, "dv": 64, "layout": "time", "ragged": False, "pool": False},
        # one long document: few heads, many tokens
        {"name": "prompt b1 t8192 h16 d128 bf16", "kind": "prompt", "dtype": "bf16", "batch": 1, "tokens": 8192, "heads": 16, "kv_heads": 16,
         "dk": 128, "dv": 128, "layout": "fused", "ragged": False, "pool": False},
        # a full padded batch of uneven prompts, continued from the pool's states: the largest call
        {"name": "prompt b16 t2048 h16 d128 bf16", "kind": "prompt", "dtype": "bf16", "batch": 16, "tokens": 2048, "heads": 16, "kv_heads": 16,
         "dk": 128, "dv": 128, "layout": "fused", "ragged": True, "pool": True},
        # one token of one sequence: latency
        {"name": "step b1 h16 d128 bf16", "kind": "step", "dtype": "bf16", "batch": 1, "heads": 16, "kv_heads": 16, "dk": 128, "dv": 128,
         "layout": "fused", "pool": False},
        # a batch of sequences with odd head sizes and shared keys, states in any order in their pool
        {"name": "step b33 h12 d72x40 f32", "kind": "step", "dtype": "f32", "batch": 33, "heads": 12, "kv_heads": 4, "dk": 72, "dv": 40,
         "layout": "batch", "pool": True},
        # a full serving batch: the states' traffic is everything
        {"name": "step b96 h16 d128 bf16", "kind": "step", "dtype": "bf16", "batch": 96, "heads": 16, "kv_heads": 16, "dk": 128, "dv": 128,
         "layout": "fused", "pool": True},
        # the answer of one sequence, with five alternatives: latency
        {"name": "logprobs r1 v32000 f32 top5", "kind": "logprobs", "dtype": "f32", "rows": 1, "vocab": 32000, "top": 5, "masked": False},
        # a batch under a constraint that leaves a fifth of an odd vocabulary
        {"name": "logprobs r48 v50001 f16 top20", "kind": "logprobs", "dtype": "f16", "rows": 48, "vocab": 50001, "top": 20, "masked": True},
        # a serving batch, large vocabulary, alternatives wanted
        {"name": "logprobs r256 v131072 bf16 top20", "kind": "logprobs", "dtype": "bf16", "rows": 256, "vocab": 131072, "top": 20, "masked": False},
        # scoring whole prompts: every position's token, no alternatives
        {"name": "logprobs r4096 v32000 bf16", "kind": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 32000, "top": 0, "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "step", "logprobs"))
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    if kind == "logprobs":
        vocab = _log(rng, 100, 262144)
        rows = _log(rng, 1, min(4096, max(1, 4096 * 32000 // vocab)))
        if dtype == "f32":
            rows = max(1, rows // 2)
        return {"kind": kind, "dtype": dtype, "rows": rows, "vocab": vocab, "top": rng.choice((0, 1, 5, 20, rng.randint(2, 50))),
                "masked": rng.random() < 0.3}
    group = rng.choice((1, 1, 1, 2, 3, 4))
    kv_heads = _log(rng, 1, 32 // group)
    dk = rng.choice((64, 128, 128, rng.randint(16, 128)))
    dv = rng.choice((dk, dk, rng.randint(16, 128)))
    head = {"kind": kind, "dtype": dtype, "heads": kv_heads * group, "kv_heads": kv_heads, "dk": dk, "dv": dv,
            "layout": rng.choice(("batch", "fused")), "pool": rng.random() < 0.5}
    if kind == "step":
        head["batch"] = _log(rng, 1, min(512, max(1, MOST_STATE // (kv_heads * group * dk * dv))))
        return head
    rows = MOST_ROWS * 2 // (SIZES[dtype] * kv_heads * group * max(dk, dv))  # tokens that the largest listed prompt's traffic pays for
    tokens = min(_log(rng, 1, 8192), rows)
    head.update(tokens=tokens, batch=_log(rng, 1, min(64, rows // tokens)), ragged=rng.random() < 0.5)
    head["layout"] = rng.choice(("batch", "fused", "time"))
    return head


def _lengths(case):
    """Tokens of each sequence: from all of them down to none, in an order of their own."""
    b, t = case["batch"], case["tokens"]
    if not case.get("ragged"):
        return [t] * b
    got = [t - (i * t) // max(1, b - 1) if b > 1 else (t + 1) // 2 for i in range(b)]
    random.Random(b * 10007 + t).shuffle(got)
    return got


def _heads(case, gen, shape, time_major=False):
    """q, k, v of sizes shape + [heads, channels]: tensors of their own, or the three parts of one fused projection."""
    h, g, dk, dv, dtype = case["heads"], case["kv_heads"], case["dk"], case["dv"], DTYPES[case["dtype"]]
    if time_major:
        shape = (shape[1], shape[0])
    if case["layout"] == "fused":
        x = torch.randn(*shape, h * dk + g * dk + g * dv, generator=gen, device=DEVICE).to(dtype)
        q, k, v = x.split([h * dk, g * dk, g * dv], dim=-1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (g, dk)), v.unflatten(-1, (g, dv))
    qkv = [torch.randn(*shape, n, d, generator=gen, device=DEVICE).to(dtype) for n, d in ((h, dk), (g, dk), (g, dv))]
    return tuple(x.transpose(0, 1) for x in qkv) if time_major else tuple(qkv)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    st = dict(case)
    if case["kind"] == "logprobs":
        r, n = case["rows"], case["vocab"]
        logits = torch.randn(r, n, generator=gen, device=DEVICE) * 3
        if case["masked"]:
            logits.masked_fill_(torch.rand(n, generator=gen, device=DEVICE) > 0.2, -math.inf)
            logits[:, 0] = 0.0  # (a token that ends the text stays)
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        st["ids"] = torch.randint(0, n, (r,), generator=gen, device=DEVICE)
        return st
    b, h, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    shape = (b, case["tokens"]) if case["kind"] == "prompt" else (b,)
    st["q"], st["k"], st["v"] = _heads(case, gen, shape, case["layout"] == "time")
    # heads that forget within two tokens up to heads that remember some 250
    st["log_decay"] = -torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEVICE, dtype=torch.float32) / h)
    st["scale"] = dk ** -0.5
    st["state"] = st["slots"] = st["lengths"] = None
    if case["pool"]:
        n = b + b // 4 + 1
        st["state"] = torch.randn(n, h, dk, dv, generator=gen, device=DEVICE) * 4
        st["slots"] = torch.randperm(n, generator=gen, device=DEVICE)[:b].to(torch.int32)
    elif case["kind"] == "step":
        st["state"] = torch.randn(b, h, dk, dv, generator=gen, device=DEVICE) * 4
    if case.get("ragged"):
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _plain_start(st):
    return st["state"] if st["slots"] is None else st["state"][st["slots"].long()]


def _plain_end(st, final):
    if st["slots"] is None:
        st["state"].copy_(final)
    else:
        st["state"][st["slots"].long()] = final
    return st["state"]


def _plain_prompt(st):
    group = st["heads"] // st["kv_heads"]
    q = st["q"].float().transpose(1, 2)  # [B, H, T, D]
    k = st["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = st["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    b, h, t, dk = q.shape
    dv = v.size(-1)
    g = st["log_decay"].view(1, h, 1)
    at = torch.arange(t, device=q.device)
    length = torch.full((b,), t, device=q.device) if st["lengths"] is None else st["lengths"]
    there = at.view(1, 1, t) < length.view(b, 1, 1)
    k = k * there[..., None]
    v = v * there[..., None]
    first = None if st["state"] is None else _plain_start(st)
    # the state behind the last token of each sequence
    left = (length.view(b, 1, 1) - 1 - at).clamp(min=0)
    final = (k * torch.exp(g * left)[..., None]).transpose(2, 3) @ v
    if first is not None:
        final = final + torch.exp(g * length.view(b, 1, 1))[..., None] * first
    # outputs, a chunk of tokens at a time: within the chunk, and from the state in front of it
    n = -(-t // CHUNK)
    pad = (0, 0, 0, n * CHUNK - t)
    q, k, v = (torch.nn.functional.pad(x, pad).unflatten(2, (n, CHUNK)) for x in (q, k, v))
    c = torch.arange(CHUNK, device=q.device)
    apart = c[:, None] - c[None, :]
    inside = torch.where(apart >= 0, torch.exp(g[..., None] * apart.clamp(min=0)), 0.0)  # [1, H, C, C]
    out = ((q @ k.transpose(3, 4)) * inside[:, :, None]) @ v
    ends = (k * torch.exp(g * (CHUNK - 1 - c))[:, :, None, :, None]).transpose(3, 4) @ v  # [B, H, n, Dk, Dv]
    m = torch.arange(n, device=q.device)
    chunks = m[:, None] - 1 - m[None, :]
    carry = torch.where(chunks >= 0, torch.exp(g[..., None] * CHUNK * chunks.clamp(min=0)), 0.0)  # [1, H, n, n]
    front = (carry @ ends.flatten(3)).unflatten(3, (dk, dv))
    if first is not None:
        front = front + torch.exp(g * CHUNK * m)[..., None, None] * first[:, :, None]
    out = out + (q * torch.exp(g * (c + 1))[:, :, None, :, None]) @ front
    out = out.flatten(2, 3)[:, :, :t] * st["scale"] * there[..., None]
    out = out.transpose(1, 2).to(st["q"].dtype)
    return out, (final if first is None else _plain_end(st, final))


def _plain_step(st):
    group = st["heads"] // st["kv_heads"]
    q, k, v = st["q"].float(), st["k"].float().repeat_interleave(group, 1), st["v"].float().repeat_interleave(group, 1)
    final = torch.exp(st["log_decay"])[:, None, None] * _plain_start(st) + k[..., None] * v[..., None, :]
    out = ((q[..., None, :] @ final)[..., 0, :] * st["scale"]).to(st["q"].dtype)
    return out, _plain_end(st, final)


def _plain_logprobs(st):
    x = st["logits"].float()
    most = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(dim=1, keepdim=True)
    lp = x - most - torch.log(total)
    entropy = -torch.where(e > 0, e / total * lp, 0.0).sum(dim=1)
    token = lp.gather(1, st["ids"][:, None])[:, 0]
    top = st["top"]
    if top:
        best = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    else:
        best = torch.empty(x.size(0), 0, dtype=torch.int64, device=x.device)
    return token, entropy, lp.gather(1, best), best


def run(st):
    if own:
        from functs_b200 import ops
        if st["kind"] == "logprobs":
            return ops.token_logprobs(st["logits"], st["ids"], top=st["top"])
        if st["kind"] == "step":
            out = ops.linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"], scale=st["scale"], slots=st["slots"])
            return out, st["state"]
        return ops.linear_attention(st["q"], st["k"], st["v"], st["log_decay"], scale=st["scale"], state=st["state"], slots=st["slots"],
                                    lengths=st["lengths"])
    if st["kind"] == "logprobs":
        return _plain_logprobs(st)
    return _plain_step(st) if st["kind"] == "step" else _plain_prompt(st)


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "logprobs":
        r, n = case["rows"], case["vocab"]
        return {"bytes": r * (n * size + 16 + case["top"] * 12), "flops": 4 * r * n}
    b, h, g, dk, dv = case["batch"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
    tokens = sum(_lengths(case)) if case["kind"] == "prompt" else b
    padded = b * case["tokens"] if case["kind"] == "prompt" else b
    read = tokens * (h * dk + g * (dk + dv)) * size + (b * h * dk * dv * 4 if case["pool"] or case["kind"] == "step" else 0)
    wrote = padded * h * dv * size + b * h * dk * dv * 4
    return {"bytes": read + wrote, "flops": 4 * tokens * h * dk * dv}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        x = st["logits"].double()
        total = torch.logsumexp(x, dim=1)
        p = torch.exp(x - total[:, None])
        entropy = total - (p * torch.where(p > 0, x, 0.0)).sum(dim=1)
        order = torch.argsort(-x, dim=1, stable=True)[:, : case["top"]]
        rows = torch.arange(x.size(0), device=x.device)
        return x[rows, st["ids"]] - total, entropy, torch.take_along_dim(x, order, 1) - total[:, None], order
    prompt = case["kind"] == "prompt"
    h, g = case["heads"], case["kv_heads"]
    share = torch.arange(h, device=DEVICE) // (h // g)
    pool = st["state"]
    where = torch.arange(case["batch"], device=DEVICE) if st["slots"] is None else st["slots"].long()
    s = torch.zeros(case["batch"], h, case["dk"], case["dv"], dtype=torch.float64, device=DEVICE) if pool is None else pool.double()[where]
    decay = torch.exp(st["log_decay"].double())[None, :, None, None]
    length = torch.tensor(_lengths(case) if prompt else [1] * case["batch"], device=DEVICE)
    steps = case["tokens"] if prompt else 1
    outs = torch.zeros(case["batch"], steps, h, case["dv"], dtype=torch.float64, device=DEVICE)
    for t in range(steps):
        q, k, v = ((x[:, t] if prompt else x).double() for x in (st["q"], st["k"], st["v"]))
        new = torch.einsum("bhk,bhv->bhkv", k[:, share], v[:, share]).addcmul_(decay, s)
        live = (t < length)[:, None, None, None]
        s = torch.where(live, new, s)
        outs[:, t] = torch.einsum("bhk,bhkv->bhv", q, s) * st["scale"] * live[..., 0]
    if pool is None:
        final = s
    else:
        final = pool.double()
        final[where] = s
    return (outs if prompt else outs[:, 0]), final
