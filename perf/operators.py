"""Cases for the operators between the projections of a decoder block: rotary positions, block tables and slot maps,
the paged cache held in 4 bits, and the attention that reads it.

Every case is one call (or the pair of calls a serving step makes together) on inputs of real use.  `own` chooses between
the plain form, elementary torch operations in 32 bits, and the framework's calls.

The cache of one layer, block by block (`bs` tokens each, `h` heads, `d` elements a head):
  k_codes [blocks, h, bs, d/2] bytes       byte j of a token holds elements 2j (low four bits) and 2j + 1 (high)
  v_codes [blocks, h, bs/2, d/4, 2, 2]     two tokens share a row of words: four elements of the even token, then the
                                           same four of the odd one, packed as above
  k_params, v_params [blocks, h, bs, 2]    BF16 scale and minimum of the token's vector; value = minimum + scale * code
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GUARD = 4  # rows behind the last token


def listed():
    return [
        # one decode step of 16 requests: every head rotated, bf16; nothing but latency
        dict(name="rope_decode", kind="rope", tokens=16, q_heads=32, k_heads=8, head_dim=128, rotary_dim=128, layout="half",
             scaling="none", dtype="bf16", far=8191, mix=1),
        # a long prompt: a quarter of each wide head, neighbouring pairs, positions near a million, frequencies stretched
        dict(name="rope_prompt_far", kind="rope", tokens=16383, q_heads=16, k_heads=4, head_dim=256, rotary_dim=64,
             layout="interleaved", scaling="yarn", dtype="fp16", far=1000000, mix=2),
        # the tables of one decode step
        dict(name="tables_decode", kind="tables", requests=64, cached=4000, new=1, block_size=16, mix=3),
        # a large batch: prompts, drafts and idle requests together, part of the drafts given back
        dict(name="tables_mixed", kind="tables", requests=1000, cached=3000, new=400, block_size=64, mix=4),
        # the keys and values of one decode step, 8 heads
        dict(name="append_decode", kind="append", requests=64, cached=2000, new=1, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16", mix=5),
        # the keys and values of prompts of 16 thousand tokens in all
        dict(name="append_prompt", kind="append", requests=5, cached=100, new=4500, kv_heads=8, head_dim=128, block_size=64,
             dtype="bf16", mix=6),
        # one request's next token, a short context (hidden 1024 as 8 heads of 128)
        dict(name="attend_one_short", kind="attend", requests=1, length=333, new=1, q_heads=8, kv_heads=2, head_dim=128,
             block_size=16, dtype="bf16", window=0, mix=7),
        # a serving batch: 64 requests of up to 6 thousand tokens, 64 query heads on 8 (hidden 8192)
        dict(name="attend_batch", kind="attend", requests=64, length=6000, new=1, q_heads=64, kv_heads=8, head_dim=128,
             block_size=64, dtype="bf16", window=0, mix=8),
        # one request far into a long context: the length is all there is to split
        dict(name="attend_one_long", kind="attend", requests=1, length=200003, new=1, q_heads=32, kv_heads=8, head_dim=128,
             block_size=32, dtype="bf16", window=0, mix=9),
        # four drafted tokens and the last accepted one, wide heads
        dict(name="attend_drafts", kind="attend", requests=12, length=9000, new=5, q_heads=8, kv_heads=2, head_dim=256,
             block_size=64, dtype="bf16", window=0, mix=10),
        # as many key heads as query heads, narrow, each token sees the last 1000 only (hidden 1024 as 16 heads of 64)
        dict(name="attend_window", kind="attend", requests=33, length=5000, new=1, q_heads=16, kv_heads=16, head_dim=64,
             block_size=16, dtype="fp16", window=1000, mix=11),
        # prompts behind a shared context: two thousand rows and more each
        dict(name="attend_prompt", kind="attend", requests=3, length=8100, new=4000, q_heads=32, kv_heads=8, head_dim=128,
             block_size=64, dtype="bf16", window=0, mix=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "tables", "append", "attend", "attend", "attend"])
    mix = rng.randrange(1 << 30)
    block_size = rng.choice([16, 32, 64, 128])
    if kind == "rope":
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        q = kv * rng.choice([1, 2, 5, 8])
        return dict(kind=kind, tokens=_log(rng, 1, min(16000, 40000000 // ((q + kv) * dim))), q_heads=q, k_heads=kv, head_dim=dim,
                    rotary_dim=rng.choice([dim, dim // 2, 32, 24]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "banded"]), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    far=_log(rng, 100, 1000000), mix=mix)
    if kind == "tables":
        return dict(kind=kind, requests=_log(rng, 1, 1500), cached=_log(rng, 1, 4000), new=_log(rng, 1, 200), block_size=block_size, mix=mix)
    if kind == "append":
        return dict(kind=kind, requests=_log(rng, 1, 40), cached=_log(rng, 1, 3000), new=_log(rng, 1, 200), kv_heads=rng.choice([1, 2, 4, 8]),
                    head_dim=rng.choice([64, 128, 256]), block_size=block_size, dtype=rng.choice(["bf16", "fp16", "fp32"]), mix=mix)
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16])
    common = dict(kind=kind, q_heads=kv * group, kv_heads=kv, head_dim=rng.choice([64, 128, 256]), block_size=block_size,
                  dtype=rng.choice(["bf16", "fp16"]), window=rng.choice([0, 0, 0, _log(rng, 1, 3000)]), mix=mix)
    if rng.random() < 0.6:
        requests = _log(rng, 1, 64)
        return dict(common, requests=requests, length=_log(rng, 1, 100000 // requests), new=rng.choice([1, 1, 1, 2, 4, 9]))
    requests = rng.choice([1, 2, 3, 5])
    length = _log(rng, 32, min(8000 // requests, int(math.sqrt(3e11 / (requests * common["q_heads"] * common["head_dim"])))))
    return dict(common, requests=requests, length=length, new=_log(rng, 16, length))


# ---- sizes of a case: a function of the case alone ------------------------------------------------------------------
def _lengths(case):
    """(tokens in the cache before the step, tokens of the step) of every request; ragged, some requests idle."""
    rng = random.Random(case["mix"])
    cached, new = [], []
    for r in range(case["requests"]):
        if case["kind"] == "attend":
            total = max(1, case["length"] if r == 0 else int(case["length"] * (0.3 + 0.7 * rng.random())))
            n = case["new"]
            if n > 16 and r:
                n = int(n * (0.3 + 0.7 * rng.random()))
            n = max(1, min(n, total))
            cached.append(total - n)
            new.append(n)
        else:
            cached.append(int(case["cached"] * rng.random()))
            n = case["new"]
            if n > 1 and r:
                n = 0 if rng.random() < 0.05 else 1 + int(n * rng.random())
            new.append(n)
    return cached, new


def _blocks(tokens, size):
    return -(-tokens // size)


def _visible(case):
    """Per request (query rows, cache tokens that some row sees, pairs of a row and a token it sees)."""
    out = []
    for c, n in zip(*_lengths(case)):
        window = case["window"] or c + n
        pairs = sum(min(c + i + 1, window) for i in range(n))
        out.append((n, c + n - max(0, c + 1 - window), pairs))
    return out


def work(case):
    if case["kind"] == "rope":
        size = 4 if case["dtype"] == "fp32" else 2
        heads = case["tokens"] * (case["q_heads"] + case["k_heads"])
        return {"bytes": 2 * heads * case["head_dim"] * size + 4 * case["tokens"], "flops": 3 * heads * case["rotary_dim"]}
    cached, new = _lengths(case)
    tokens = sum(new)
    if case["kind"] == "tables":
        bs = case["block_size"]
        fresh = sum(_blocks(c + n, bs) - _blocks(c, bs) for c, n in zip(cached, new))
        back = sum(_blocks(c + n, bs) - _blocks(c + k, bs) for c, n, k in zip(cached, new, _kept(case, new)))
        return {"bytes": 8 * tokens + 8 * fresh + 8 * back + 28 * case["requests"], "flops": tokens + case["requests"]}
    dim, heads = case["head_dim"], case["kv_heads"]
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "fp32" else 2
        vectors = 2 * tokens * heads
        return {"bytes": 2 * vectors * dim * size + 2 * vectors * (dim // 2 + 4) + 4 * tokens, "flops": 8 * vectors * dim}
    seen = _visible(case)
    bytes_ = sum(t for _, t, _ in seen) * heads * (dim + 8) + 2 * 2 * sum(n for n, _, _ in seen) * case["q_heads"] * dim
    return {"bytes": bytes_, "flops": 4 * sum(p for _, _, p in seen) * case["q_heads"] * dim}


def _kept(case, new):
    """Tokens of the step that stay when part of the drafts is given back."""
    rng = random.Random(case["mix"] + 1)
    return [int((n + 1) * rng.random()) for n in new]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _scaling(case):
    return {"none": {}, "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=4.0),
            "yarn": dict(scaling="yarn", factor=8.0, original=32768, fast=32.0, slow=1.0),
            "banded": dict(scaling="banded", factor=8.0, original=8192, fast=4.0, slow=1.0)}[case["scaling"]]


def _keys_values(gen, tokens, heads, dim, dtype):
    """Keys with a few strong channels and values without, as projections give them."""
    k = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    k *= 1.0 + 4.0 * (torch.rand((heads, dim), generator=gen, device="cuda") > 0.95)
    k += 0.5 * torch.randn((heads, dim), generator=gen, device="cuda")
    v = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    return k.to(dtype), v.to(dtype)


def _empty_cache(gen, blocks, heads, bs, dim):
    """A cache as it is found: memory that other requests have used, and parameters that are no numbers."""
    make = dict(generator=gen, dtype=torch.uint8, device="cuda")
    return dict(k_codes=torch.randint(0, 256, (blocks, heads, bs, dim // 2), **make),
                v_codes=torch.randint(0, 256, (blocks, heads, bs // 2, dim // 4, 2, 2), **make),
                k_params=torch.full((blocks, heads, bs, 2), math.nan, dtype=torch.bfloat16, device="cuda"),
                v_params=torch.full((blocks, heads, bs, 2), math.nan, dtype=torch.bfloat16, device="cuda"))


def _table(gen, counts, spare):
    """Rows of block numbers for `counts` blocks a request, taken out of a shuffled pool; the rest of the pool."""
    pool = torch.randperm(sum(counts) + spare, generator=gen, device="cuda").to(torch.int32)
    width = max(max(counts), 1)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = pool[at:at + n]
        at += n
    return table, pool[at:].clone()


def _slots(table, bs, cached, new):
    """The slot of every token of the step, requests one after another."""
    rows = []
    for r, (c, n) in enumerate(zip(cached, new)):
        pos = torch.arange(c, c + n, device="cuda")
        rows.append(table[r, pos // bs].long() * bs + pos % bs)
    return torch.cat(rows).to(torch.int32)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["mix"] % 1000003)
    if case["kind"] == "rope":
        dtype, n, dim = DTYPES[case["dtype"]], case["tokens"], case["head_dim"]
        q = torch.randn((n, case["q_heads"], dim), generator=gen, device="cuda").to(dtype)
        k = torch.randn((n, case["k_heads"], dim), generator=gen, device="cuda").to(dtype)
        start = torch.randint(0, case["far"] + 1, (1,), generator=gen, device="cuda")
        return dict(q=q, k=k, positions=((start + torch.arange(n, device="cuda")) % (case["far"] + 1)).to(torch.int32))
    cached, new = _lengths(case)
    bs = case["block_size"]
    if case["kind"] == "tables":
        width = max(_blocks(c + n, bs) for c, n in zip(cached, new))
        before, _ = _table(gen, [_blocks(c, bs) for c in cached], 0)
        fresh = sum(_blocks(c + n, bs) - _blocks(c, bs) for c, n in zip(cached, new))
        held = sum(_blocks(c, bs) for c in cached)
        table = torch.full((len(cached), max(width, 1)), -1, dtype=torch.int32, device="cuda")
        table[:, :min(before.shape[1], table.shape[1])] = before[:, :table.shape[1]]
        free = torch.zeros(held + fresh + 7, dtype=torch.int32, device="cuda")
        free[:fresh + 7] = held + torch.randperm(fresh + 7, generator=gen, device="cuda").to(torch.int32)
        return dict(table=table, free=free, count=_ints([fresh + 7]), blocks=held + fresh + 7, cached=_ints(cached), new=_ints(new),
                    keep=_ints([c + k for c, k in zip(cached, _kept(case, new))]), capacity=sum(new) + GUARD)
    heads, dim, dtype = case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    table, _ = _table(gen, [_blocks(c + n, bs) for c, n in zip(cached, new)], 5)
    cache = _empty_cache(gen, int(table.max()) + 5, heads, bs, dim)
    if case["kind"] == "append":
        k, v = _keys_values(gen, sum(new), heads, dim, dtype)
        return dict(cache=cache, k=k, v=v, slots=_slots(table, bs, cached, new))
    for r, total in enumerate(c + n for c, n in zip(cached, new)):  # what earlier steps have stored
        for at in range(0, total, 16384):
            n = min(16384, total - at)
            k, v = _keys_values(gen, n, heads, dim, dtype)
            _plain_append(cache, bs, k, v, _slots(table[r:r + 1], bs, [at], [n]).long())
    q = torch.randn((sum(new) + GUARD, case["q_heads"], dim), generator=gen, device="cuda").to(dtype)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(cache=cache, table=table, q=q, lens=_ints([c + n for c, n in zip(cached, new)]), starts=_ints(starts))


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] == "rope":
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
        if not own:
            state["turns"], state["amplitude"] = _plain_turns(case)
    elif case["kind"] == "tables":
        n = case["requests"]
        state.update(table2=state["table"].clone(), free2=state["free"].clone(), count_out=_ints([0]), count2=_ints([0]), status=_ints([0, 0]),
                     status2=_ints([0, 0]), total=_ints([0] * n), total2=_ints([0] * n), starts=_ints([0] * (n + 1)),
                     slots=_ints([0] * state["capacity"]), positions=_ints([0] * state["capacity"]))
    elif case["kind"] == "append":
        state["k_back"], state["v_back"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
    else:
        state["out"] = torch.zeros_like(state["q"])
        state["host"] = [(c + n, n) for c, n in zip(*_lengths(case))]
    if own:
        state["calls"] = _own_calls(case, state)
    return state


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _own_calls(case, state):
    import infer_b200 as B
    kinds = {"bf16": B.BF16, "fp16": B.FP16, "fp32": B.FP32}
    if case["kind"] == "rope":
        host, amplitude = B.rope_turns(case["rotary_dim"], base=10000.0, **_scaling(case))
        state["turns"] = torch.from_numpy(host).to("cuda")
        desc = B.rope_desc(dtype=kinds[case["dtype"]], layout=B.ROPE_HALF if case["layout"] == "half" else B.ROPE_INTERLEAVED,
                           tokens=case["tokens"], head_dim=case["head_dim"], rotary_dim=case["rotary_dim"], positions=state["positions"],
                           turns=state["turns"], amplitude=amplitude, q=state["q"], q_out=state["q_out"], q_heads=case["q_heads"],
                           k=state["k"], k_out=state["k_out"], k_heads=case["k_heads"])
        return lambda: B.rope(desc)
    if case["kind"] == "tables":
        common = dict(requests=case["requests"], max_blocks=state["table"].shape[1], block_size=case["block_size"], blocks=state["blocks"])
        assign = B.kv4_assign_desc(cached_lens=state["cached"], new_lens=state["new"], free_blocks=state["free"], free_count=state["count"],
                                   free_count_out=state["count_out"], block_table=state["table"], total_lens=state["total"],
                                   query_start=state["starts"], tokens=state["capacity"], slots=state["slots"],
                                   positions=state["positions"], status=state["status"], **common)
        release = B.kv4_release_desc(lens=state["total"], keep_lens=state["keep"], free_blocks=state["free2"], free_count=state["count_out"],
                                     free_count_out=state["count2"], block_table=state["table"], lens_out=state["total2"],
                                     status=state["status2"], **common)

        def step():
            B.kv4_assign(assign)
            B.kv4_release(release)
        return step
    c = state["cache"]
    cache = B.kv4_cache(k_codes=c["k_codes"], v_codes=c["v_codes"], k_params=c["k_params"], v_params=c["v_params"], blocks=c["k_codes"].shape[0],
                        block_size=case["block_size"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    if case["kind"] == "append":
        tokens = state["k"].shape[0]
        append = B.kv4_append_desc(cache=cache, dtype=kinds[case["dtype"]], tokens=tokens, k=state["k"], v=state["v"], slots=state["slots"])
        gather = B.kv4_gather_desc(cache=cache, dtype=kinds[case["dtype"]], tokens=tokens, slots=state["slots"], k_out=state["k_back"],
                                   v_out=state["v_back"])

        def both():
            B.kv4_append(append)
            B.kv4_gather(gather)
        return both
    desc = B.kv4_attention_desc(cache=cache, dtype=kinds[case["dtype"]], requests=case["requests"], tokens=state["q"].shape[0] - GUARD,
                                q_heads=case["q_heads"], q=state["q"], out=state["out"], block_table=state["table"],
                                max_blocks=state["table"].shape[1], total_lens=state["lens"], query_start=state["starts"],
                                max_query=max(n for _, n in state["host"]), scale=case["head_dim"] ** -0.5, causal=True, window=case["window"])
    state["workspace"] = B.kv4_attention_workspace(torch, desc)
    return lambda: B.kv4_attention(desc)


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plain_turns(case):
    """Turns per position of every pair (64 bits) and the factor of the cosines and sines."""
    dim, s = case["rotary_dim"], _scaling(case)
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    base = 10000.0
    kind = s.get("scaling", "none")
    if kind == "ntk":
        base = base * s["factor"] ** (dim / (dim - 2))
    turns = base ** (-2.0 * i / dim) / (2.0 * math.pi)
    if kind == "linear":
        return turns / s["factor"], 1.0
    if kind == "yarn":  # a linear ramp between the pairs that turn `fast` and `slow` times in the original length
        def pair(count):
            return dim * math.log(s["original"] / (count * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair(s["fast"])), 0), min(math.ceil(pair(s["slow"])), dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return turns / s["factor"] * ramp + turns * (1.0 - ramp), 0.1 * math.log(s["factor"]) + 1.0
    if kind == "banded":  # by the turns made in the original length: many are kept, few are stretched, a blend between
        made = turns * s["original"]
        keep = ((made - s["slow"]) / (s["fast"] - s["slow"])).clamp(0.0, 1.0)
        return turns * keep + turns / s["factor"] * (1.0 - keep), 1.0
    return turns, 1.0


def _plain_rope(case, state):
    angle = state["positions"].double()[:, None] * state["turns"][None, :]
    angle = (angle - angle.round()) * (2.0 * math.pi)
    cos, sin = (angle.cos() * state["amplitude"]).float()[:, None, :], (angle.sin() * state["amplitude"]).float()[:, None, :]
    r = case["rotary_dim"]
    outs = []
    for x in (state["q"], state["k"]):
        y = x.float()
        if case["layout"] == "half":
            a, b = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        else:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        outs.append(torch.cat((turned, y[..., r:]), dim=-1).to(x.dtype))
    return outs


def _plain_tables(case, state):
    bs, cached, new, table = case["block_size"], state["cached"].long(), state["new"].long(), state["table"]
    width, zero = table.shape[1], torch.zeros(1, dtype=torch.int64, device="cuda")
    total = cached + new
    have, need = (cached + bs - 1) // bs, (total + bs - 1) // bs
    first = torch.cat((zero, (need - have).cumsum(0)))
    column = torch.arange(width, device="cuda")[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    order = first[:-1, None] + column - have[:, None]
    top = state["count"].long() - 1
    table = torch.where(fresh, state["free"][(top - order).clamp(0, state["blocks"] - 1)], table)
    starts = torch.cat((zero, new.cumsum(0)))
    row = torch.arange(state["capacity"], device="cuda")
    request = (torch.searchsorted(starts, row, right=True) - 1).clamp(0, case["requests"] - 1)
    position = row - starts[request] + cached[request]
    inside = row < starts[-1]
    slot = table[request, (position // bs).clamp(0, width - 1)].long() * bs + position % bs
    count = state["count"].long() - first[-1]
    # what is given back goes on the stack so that the block taken last lies deepest
    keep = state["keep"].long()
    kept = (keep + bs - 1) // bs
    back = torch.cat((zero, (need - kept).cumsum(0)))
    gone = (column >= kept[:, None]) & (column < need[:, None])
    place = count + back[-1] - 1 - (back[:-1, None] + column - kept[:, None])
    free = torch.cat((state["free2"], state["free2"][:1]))  # one place more for the entries that stay where they are
    free[torch.where(gone, place, state["blocks"]).flatten()] = table.flatten()
    out = dict(table=table, total=total, starts=starts, slots=torch.where(inside, slot, -1), positions=torch.where(inside, position, -1),
               count=count, free=free[:-1], count2=count + back[-1], total2=keep, status=zero, status2=zero)
    return {name: t.to(torch.int32) for name, t in out.items()}


def _plain_quantise(x):
    """Codes (0 .. 15) and BF16 scale and minimum of every vector; borders are decided in 64 bits."""
    x = x.float()
    low, high = x.amin(-1), x.amax(-1)
    minimum = low.to(torch.bfloat16)
    bits = minimum.view(torch.int16)
    step = torch.where(bits < 0, 1, -1).to(torch.int16)  # one BF16 number down
    minimum = torch.where(minimum.float() > low, bits + step, bits).view(torch.bfloat16)
    spread = high.double() - minimum.double()
    scale = (spread / 15.0).to(torch.float32).to(torch.bfloat16)
    bits = scale.view(torch.int16)
    bits = torch.where(15.0 * scale.double() < spread, bits + 1, bits)
    below = (bits - 1).view(torch.bfloat16)
    bits = torch.where((bits > 0) & (15.0 * below.double() >= spread), bits - 1, bits)
    scale = bits.to(torch.int16).view(torch.bfloat16)
    scale = torch.where((spread > 0) & (scale.float() < 2.0 ** -126), 2.0 ** -126, scale.float()).to(torch.bfloat16)
    inverse = torch.where(spread > 0, scale.double(), 1.0)
    codes = ((x.double() - minimum.double()[..., None]) / inverse[..., None]).round().clamp(0.0, 15.0)
    return codes.to(torch.uint8), torch.stack((scale, minimum), dim=-1)


def _plain_append(cache, bs, k, v, slots):
    block, off = slots // bs, slots % bs
    codes, params = _plain_quantise(k)
    cache["k_codes"][block, :, off] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    cache["k_params"][block, :, off] = params
    codes, params = _plain_quantise(v)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    cache["v_codes"][block, :, off // 2, :, off % 2] = packed.unflatten(-1, (-1, 2))
    cache["v_params"][block, :, off] = params


def _plain_values(packed, params):
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2).float()
    return params[..., 1:].float() + params[..., :1].float() * codes


def _plain_read(cache, bs, slots):
    """Keys and values of slots, [tokens, heads, dim] in 32 bits."""
    block, off = slots // bs, slots % bs
    k = _plain_values(cache["k_codes"][block, :, off], cache["k_params"][block, :, off])
    v = _plain_values(cache["v_codes"][block, :, off // 2, :, off % 2].flatten(-2), cache["v_params"][block, :, off])
    return k, v


def _plain_attend(case, state):
    group, bs, scale = case["q_heads"] // case["kv_heads"], case["block_size"], case["head_dim"] ** -0.5
    out, row = state["out"], 0
    for r, (total, n) in enumerate(state["host"]):
        first = max(0, total - n + 1 - case["window"]) if case["window"] else 0
        pos = torch.arange(first, total, device="cuda")
        k, v = _plain_read(state["cache"], bs, state["table"][r, pos // bs].long() * bs + pos % bs)
        k, v = k.permute(1, 2, 0), v.transpose(0, 1)
        rows = max(1, min(n, (1 << 28) // (case["q_heads"] * pos.numel())))
        for at in range(0, n, rows):
            m = min(rows, n - at)
            q = state["q"][row + at:row + at + m].float().unflatten(1, (-1, group)).permute(1, 2, 0, 3).flatten(1, 2)
            scores = torch.matmul(q, k) * scale
            me = (total - n + at + torch.arange(m, device="cuda")).repeat(group)[:, None]
            hidden = pos[None, :] > me
            if case["window"]:
                hidden = hidden | (pos[None, :] <= me - case["window"])
            scores = scores.masked_fill(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            y = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            out[row + at:row + at + m] = y.unflatten(1, (group, m)).permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
        row += n
    return out


def run(state):
    case = state["case"]
    if own:
        state["calls"]()
        if case["kind"] == "rope":
            return [state["q_out"], state["k_out"]]
        if case["kind"] == "tables":
            return dict(table=state["table"], total=state["total"], starts=state["starts"], slots=state["slots"],
                        positions=state["positions"], count=state["count_out"], free=state["free2"], count2=state["count2"],
                        total2=state["total2"], status=state["status"][:1], status2=state["status2"][:1])
        if case["kind"] == "append":
            return [state["k_back"], state["v_back"]]
        return state["out"]
    if case["kind"] == "rope":
        return _plain_rope(case, state)
    if case["kind"] == "tables":
        return _plain_tables(case, state)
    if case["kind"] == "append":
        slots = state["slots"].long()
        _plain_append(state["cache"], case["block_size"], state["k"], state["v"], slots)
        return [x.to(y.dtype) for x, y in zip(_plain_read(state["cache"], case["block_size"], slots), (state["k"], state["v"]))]
    return _plain_attend(case, state)


# ---- the definitions in 64 bits, apart from all of the above ---------------------------------------------------------
def _exact_turns(case):
    dim, s = case["rotary_dim"], _scaling(case)
    kind, base, amplitude, turns = s.get("scaling", "none"), 10000.0, 1.0, []
    if kind == "ntk":
        base *= math.pow(s["factor"], dim / (dim - 2.0))
    if kind == "yarn":
        amplitude = 1.0 + math.log(s["factor"]) / 10.0
        edges = [dim * math.log(s["original"] / (2.0 * math.pi * c)) / math.log(base) / 2.0 for c in (s["fast"], s["slow"])]
        low, high = max(0, math.floor(edges[0])), min(dim - 1, math.ceil(edges[1]))
    for i in range(dim // 2):
        t = math.exp(-math.log(base) * 2.0 * i / dim) / (2.0 * math.pi)
        if kind == "linear":
            t /= s["factor"]
        elif kind == "yarn":
            mix = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            t = mix * t / s["factor"] + (1.0 - mix) * t
        elif kind == "banded":
            mix = min(1.0, max(0.0, (t * s["original"] - s["slow"]) / (s["fast"] - s["slow"])))
            t = mix * t + (1.0 - mix) * t / s["factor"]
        turns.append(t)
    return np.array(turns), amplitude


def _exact_rope(case, inputs):
    turns, amplitude = _exact_turns(case)
    phase = inputs["positions"].cpu().numpy().astype(np.float64)[:, None] * turns
    z = torch.from_numpy(amplitude * np.exp(2j * np.pi * (phase - np.floor(phase)))).cuda()[:, None, :]
    r, outs = case["rotary_dim"], []
    for x in (inputs["q"], inputs["k"]):
        y = x.double()
        one, two = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        w = torch.complex(y[..., one], y[..., two]) * z
        out = y.clone()
        out[..., one], out[..., two] = w.real, w.imag
        outs.append(out)
    return outs


def _exact_tables(case, inputs):
    bs = case["block_size"]
    table, stack = inputs["table"].cpu().tolist(), inputs["free"].cpu().tolist()
    other, top = list(stack), int(inputs["count"][0])
    cached, new = _lengths(case)
    slots, positions, starts = [], [], [0]
    for r, (c, n) in enumerate(zip(cached, new)):
        for b in range(_blocks(c, bs), _blocks(c + n, bs)):
            top -= 1
            table[r][b] = stack[top]
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r][p // bs] * bs + p % bs)
        starts.append(starts[-1] + n)
    keep = [c + k for c, k in zip(cached, _kept(case, new))]
    back = [table[r][b] for r, k in enumerate(keep) for b in range(_blocks(k, bs), _blocks(cached[r] + new[r], bs))]
    other[top:top + len(back)] = back[::-1]
    out = dict(table=table, total=[c + n for c, n in zip(cached, new)], starts=starts, slots=slots + [-1] * GUARD,
               positions=positions + [-1] * GUARD, count=[top], free=other, count2=[top + len(back)], total2=keep, status=[0], status2=[0])
    return {name: _ints(values) for name, values in out.items()}


def _exact_append(x):
    x = x.double()

    def eight_bits(value, rounded):  # to eight significant bits, down or up
        m, e = torch.frexp(value)
        return torch.ldexp(rounded(m * 256.0) / 256.0, e)
    low = eight_bits(x.amin(-1), torch.floor)
    step = eight_bits((x.amax(-1) - low) / 15.0, torch.ceil)
    low, step = low[..., None], step[..., None]
    return low + step * torch.clamp(torch.round((x - low) / torch.where(step > 0, step, 1.0)), 0, 15)


def _exact_attend(case, inputs):
    c, bs, dim, heads = inputs["cache"], case["block_size"], case["head_dim"], case["kv_heads"]
    group = case["q_heads"] // heads
    table = inputs["table"].long()
    out = torch.zeros(inputs["q"].shape, dtype=torch.float64, device="cuda")
    shift = torch.tensor([0, 4], device="cuda")
    row = 0
    for r, (cached, n) in enumerate(zip(*_lengths(case))):
        total = cached + n
        mine = table[r, :_blocks(total, bs)]
        for h in range(heads):
            def full(codes, params):
                return (params[:, 1].double()[:, None] + params[:, 0].double()[:, None] * codes.double())[:total]
            kc = ((c["k_codes"][mine, h].to(torch.int32)[..., None] >> shift) & 15).reshape(-1, dim)
            vc = ((c["v_codes"][mine, h].to(torch.int32)[..., None] >> shift) & 15).reshape(-1, dim // 4, 2, 4)
            vc = vc.transpose(1, 2).reshape(-1, dim)
            k, v = full(kc, c["k_params"][mine, h].reshape(-1, 2)), full(vc, c["v_params"][mine, h].reshape(-1, 2))
            for i in range(0, n, 512):
                m = min(512, n - i)
                q = inputs["q"][row + i:row + i + m, h * group:(h + 1) * group].double()
                s = torch.einsum("mgd,td->mgt", q, k) / math.sqrt(dim)
                t = torch.arange(total, device="cuda")[None, :]
                at = cached + i + torch.arange(m, device="cuda")[:, None]
                seen = t <= at
                if case["window"]:
                    seen &= t > at - case["window"]
                w = torch.softmax(torch.where(seen[:, None, :], s, -math.inf), dim=-1)
                out[row + i:row + i + m, h * group:(h + 1) * group] = torch.einsum("mgt,td->mgd", w, v)
        row += n
    return out


def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, inputs)
    if case["kind"] == "tables":
        return _exact_tables(case, inputs)
    if case["kind"] == "append":
        return [_exact_append(inputs["k"]), _exact_append(inputs["v"])]
    return _exact_attend(case, inputs)
