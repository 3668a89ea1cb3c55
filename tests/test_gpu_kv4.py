"""GPU: rotary positions, block tables, the 4-bit cache and its attention against plain implementations in 64 bits.

Tolerances count roundings.  eps(t) / 2 is the largest relative error of one rounding to type t.
* rope: FP32 cosine and sine are within 2 units in the last place (2^-22 of 1), two products and a sum add at most three
  roundings of 2^-24 of |x1| + |x2|: 2^-21 (|x1| + |x2|) * amplitude, then one rounding to the output type.
* the cache's codes and parameters are defined exactly: bit for bit.
* attention: q and codes enter exactly, scores are FP32 sums of at most 256 products of both signs of the minimum and the
  code part.  With A = scale * sum |q| * (|min| + 15 s) the score is off by at most 2^-23 * (256 / 16 + 8) * A (the matrix
  instruction adds 16 products at a time and truncates, a unit of 2^-23 each time), which multiplies a probability by at most
  1 + that; a probability (times its scale, with few rows) is rounded to 11 bits, 2^-12.  With more than 128 rows a kv head values enter
  rounded to 11 bits, 2^-12 * |v| each, which the bound below holds room for (the probabilities' part is 2^-12 * |v| then, and
  |v| <= spread), and with BF16 queries the keys too: 2^-12 * A more on a score.  Weights off by a relative w each move a weighted mean
  of values by at most 2 w * mean(|v - out|) <= 2 w * spread, spread the largest |v - out|.  The sums over tokens add
  2^-23 * (tokens / 16 + 8) * (|v| + 15 s) in the worst case; one rounding to the output type ends it."""
import ctypes as C
import math

import numpy as np
import pytest

import infer_b200 as B
from tests import kv4_plain as P

pytestmark = pytest.mark.gpu
KINDS = {"bf16": B.BF16, "fp16": B.FP16, "fp32": B.FP32}


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def same(a, b):
    """Equal to the bit; how many bytes differ otherwise, and where the first one is."""
    import torch
    x, y = a.reshape(-1).contiguous(), b.reshape(-1).contiguous()
    if x.is_floating_point():  # which of the NaNs is not said
        assert torch.equal(x.isnan(), y.isnan())
        x, y = torch.where(x.isnan(), 0, x), torch.where(y.isnan(), 0, y)
    x, y = x.view(torch.uint8), y.view(torch.uint8)
    differ = (x != y).nonzero()
    assert differ.numel() == 0, f"{differ.numel()} of {x.numel()} bytes differ, first at {int(differ[0])} of shape {tuple(a.shape)}: {int(x[differ[0]])} {int(y[differ[0]])}"


def half_step(torch, dtype):
    return torch.finfo(dtype).eps / 2


def make_rope(torch, dtype, tokens, hq, hk, dim, rotary, layout, scaling, positions, seed=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = dtype_of(torch, dtype)
    rows = lambda h: torch.randn((tokens, h * dim + pad), generator=gen, device="cuda").to(dt)  # noqa: E731
    q, k = rows(hq), rows(hk)
    host, amplitude = B.rope_turns(rotary, **scaling)
    turns = torch.from_numpy(host).cuda()
    return q, k, turns, amplitude


SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=3.0),
            dict(scaling="yarn", factor=8.0, original=4096, fast=32.0, slow=1.0),
            dict(scaling="banded", factor=8.0, original=8192, fast=4.0, slow=1.0)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,layout,pad", [
    (1, 1, 1, 64, 64, "half", 0), (7, 8, 2, 128, 128, "half", 0), (33, 5, 1, 256, 64, "interleaved", 0), (3, 2, 2, 96, 24, "half", 0),
    (130, 4, 4, 80, 10, "interleaved", 0), (5, 3, 0, 128, 32, "half", 8), (700, 32, 8, 128, 128, "interleaved", 3), (2, 0, 3, 2, 2, "half", 0)])
@pytest.mark.parametrize("scaling", [0, 3])
def test_rope(cuda, dtype, tokens, hq, hk, dim, rotary, layout, pad, scaling):
    torch = cuda
    dt = dtype_of(torch, dtype)
    q, k, turns, amplitude = make_rope(torch, dtype, tokens, hq, hk, dim, rotary, layout, SCALINGS[scaling], None, seed=tokens, pad=pad)
    gen = torch.Generator(device="cuda").manual_seed(5)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    if tokens > 4:
        positions[3] = -1
    outs = [torch.full_like(x, 7.0) for x in (q, k)]
    d = B.rope_desc(dtype=KINDS[dtype], layout=B.ROPE_HALF if layout == "half" else B.ROPE_INTERLEAVED, tokens=tokens, head_dim=dim,
                    rotary_dim=rotary, positions=positions, turns=turns, amplitude=amplitude,
                    q=q if hq else None, q_out=outs[0] if hq else None, q_heads=hq, ldq=hq * dim + pad if hq else 0, ldq_out=hq * dim + pad if hq else 0,
                    k=k if hk else None, k_out=outs[1] if hk else None, k_heads=hk, ldk=hk * dim + pad if hk else 0, ldk_out=hk * dim + pad if hk else 0)
    B.rope(d)
    table, amp = P.turns(rotary, **SCALINGS[scaling])
    for x, y, heads in ((q, outs[0], hq), (k, outs[1], hk)):
        if not heads:
            continue
        body = x[:, :heads * dim].reshape(tokens, heads, dim)
        want, size = P.rope(torch, body, positions, torch.from_numpy(table).cuda(), amp, layout)
        got = y[:, :heads * dim].reshape(tokens, heads, dim)
        keep = positions >= 0
        limit = 2.0 ** -21 * size + half_step(torch, dt) * want.abs() + torch.finfo(dt).smallest_normal * half_step(torch, dt)
        limit = limit * (1 + 2.0 ** -8)
        bad = (got.double() - want).abs() > limit
        assert not bad[keep].any(), (got.double() - want).abs()[keep].max()
        assert (got[~keep] == 7.0).all() and (y[:, heads * dim:] == 7.0).all()
        assert torch.equal(got[keep][..., rotary:], body[keep][..., rotary:])
        # in place gives the same bits
    if hq and hk:
        qi, ki = q.clone(), k.clone()
        d2 = B.rope_desc(dtype=KINDS[dtype], layout=d.layout, tokens=tokens, head_dim=dim, rotary_dim=rotary, positions=positions, turns=turns,
                         amplitude=amplitude, q=qi, q_out=qi, q_heads=hq, ldq=hq * dim + pad, ldq_out=hq * dim + pad, k=ki, k_out=ki, k_heads=hk,
                         ldk=hk * dim + pad, ldk_out=hk * dim + pad)
        B.rope(d2)
        keep = positions >= 0
        assert torch.equal(qi[keep][:, :hq * dim], outs[0][keep][:, :hq * dim]) and torch.equal(ki[keep][:, :hk * dim], outs[1][keep][:, :hk * dim])
    assert B.last_variant() == "rope" and B.device_status() == 0


# ---- tables -------------------------------------------------------------------------------------------------------------
class Tables:
    def __init__(self, torch, cached, new, bs, capacity, spare=3, width=None, seed=0, short=0):
        rng = np.random.default_rng(seed)
        self.n, self.bs = len(cached), bs
        held = [P.blocks(c, bs) for c in cached]
        need = [P.blocks(c + x, bs) for c, x in zip(cached, new)]
        fresh = sum(need) - sum(held)
        self.blocks = sum(need) + spare
        self.width = width or max(max(need), 1)
        ids = rng.permutation(self.blocks).astype(np.int32)
        table = np.full((self.n, self.width), -1, np.int32)
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = ids[at:at + h]
            at += h
        free = np.zeros(self.blocks, np.int32)
        count = fresh + spare - short
        free[:count] = ids[at:at + count]
        i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")  # noqa: E731
        self.cached, self.new, self.table, self.free, self.count = i32(cached), i32(new), i32(table), i32(free), i32([count])
        self.status, self.total, self.starts = i32([0, 0]), i32([9] * self.n), i32([9] * (self.n + 1))
        self.slots, self.positions = i32([9] * (capacity + 2)), i32([9] * (capacity + 2))
        self.capacity = capacity
        self.host = (list(cached), list(new), table.copy(), free.copy(), count)

    def assign(self, in_place=False):
        self.count_out = self.count if in_place else self.count.clone() * 0
        self.total_out = self.cached if in_place else self.total
        return B.kv4_assign_desc(requests=self.n, max_blocks=self.width, block_size=self.bs, blocks=self.blocks, tokens=self.capacity,
                                 cached_lens=self.cached, new_lens=self.new, free_blocks=self.free, free_count=self.count,
                                 free_count_out=self.count_out, block_table=self.table, total_lens=self.total_out, query_start=self.starts,
                                 slots=self.slots, positions=self.positions, status=self.status)


@pytest.mark.parametrize("n,cached,new,bs", [(1, 0, 1, 16), (1, 15, 1, 16), (1, 16, 1, 16), (3, 100, 40, 32), (64, 3000, 1, 16), (1, 0, 5000, 64),
                                             (1024, 70, 9, 128), (1025, 300, 30, 16), (2500, 40, 20, 256)])
@pytest.mark.parametrize("in_place", [False, True])
def test_assign_and_release(cuda, n, cached, new, bs, in_place):
    torch = cuda
    rng = np.random.default_rng(n + cached)
    c = [cached] if n == 1 else rng.integers(0, cached + 1, n).tolist()
    x = [new] if n == 1 else rng.integers(0, new + 1, n).tolist()
    t = Tables(torch, c, x, bs, sum(x) + 3, seed=n)
    want = P.assign(*t.host, bs, t.capacity)
    d = t.assign(in_place)
    B.kv4_assign(d)
    got = dict(table=t.table, total=t.total_out, starts=t.starts, slots=t.slots, positions=t.positions, count=t.count_out)
    host = {name: v.cpu().numpy() for name, v in got.items()}
    assert host["slots"][t.capacity:].tolist() == [9, 9] and host["positions"][t.capacity:].tolist() == [9, 9], "write behind the rows"
    for name, w in want.items():
        h = host[name][:t.capacity] if name in ("slots", "positions") else host[name].reshape(np.asarray(w).shape)
        assert np.array_equal(h, np.asarray(w)), name
    assert t.status.cpu().tolist() == [0, 0]
    # everything back: the stack is as it was
    free0 = t.host[3]
    keep = torch.tensor(c, dtype=torch.int32, device="cuda")
    lens_out = t.total_out if in_place else torch.empty_like(t.total_out)
    count2 = t.count_out if in_place else torch.empty_like(t.count_out)
    scratch = t.free.clone()
    scratch[int(host["count"][0]):] = -5
    r = B.kv4_release_desc(requests=n, max_blocks=t.width, block_size=bs, blocks=t.blocks, lens=t.total_out, keep_lens=keep, free_blocks=scratch,
                           free_count=t.count_out, free_count_out=count2, block_table=t.table, lens_out=lens_out, status=t.status)
    B.kv4_release(r)
    assert int(count2[0]) == t.host[4] and t.status.cpu().tolist() == [0, 0]
    assert np.array_equal(scratch.cpu().numpy()[:t.host[4]], free0[:t.host[4]])
    assert lens_out.cpu().tolist() == c


@pytest.mark.parametrize("case,code", [("blocks", B.KV4_NO_BLOCKS), ("width", B.KV4_TABLE_FULL), ("rows", B.KV4_TOO_MANY_TOKENS), ("length", B.KV4_BAD_LENGTH),
                                       ("negative", B.KV4_BAD_LENGTH)])
def test_assign_refuses_as_a_whole(cuda, case, code):
    torch = cuda
    c, x = [20, 0, 33], [30, 5, 40]
    t = Tables(torch, c, x, 16, 75, spare=0, short=1 if case == "blocks" else 0)
    d = t.assign()
    if case == "width":
        d.max_blocks = t.width - 1
    if case == "rows":
        d.tokens = 74
    if case == "length":
        t.new[1] = -1
    if case == "negative":
        t.cached[1] = -4
    before = t.table.clone()
    B.kv4_assign(d)
    assert t.status.cpu().tolist() == [code, 0]
    assert torch.equal(t.table, before) and int(t.count_out[0]) == int(t.count[0])
    assert t.starts.cpu().tolist() == [0] * 4 and t.total.cpu().tolist() == [20, 0, 33]
    assert (t.slots[:74] == -1).all() and (t.positions[:74] == -1).all()


def test_release_refuses_as_a_whole(cuda):
    torch = cuda
    t = Tables(torch, [20, 0, 33], [30, 5, 40], 16, 75, spare=2)
    B.kv4_assign(t.assign())
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for keep, count, width, code in (([51, 0, 0], None, None, B.KV4_BAD_LENGTH), ([0, -1, 0], None, None, B.KV4_BAD_LENGTH),
                                     ([0, 0, 0], t.blocks, None, B.KV4_NO_BLOCKS), ([0, 0, 0], None, t.width - 1, B.KV4_TABLE_FULL)):
        free, out, lens = t.free.clone(), i32([0]), i32([0, 0, 0])
        have = t.count_out if count is None else i32([count])
        B.kv4_release(B.kv4_release_desc(requests=3, max_blocks=width or t.width, block_size=16, blocks=t.blocks, lens=t.total, keep_lens=i32(keep),
                                         free_blocks=free, free_count=have, free_count_out=out, block_table=t.table, lens_out=lens, status=t.status))
        assert t.status.cpu().tolist() == [code, 0] and torch.equal(free, t.free) and int(out[0]) == int(have[0])
        assert lens.cpu().tolist() == t.total.cpu().tolist()


# ---- cache --------------------------------------------------------------------------------------------------------------
def special_vectors(torch, tokens, heads, dim, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    x[0] = 0.0
    if tokens > 6:
        x[1] = 3.25                                   # constant
        x[2] = torch.arange(dim, device="cuda") % 16  # on and between the codes
        x[3] = (torch.arange(dim, device="cuda") % 31) * 0.5  # halves: ties
        x[4] *= 1e-30 if dtype != torch.float16 else 1e-6
        x[5] = x[5] * 1e-3 + 100.0
        x[6, :, 0] = -6e4
    return x.to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,heads,dim,bs", [(1, 1, 64, 16), (37, 3, 128, 16), (300, 2, 256, 64), (65, 8, 64, 256)])
def test_append_and_gather(cuda, dtype, tokens, heads, dim, bs):
    torch = cuda
    dt = dtype_of(torch, dtype)
    blocks = P.blocks(tokens, bs) + 3
    cache = P.new_cache(torch, blocks, heads, bs, dim, seed=1)
    before = {n: t.clone() for n, t in cache.items()}
    k, v = special_vectors(torch, tokens, heads, dim, dt, 2), special_vectors(torch, tokens, heads, dim, dt, 3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:tokens].to(torch.int32)
    if tokens > 20:
        slots[17] = -1
        k[9, 0, 1], v[10, heads - 1, dim - 1], k[11, 0, 0] = math.nan, math.inf, -math.inf
    b = P.bind(B, cache, bs)
    ldk = heads * dim + 5
    wide = torch.zeros((tokens, ldk), dtype=dt, device="cuda")
    wide[:, :heads * dim] = k.reshape(tokens, -1)
    for kk, ld in ((k, 0), (wide, ldk)):  # dense and vector loads; a stride that allows none
        for n in cache:
            cache[n].copy_(before[n])
        B.kv4_append(B.kv4_append_desc(cache=b, dtype=KINDS[dtype], tokens=tokens, k=kk, v=v, slots=slots, ldk=ld))
        want = P.append(torch, {n: t.clone() for n, t in before.items()}, bs, k, v, slots)
        for n in cache:
            same(cache[n], want[n])
    assert B.last_variant() == "kv4_append"
    kb, vb = torch.full((tokens, heads, dim), 7.0, dtype=dt, device="cuda"), torch.full((tokens, heads, dim), 7.0, dtype=dt, device="cuda")
    B.kv4_gather(B.kv4_gather_desc(cache=b, dtype=KINDS[dtype], tokens=tokens, slots=slots, k_out=kb, v_out=vb))
    keep = slots >= 0
    for got, (mean, size) in zip((kb, vb), P.read(torch, cache, bs, slots.clamp(min=0).long())):
        mean, size = mean[keep], size[keep]
        g = got[keep].double()
        nan = mean.isnan()
        assert torch.equal(g.isnan(), nan)
        limit = 2.0 ** -23 * size + half_step(torch, dt) * mean.abs() * (1 + 2.0 ** -8) + torch.finfo(dt).smallest_normal * half_step(torch, dt)
        assert ((g - mean).abs() <= limit)[~nan].all()
        assert (got[~keep] == 7.0).all()
    only = torch.empty_like(vb)
    B.kv4_gather(B.kv4_gather_desc(cache=b, dtype=KINDS[dtype], tokens=tokens, slots=slots, v_out=only))
    same(only[keep], vb[keep])
    assert B.device_status() == 0


def test_slots_beyond_the_cache_are_skipped_and_reported(cuda):
    torch = cuda
    cache = P.new_cache(torch, 2, 1, 16, 64, seed=1)
    before = {n: t.clone() for n, t in cache.items()}
    b = P.bind(B, cache, 16)
    k = torch.randn((3, 1, 64), device="cuda", dtype=torch.bfloat16)
    slots = torch.tensor([32, 1 << 30, 5], dtype=torch.int32, device="cuda")
    B.kv4_append(B.kv4_append_desc(cache=b, dtype=B.BF16, tokens=3, k=k, v=k, slots=slots))
    want = P.append(torch, before, 16, k[2:], k[2:], slots[2:])
    for n in cache:
        same(cache[n], want[n])
    assert B.device_status() >> 16 == 40
    out = torch.full_like(k, 3.0)
    B.kv4_gather(B.kv4_gather_desc(cache=b, dtype=B.BF16, tokens=3, slots=slots, k_out=out))
    assert (out[:2] == 3.0).all() and not (out[2] == 3.0).all()
    assert B.device_status() >> 16 == 41


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,layout", [(1, 4, 1, 128, 128, "half"), (70, 8, 2, 64, 32, "interleaved"), (900, 4, 4, 128, 128, "half"),
                                                            (5, 0, 2, 256, 24, "half"), (9, 3, 1, 64, 6, "interleaved")])
def test_rope_in_the_append_launch(cuda, dtype, tokens, hq, hk, dim, rotary, layout):
    """The bytes of fth_b200_rope followed by fth_b200_kv4_append."""
    torch = cuda
    dt, bs = dtype_of(torch, dtype), 16
    q, k, turns, amplitude = make_rope(torch, dtype, tokens, hq, hk, dim, rotary, layout, SCALINGS[3], None, seed=tokens)
    v = torch.randn((tokens, hk, dim), device="cuda").to(dt)
    positions = torch.arange(1000, 1000 + tokens, device="cuda", dtype=torch.int32)
    slots = torch.randperm((P.blocks(tokens, bs) + 1) * bs, device="cuda")[:tokens].to(torch.int32)
    if tokens > 4:
        positions[4], slots[4] = -1, -1
    common = dict(dtype=KINDS[dtype], layout=B.ROPE_HALF if layout == "half" else B.ROPE_INTERLEAVED, tokens=tokens, head_dim=dim, rotary_dim=rotary,
                  positions=positions, turns=turns, amplitude=amplitude, q_heads=hq, k_heads=hk, q=q if hq else None, k=k)
    one, two = (P.new_cache(torch, P.blocks(tokens, bs) + 1, hk, bs, dim, seed=1) for _ in range(2))
    qa, qb, kr = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.zeros_like(k)
    B.rope(B.rope_desc(q_out=qa if hq else None, k_out=kr, **common))
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, one, bs), dtype=KINDS[dtype], tokens=tokens, k=kr, v=v, slots=slots))
    fused = B.rope_desc(q_out=qb if hq else None, **common)
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, two, bs), dtype=KINDS[dtype], tokens=tokens, k=k, v=v, slots=slots, rope=fused))
    assert B.last_variant() == "rope_kv4_append"
    for n in one:
        same(one[n], two[n])
    same(qa, qb)
    assert B.device_status() == 0


def key_rounding(dtype, rows):
    return 2.0 ** -12 if dtype == "bf16" and rows > 128 else 0.0


# ---- attention ----------------------------------------------------------------------------------------------------------
def attend(torch, *, dtype, lens, new, hq, hk, dim, bs, window=0, causal=True, seed=0, q_gain=1.0, v_gain=None, lse=True, starts=True, guard=2, scale=None,
           mutate=None, pad=0, max_query=None):
    """Runs one call and checks it; returns the inputs for more."""
    dt = dtype_of(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    requests, rows = len(lens), sum(new)
    need = [P.blocks(n, bs) for n in lens]
    width = max(max(need), 1)
    blocks = sum(need) + 2
    ids = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    cache = P.new_cache(torch, blocks, hk, bs, dim, seed=seed + 1)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at:at + n]
        at += n
        if lens[r]:
            kv = torch.randn((2, lens[r], hk, dim), generator=gen, device="cuda")
            if v_gain is not None:
                kv[1] *= v_gain(torch, lens[r])[:, None, None]
            pos = torch.arange(lens[r], device="cuda")
            P.append(torch, cache, bs, kv[0].to(dt), kv[1].to(dt), (table[r, pos // bs].long() * bs + pos % bs).to(torch.int32))
    q = (torch.randn((rows + guard, hq * dim + pad), generator=gen, device="cuda") * q_gain).to(dt)
    start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    stat = torch.full((rows + guard, hq), 7.0, device="cuda")
    if mutate:
        mutate(cache=cache, table=table, q=q, length=length, start=start)
    d = B.kv4_attention_desc(cache=P.bind(B, cache, bs), dtype=KINDS[dtype], requests=requests, tokens=rows + (guard if starts else 0), q_heads=hq, q=q, out=out,
                             ldq=hq * dim + pad, ldo=hq * dim + pad, block_table=table, max_blocks=width, total_lens=length,
                             query_start=start if starts else None, max_query=max_query or (max(max(new), 1) if starts else 1),
                             scale=scale if scale is not None else dim ** -0.5, causal=causal, window=window, lse=stat if lse else None)
    ws = B.kv4_attention_workspace(torch, d)
    B.kv4_attention(d)
    first = out.clone()
    if lse:
        stat1 = stat.clone()
    B.kv4_attention(d)  # the workspace is ready again, and the result is the same to the bit
    same(out, first)
    if lse:
        same(stat, stat1)
    assert (out[rows:] == 7.0).all() and (out[:, hq * dim:] == 7.0).all() and (stat[rows:] == 7.0).all(), "rows behind the last were written"
    assert not ws[:4096].any(), "arrival counters are not back at zero"
    got = out[:rows, :hq * dim].reshape(rows, hq, dim).double()
    want, want_lse, limit, limit_lse = P.attention(torch, cache, bs, table, q[:rows, :hq * dim].reshape(rows, hq, dim), lens, new, hk,
                                                   d.scale, causal, window, key_rounding=key_rounding(dtype, d.max_query * hq // hk))
    step = half_step(torch, dt)
    limit = limit + step * want.abs() + torch.finfo(dt).smallest_normal * step
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    worst = ((got - want).abs() / limit)[~nan]
    if worst.numel():
        print(f"attention {dtype} lens {lens[:4]} new {new[:4]} heads {hq}/{hk} dim {dim}: worst {float(worst.max()):.3f} of the limit")
        assert worst.max() <= 1.0
    if lse:
        g = stat[:rows].double()
        empty = want_lse == -math.inf
        assert torch.equal(g == -math.inf, empty)
        good = ~(empty | want_lse.isnan())
        assert ((g - want_lse).abs() <= limit_lse)[good].all()
    assert B.device_status() == 0
    return dict(desc=d, q=q, out=out, cache=cache, table=table, length=length, ws=ws, start=start, lse=stat)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new,hq,hk,bs", [
    ([1], [1], 1, 1, 16), ([333], [1], 8, 2, 16), ([17, 128, 129, 1000], [1, 1, 1, 1], 5, 5, 16), ([700, 1, 64], [1, 1, 1], 16, 1, 64),
    ([4000], [1], 14, 2, 32), ([50] * 140, [1] * 140, 4, 4, 16), ([300, 40, 999], [5, 1, 3], 8, 2, 128), ([260, 31], [9, 0], 12, 4, 256)])
def test_attention_of_few_rows(cuda, dtype, dim, lens, new, hq, hk, bs):
    attend(cuda, dtype=dtype, lens=lens, new=new, hq=hq, hk=hk, dim=dim, bs=bs, seed=len(lens) + dim)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new,hq,hk,bs", [([200], [200], 4, 4, 16), ([700, 33, 129], [513, 33, 128], 8, 2, 64), ([1000], [70], 7, 1, 32),
                                               ([90, 0, 300], [64, 0, 299], 16, 1, 128), ([2500], [40], 16, 2, 64)])
def test_attention_of_many_rows(cuda, dtype, dim, lens, new, hq, hk, bs):
    attend(cuda, dtype=dtype, lens=lens, new=new, hq=hq, hk=hk, dim=dim, bs=bs, seed=len(lens) + dim)


@pytest.mark.parametrize("window,causal", [(1, True), (16, True), (100, True), (5000, True), (0, False), (37, False)])
@pytest.mark.parametrize("lens,new", [([400, 129, 3], [1, 1, 1]), ([400, 129, 3], [200, 100, 3]), ([900], [6])])
def test_windows_and_no_mask(cuda, window, causal, lens, new):
    for dim in (64, 128):
        attend(cuda, dtype="fp16", lens=lens, new=new, hq=4, hk=2, dim=dim, bs=16, window=window, causal=causal, seed=3)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 2, 70]])
def test_rows_that_see_nothing(cuda, new):
    """More rows than tokens, and requests without tokens: zeros and -infinity."""
    r = attend(cuda, dtype="bf16", lens=[0, 1, 50], new=new, hq=8, hk=2, dim=128, bs=16, seed=6)
    assert (r["out"][:new[0], :] == 0).all() and (r["lse"][:new[0]] == -math.inf).all()


@pytest.mark.parametrize("new", [1, 90])
def test_one_row_each_without_row_offsets_and_strided_rows(cuda, new):
    if new == 1:
        attend(cuda, dtype="bf16", lens=[70, 300, 5], new=[1, 1, 1], hq=8, hk=2, dim=128, bs=16, seed=8, starts=False, guard=0)
    attend(cuda, dtype="bf16", lens=[170, 300, 95], new=[new] * 3, hq=8, hk=2, dim=128, bs=16, seed=8, pad=9)
    attend(cuda, dtype="fp16", lens=[170, 300, 95], new=[new] * 3, hq=8, hk=2, dim=64, bs=16, seed=8, pad=8)


@pytest.mark.parametrize("new", [1, 90])
def test_long_requests_are_split_and_joined(cuda, new):
    attend(cuda, dtype="bf16", lens=[40000, 3, 1500], new=[new, 1, 1], hq=8, hk=1, dim=128, bs=64, seed=9)


@pytest.mark.parametrize("new", [1, 64])
@pytest.mark.parametrize("gain", [1e-20, 1e-4, 30.0, 1e4])
def test_sizes_of_queries(cuda, new, gain):
    """Tiny queries (all tokens weigh alike) and huge ones (one token wins)."""
    if gain == 1e-20:
        attend(cuda, dtype="bf16", lens=[500], new=[new], hq=4, hk=1, dim=128, bs=16, q_gain=gain)
    else:
        attend(cuda, dtype="fp16", lens=[500], new=[new], hq=4, hk=1, dim=128, bs=16, q_gain=gain, scale=1.0 if gain < 100 else 1e-4)
    attend(cuda, dtype="bf16", lens=[500], new=[new], hq=4, hk=1, dim=64, bs=16, scale=-0.125)


@pytest.mark.parametrize("new", [1, 64])
def test_values_of_very_different_sizes(cuda, new):
    attend(cuda, dtype="bf16", lens=[700], new=[new], hq=4, hk=1, dim=128, bs=16,
           v_gain=lambda torch, n: torch.exp2(torch.arange(n, device="cuda") % 9 * 2.0 - 8.0))
    attend(cuda, dtype="bf16", lens=[700], new=[new], hq=4, hk=1, dim=128, bs=16, v_gain=lambda torch, n: (torch.arange(n, device="cuda") % 2).float())
    attend(cuda, dtype="bf16", lens=[700], new=[new], hq=4, hk=1, dim=128, bs=16, v_gain=lambda torch, n: torch.zeros(n, device="cuda"))


@pytest.mark.parametrize("new", [1, 64])
def test_numbers_that_are_none(cuda, new):
    """A NaN in a query spoils its row, a NaN key or value the rows that see it, one behind the mask nothing."""
    torch = cuda

    def nan_query(q, **_):
        q[0, 5] = math.nan

    def nan_token(cache, table, **_):
        slot = int(table[0, 4]) * 16
        cache["k_params"][slot // 16, 0, 3, 0] = math.nan
    attend(cuda, dtype="bf16", lens=[100, 200], new=[new, new], hq=4, hk=2, dim=128, bs=16, mutate=nan_query)
    attend(cuda, dtype="bf16", lens=[100, 200], new=[new, new], hq=4, hk=2, dim=128, bs=16, mutate=nan_token)
    attend(cuda, dtype="bf16", lens=[100, 200], new=[new, new], hq=4, hk=2, dim=128, bs=16, mutate=nan_token, window=20)


@pytest.mark.parametrize("new", [1, 64])
def test_block_numbers_outside_the_cache_hide_their_tokens(cuda, new):
    torch = cuda
    r = attend(cuda, dtype="bf16", lens=[200], new=[new], hq=4, hk=2, dim=128, bs=16)
    table = r["table"].clone()
    for bad in (-1, 1 << 30, int(r["cache"]["k_codes"].shape[0])):
        r["table"][0, 2] = bad
        B.kv4_attention(r["desc"])
        assert B.device_status() >> 16 == 42
        got = r["out"][:new].reshape(new, 4, 128).double()
        want, _, limit, _ = P.attention(torch, r["cache"], 16, table, r["q"][:new].reshape(new, 4, 128), [200], [new], 2, 128 ** -0.5, True, 0, hidden=range(32, 48), key_rounding=key_rounding("bf16", 2 * new))
        assert ((got - want).abs() <= limit + 2.0 ** -8 * want.abs() + 1e-30).all()
        r["table"].copy_(table)


def test_lengths_change_under_a_captured_step(cuda):
    """assign -> rope + append -> attention, captured once and replayed as the requests grow; a second graph shares the
    workspace; every step is compared with the plain one."""
    torch = cuda
    n, hq, hk, dim, bs, width = 3, 8, 2, 128, 16, 40
    blocks = n * width
    cache = P.new_cache(torch, blocks, hk, bs, dim, seed=1)
    mirror = {k: t.clone() for k, t in cache.items()}
    b = P.bind(B, cache, bs)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, new = i32([0] * n), i32([0] * n)
    free, count, status = torch.randperm(blocks, device="cuda").to(torch.int32), i32([blocks]), i32([0, 0])
    table, starts = i32([[-1] * width] * n), i32([0] * (n + 1))
    capacity = 64
    slots, positions = i32([0] * capacity), i32([0] * capacity)
    host, amplitude = B.rope_turns(dim)
    turns = torch.from_numpy(host).cuda()
    dt = torch.bfloat16
    q, k, v = (torch.zeros((capacity, h, dim), dtype=dt, device="cuda") for h in (hq, hk, hk))
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    assign = B.kv4_assign_desc(requests=n, max_blocks=width, block_size=bs, blocks=blocks, tokens=capacity, cached_lens=lens, new_lens=new, free_blocks=free,
                               free_count=count, free_count_out=count, block_table=table, total_lens=lens, query_start=starts, slots=slots,
                               positions=positions, status=status)
    turn = B.rope_desc(dtype=B.BF16, layout=B.ROPE_HALF, tokens=capacity, head_dim=dim, rotary_dim=dim, positions=positions, turns=turns, amplitude=amplitude,
                       q=q, q_out=qr, q_heads=hq, k=k, k_heads=hk)
    append = B.kv4_append_desc(cache=b, dtype=B.BF16, tokens=capacity, k=k, v=v, slots=slots, rope=turn)
    descs = [B.kv4_attention_desc(cache=b, dtype=B.BF16, requests=n, tokens=capacity, q_heads=hq, q=qr, out=o, block_table=table, max_blocks=width,
                                  total_lens=lens, query_start=starts, max_query=capacity, scale=dim ** -0.5) for o in (out, torch.zeros_like(out))]
    ws = B.kv4_attention_workspace(torch, descs[0])
    descs[1].workspace, descs[1].workspace_bytes = descs[0].workspace, descs[0].workspace_bytes

    def step(d):
        B.kv4_assign(assign)
        B.kv4_append(append)
        B.kv4_attention(d)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(side):
        step(descs[0])  # new = 0: looks things up outside the capture
        torch.cuda.synchronize()
        for d in descs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                step(d)
            graphs.append(g)
    have = [0] * n
    for i, grow in enumerate([[30, 1, 5], [1, 1, 1], [1, 0, 1], [2, 33, 1], [1, 1, 1]]):
        new.copy_(i32(grow))
        rows = sum(grow)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda").to(dt))
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        have = [a + g for a, g in zip(have, grow)]
        assert status.cpu().tolist() == [0, 0] and lens.cpu().tolist() == have
        # the plain step: keys turned by the framework's own rope (tested above), everything else in 64 bits
        kr = torch.empty_like(k)
        qp = torch.empty_like(q)
        B.rope(B.rope_desc(dtype=B.BF16, layout=B.ROPE_HALF, tokens=capacity, head_dim=dim, rotary_dim=dim, positions=positions, turns=turns,
                           amplitude=amplitude, q=q, q_out=qp, q_heads=hq, k=k, k_out=kr, k_heads=hk))
        P.append(torch, mirror, bs, kr[:rows], v[:rows], slots[:rows])
        for name in cache:
            same(cache[name], mirror[name])
        want, _, limit, _ = P.attention(torch, mirror, bs, table, qp[:rows], have, grow, hk, dim ** -0.5, True, 0, key_rounding=key_rounding("bf16", 4 * capacity))
        got = (out if i % 2 == 0 else descs[1]._keep[2])[:rows].double()
        assert ((got - want).abs() <= limit + 2.0 ** -8 * want.abs() + 1e-30).all()
    del graphs, ws
    assert B.device_status() == 0


def test_a_cache_beyond_four_gigabytes(cuda):
    """Blocks at the far end of a cache whose codes pass 2^32 bytes."""
    torch = cuda
    hk, dim, bs = 8, 256, 256
    blocks = (1 << 32) // (hk * bs * dim // 2) + 40
    cache = P.new_cache(torch, blocks, hk, bs, dim, seed=None)
    b = P.bind(B, cache, bs)
    lens = [700]
    table = torch.tensor([[blocks - 1, 3, blocks - 7]], dtype=torch.int32, device="cuda")
    pos = torch.arange(700, device="cuda")
    slots = (table[0, pos // bs].long() * bs + pos % bs).to(torch.int32)
    k, v = (torch.randn((700, hk, dim), device="cuda").to(torch.bfloat16) for _ in range(2))
    B.kv4_append(B.kv4_append_desc(cache=b, dtype=B.BF16, tokens=700, k=k, v=v, slots=slots))
    kb = torch.empty_like(k)
    B.kv4_gather(B.kv4_gather_desc(cache=b, dtype=B.BF16, tokens=700, slots=slots, k_out=kb))
    assert float((kb.float() - k.float()).abs().max()) < 0.5 * float((k.float().amax(-1) - k.float().amin(-1)).max()) / 15 * 1.02 + 0.03
    for new in (1, 100):
        q = torch.randn((new, 16, dim), device="cuda").to(torch.bfloat16)
        out = torch.empty_like(q)
        d = B.kv4_attention_desc(cache=b, dtype=B.BF16, requests=1, tokens=new, q_heads=16, q=q, out=out, block_table=table, max_blocks=3,
                                 total_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=dim ** -0.5, max_query=new,
                                 query_start=torch.tensor([0, new], dtype=torch.int32, device="cuda"))
        B.kv4_attention_workspace(torch, d)
        B.kv4_attention(d)
        want, _, limit, _ = P.attention(torch, cache, bs, table, q, lens, [new], hk, dim ** -0.5, True, 0, key_rounding=key_rounding("bf16", 2 * new))
        assert ((out.double() - want).abs() <= limit + 2.0 ** -8 * want.abs()).all()
    assert B.device_status() == 0


def test_other_streams_and_two_calls_at_once(cuda):
    """Calls on two streams, each with a workspace of its own, at the same time."""
    torch = cuda
    runs = [attend(cuda, dtype="bf16", lens=[9000, 100 + i], new=[1, 1], hq=8, hk=2, dim=128, bs=16, seed=20 + i) for i in range(2)]
    want = [r["out"].clone() for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    for r in runs:
        r["out"].fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for r, s in zip(runs, streams):
            B.kv4_attention(r["desc"], stream=C.c_void_p(s.cuda_stream))
    torch.cuda.synchronize()
    for r, w in zip(runs, want):
        same(r["out"], w)
