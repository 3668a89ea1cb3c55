"""GPU: the 4-bit cache at sizes and in states beyond tests/test_gpu_kv4.py, with its helpers, plain forms and limits: many
requests, long shares of work, rows beyond max_query, numbers that are none in every place, many tokens stored at once."""
import math

import numpy as np
import pytest

import infer_b200 as B
from tests import kv4_plain as P
from tests.test_gpu_kv4 import KINDS, SCALINGS, attend, dtype_of, half_step, key_rounding, make_rope, same, special_vectors

pytestmark = pytest.mark.gpu


# ---- attention ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,hq,hk", [(1, 2, 2), (5, 4, 1), (40, 4, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_requests(cuda, new, hq, hk, dim):
    """More requests than a block has threads, some of them empty or idle, in both kernels."""
    rng = np.random.default_rng(dim + new)
    lens = [int(n) for n in rng.integers(0, 150, 700)]
    rows = [0 if rng.random() < 0.2 else int(rng.integers(1, new + 1)) for _ in lens]
    attend(cuda, dtype="bf16", lens=lens, new=rows, hq=hq, hk=hk, dim=dim, bs=16, seed=new)


@pytest.mark.parametrize("dtype,dim,hq,hk,window", [("bf16", 64, 8, 8, 0), ("fp16", 64, 8, 8, 0), ("bf16", 128, 6, 6, 9000), ("bf16", 256, 4, 4, 0)])
def test_long_shares_of_many_rows(cuda, dtype, dim, hq, hk, window):
    """Work enough that the cost of starting a unit moves the cuts; several requests, the last with few rows."""
    attend(cuda, dtype=dtype, lens=[14000, 5000, 900], new=[4100, 2300, 3], hq=hq, hk=hk, dim=dim, bs=64, seed=dim, window=window, lse=False)


@pytest.mark.parametrize("units", [1, 2, 3])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_units_of_every_length(cuda, units, dim):
    """Batches small enough that shares end with their unit, around the lengths where one more share begins."""
    for length in (1, 127, 128, 129, 255, 257, 511, 512, 513, 1024, 1025, 2049, 5000):
        lens = [max(length - 300 * r, 1) for r in range(units)]
        attend(cuda, dtype="bf16", lens=lens, new=[1] * units, hq=8, hk=2, dim=dim, bs=16, seed=length)


@pytest.mark.parametrize("new,most", [([5, 2, 7], 3), ([90, 10, 40], 33)])
def test_rows_beyond_max_query_are_not_computed(cuda, new, most):
    """The first max_query rows of a request keep their positions; the rest is left as it was."""
    torch = cuda
    hq, hk, dim, bs, lens = 8, 2, 128, 16, [300, 50, 129]
    r = attend(torch, dtype="bf16", lens=lens, new=new, hq=hq, hk=hk, dim=dim, bs=bs, seed=1)
    d = r["desc"]
    d.max_query = most
    ws = B.kv4_attention_workspace(torch, d)
    r["out"].fill_(7.0)
    B.kv4_attention(d)
    # a row of n stands at total - n + i: the first `most` of n rows are the last of total - (n - most) tokens
    at = 0
    for i, n in enumerate(new):
        kept = min(n, most)
        q = r["q"][at:at + kept].reshape(kept, hq, dim)
        want, _, limit, _ = P.attention(torch, r["cache"], bs, r["table"][i:i + 1], q, [lens[i] - (n - kept)], [kept], hk, d.scale, True, 0,
                                        key_rounding=key_rounding("bf16", most * hq // hk))
        got = r["out"][at:at + kept].reshape(kept, hq, dim).double()
        assert ((got - want).abs() <= limit + 2.0 ** -8 * want.abs() + 1e-30).all()
        assert (r["out"][at + kept:at + n] == 7.0).all()
        at += n
    del ws
    assert B.device_status() == 0


def near(torch, a, b, dtype):
    a, b = a.double(), b.double()
    assert not a.isnan().any() and b.abs().max() < 5
    assert ((a - b).abs() <= 2 * half_step(torch, dtype_of(torch, dtype)) * (b.abs() + 0.1) + 2 * 2 * 2.0 ** -12 * 10).all()


@pytest.mark.parametrize("name,which", [("k_params", 0), ("k_params", 1), ("v_params", 0), ("v_params", 1)])
@pytest.mark.parametrize("dtype,new", [("bf16", 1), ("bf16", 64), ("fp16", 64), ("bf16", 80), ("fp16", 80)])
def test_scales_and_minima_that_are_no_numbers(cuda, name, which, dtype, new):
    """The token's scale or minimum of keys or values: the rows that see it are NaN, the others (behind the mask or the window, of
    other heads and requests) are what they were up to the roundings, which depend on the rows worked on together: each result is
    within 2 * 2^-12 of |v| + |out| < 10 (a probability's rounding) and half a step of the exact one."""
    torch = cuda

    def spoil(cache, table, **_):
        for token in (60, 97):
            cache[name][int(table[0, token // 16]), 1, token % 16, which] = math.nan
    args = dict(dtype=dtype, lens=[100, 200], new=[new, new], hq=4, hk=2, dim=128, bs=16, seed=5, lse=False)
    for window in (0, 20):
        clean = attend(torch, window=window, **args)
        torch.cuda.synchronize()
        keep = clean["out"].clone()
        spoil(clean["cache"], clean["table"])
        B.kv4_attention(clean["desc"])
        rows = torch.arange(new, device="cuda") + 100 - new
        sees = torch.zeros(new, dtype=torch.bool, device="cuda")
        for token in (60, 97):
            sees |= (rows >= token) & ((rows - token < window) if window else True)
        got = clean["out"][:2 * new].view(-1, 4, 128)
        assert got[:new][sees][:, 2:].isnan().all()
        others = got.clone().view(torch.int16)
        others[:new, 2:][sees] = 0
        before = keep[:2 * new].view(-1, 4, 128).clone().view(torch.int16)
        before[:new, 2:][sees] = 0
        near(torch, others.view(keep.dtype), before.view(keep.dtype), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new", [2, 64, 80])
def test_an_infinity_in_one_row_leaves_the_others(cuda, dtype, new):
    torch = cuda
    r = attend(torch, dtype=dtype, lens=[300], new=[new], hq=4, hk=2, dim=128, bs=16, seed=4, lse=False)
    before = r["out"].clone()
    r["q"][new - 1, 7] = math.inf
    B.kv4_attention(r["desc"])
    got = r["out"].view(-1, 4, 128)
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[new - 1, 0] = False
    keep[new:] = False
    near(torch, got[keep], before.view(-1, 4, 128)[keep], dtype)
    assert got[new - 1, 0].isnan().all() and (r["out"][new:] == 7.0).all()


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("fp16", 128), ("bf16", 256)])
def test_hidden_blocks_of_many_rows(cuda, dtype, dim):
    """A block number outside the cache hides its tokens and is reported; also the first and the last block."""
    torch = cuda
    r = attend(torch, dtype=dtype, lens=[260], new=[80], hq=4, hk=2, dim=dim, bs=16)
    table = r["table"].clone()
    for column in (0, 7, 16):
        r["table"][0, column] = -1
        B.kv4_attention(r["desc"])
        assert B.device_status() >> 16 == 42
        got = r["out"][:80].reshape(80, 4, dim).double()
        want, _, limit, _ = P.attention(torch, r["cache"], 16, table, r["q"][:80].reshape(80, 4, dim), [260], [80], 2, dim ** -0.5, True, 0,
                                        hidden=range(column * 16, min(column * 16 + 16, 260)), key_rounding=key_rounding(dtype, 160))
        assert ((got - want).abs() <= limit + half_step(torch, dtype_of(torch, dtype)) * want.abs() + 1e-6 * (dtype == "fp16") + 1e-30).all()
        r["table"].copy_(table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,hq,hk", [(3, 8, 1), (5, 8, 2), (10, 4, 1), (12, 8, 2), (32, 8, 2), (33, 8, 2), (128, 1, 1), (129, 2, 2)])
def test_rows_in_blocks_of_eight_and_sixteen(cuda, dtype, dim, new, hq, hk):
    """17 .. 132 rows to a kv head: several units to a head, of which the first see less; cut and whole; few and many requests."""
    attend(cuda, dtype=dtype, lens=[1500, new, 40], new=[new, new, 1], hq=hq, hk=hk, dim=dim, bs=32, seed=new)
    attend(cuda, dtype=dtype, lens=[200 + 13 * i for i in range(60)], new=[new - i % 3 for i in range(60)], hq=hq, hk=hk, dim=dim, bs=16, seed=new, window=150)


def test_two_graphs_share_a_workspace(cuda):
    """Captured calls of both kernels on one workspace, replayed in any order, give the eager results."""
    torch = cuda
    few = attend(torch, dtype="bf16", lens=[5000, 90], new=[1, 1], hq=8, hk=2, dim=128, bs=16, seed=2)
    many = attend(torch, dtype="bf16", lens=[5000, 90], new=[70, 30], hq=8, hk=2, dim=128, bs=16, seed=3)
    ws = max((few["ws"], many["ws"]), key=lambda t: t.numel())
    graphs = []
    for r in (few, many):
        r["desc"].workspace, r["desc"].workspace_bytes = ws.data_ptr(), ws.numel()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            B.kv4_attention(r["desc"])
        graphs.append((g, r, r["out"].clone()))
    for i in (0, 1, 1, 0, 0, 1):
        g, r, want = graphs[i]
        r["out"].fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        want[-2:] = 7.0
        assert torch.equal(r["out"], want)
    assert B.device_status() == 0


# ---- storing and reading back -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,tokens,heads,dim,bs", [("bf16", 5001, 8, 64, 16), ("fp16", 2601, 8, 128, 64), ("fp32", 2600, 4, 256, 256)])
@pytest.mark.parametrize("order", ["row", "odd", "random", "holes"])
def test_many_tokens_at_once(cuda, dtype, tokens, heads, dim, bs, order):
    """Enough tokens that they are worked on in pairs: neighbours in the cache, neighbours across a block, strangers, gaps."""
    torch = cuda
    dt = dtype_of(torch, dtype)
    blocks = P.blocks(tokens, bs) + 2
    cache = P.new_cache(torch, blocks, heads, bs, dim, seed=1)
    want = {n: t.clone() for n, t in cache.items()}
    k, v = special_vectors(torch, tokens, heads, dim, dt, 2), special_vectors(torch, tokens, heads, dim, dt, 3)
    k[100, 0, 3], v[101, heads - 1, 0] = math.nan, -math.inf
    gen = torch.Generator(device="cuda").manual_seed(4)
    slots = torch.arange(tokens, device="cuda")
    if order == "odd":
        slots = slots + 1
    elif order == "random":
        slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:tokens]
    elif order == "holes":
        slots = torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.3, -1, slots)
    slots = slots.to(torch.int32)
    b = P.bind(B, cache, bs)
    B.kv4_append(B.kv4_append_desc(cache=b, dtype=KINDS[dtype], tokens=tokens, k=k, v=v, slots=slots))
    P.append(torch, want, bs, k, v, slots)
    for n in cache:
        same(cache[n], want[n])
    kb, vb = (torch.full((tokens, heads, dim), 7.0, dtype=dt, device="cuda") for _ in range(2))
    B.kv4_gather(B.kv4_gather_desc(cache=b, dtype=KINDS[dtype], tokens=tokens, slots=slots, k_out=kb, v_out=vb))
    keep = slots >= 0
    for got, (mean, size) in zip((kb, vb), P.read(torch, cache, bs, slots.clamp(min=0).long())):
        mean, size, g = mean[keep], size[keep], got[keep].double()
        nan = mean.isnan()
        assert torch.equal(g.isnan(), nan)
        limit = 2.0 ** -23 * size + half_step(torch, dt) * mean.abs() * (1 + 2.0 ** -8) + torch.finfo(dt).smallest_normal * half_step(torch, dt)
        assert ((g - mean).abs() <= limit)[~nan].all()
        assert (got[~keep] == 7.0).all()
    assert B.device_status() == 0


def test_ranges_at_the_end_of_the_numbers(cuda):
    """Differences that round up past the largest FP32 number, spreads below the smallest scale, signed zeros."""
    torch = cuda
    big = torch.finfo(torch.float32).max
    rows = [[-1.0, big], [-1e38, 2.4e38], [-big / 2, big / 2], [0.0, 1e-38], [0.0, 1e-44], [-0.0, 0.0], [-1e-40, 1e-40], [1e38, 1.5e38]]
    x = torch.zeros((len(rows), 1, 64), device="cuda")
    for i, (low, high) in enumerate(rows):
        x[i, 0] = torch.linspace(0, 1, 64, device="cuda") * 1e-3 * high
        x[i, 0, :20], x[i, 0, 40:] = low, high
    slots = torch.arange(len(rows), dtype=torch.int32, device="cuda")
    cache = P.new_cache(torch, 1, 1, 16, 64, seed=1)
    want = P.append(torch, {n: t.clone() for n, t in cache.items()}, 16, x, x, slots)
    # a range that leaves FP32 is stored with scale NaN, the codes and the minimum as zeros
    _, _, minimum = P.quantise(torch, x)
    beyond = (x.double().amax(-1) - minimum).float().isinf()[:, 0]
    assert beyond.any() and not beyond[0]
    for t in slots[beyond].tolist():
        want["k_codes"][0, :, t] = 0
        want["v_codes"].view(1, 1, 8, 16, 2, 2)[0, :, t // 2, :, t % 2] = 0
        for n in ("k_params", "v_params"):
            want[n][0, :, t, 0], want[n][0, :, t, 1] = math.nan, 0.0
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, cache, 16), dtype=B.FP32, tokens=len(rows), k=x, v=x, slots=slots))
    for n in cache:
        a, b = (t.float() + 0.0 if "params" in n else t for t in (cache[n], want[n]))   # -0 is 0
        same(a, b)
    assert B.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,layout", [(1301, 4, 2, 128, 128, "half"), (2500, 8, 2, 64, 32, "interleaved"), (4001, 0, 1, 256, 64, "half")])
def test_many_turned_tokens_at_once(cuda, dtype, tokens, hq, hk, dim, rotary, layout):
    """Blocks of several tokens, odd ones behind, rows without a slot: the bytes of the separate calls."""
    torch = cuda
    bs = 64
    q, k, turns, amplitude = make_rope(torch, dtype, tokens, hq, hk, dim, rotary, layout, SCALINGS[0], None, seed=tokens)
    v = torch.randn((tokens, hk, dim), device="cuda").to(k.dtype)
    positions = torch.arange(5, 5 + tokens, device="cuda", dtype=torch.int32)
    slots = torch.arange(1, 1 + tokens, device="cuda", dtype=torch.int32)
    slots[100], positions[100], slots[tokens - 2] = -1, -1, -1
    common = dict(dtype=KINDS[dtype], layout=B.ROPE_HALF if layout == "half" else B.ROPE_INTERLEAVED, tokens=tokens, head_dim=dim, rotary_dim=rotary,
                  positions=positions, turns=turns, amplitude=amplitude, q_heads=hq, k_heads=hk, q=q if hq else None, k=k)
    one, two = (P.new_cache(torch, P.blocks(tokens, bs) + 1, hk, bs, dim, seed=1) for _ in range(2))
    qa, qb, kr = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.zeros_like(k)
    B.rope(B.rope_desc(q_out=qa if hq else None, k_out=kr, **common))
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, one, bs), dtype=KINDS[dtype], tokens=tokens, k=kr, v=v, slots=slots))
    fused = B.rope_desc(q_out=qb if hq else None, **common)
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, two, bs), dtype=KINDS[dtype], tokens=tokens, k=k, v=v, slots=slots, rope=fused))
    for n in one:
        same(one[n], two[n])
    same(qa, qb)
    assert B.device_status() == 0


@pytest.mark.parametrize("requests,grow", [(200, 1), (256, 2), (257, 2), (300, 1), (1024, 3), (1025, 7), (2100, 5)])
def test_tables_of_every_block_size(cuda, requests, grow):
    """Few threads, many threads, several blocks, more requests than a block has threads: assign, then release, against the plain
    form; lengths in place."""
    torch = cuda
    rng = np.random.default_rng(requests)
    cached = [int(n) for n in rng.integers(0, 60, requests)]
    new = [int(n) for n in rng.integers(0, grow + 1, requests)]
    bs, width = 16, 6
    blocks = sum(P.blocks(c + n, bs) for c, n in zip(cached, new)) + 5
    order = rng.permutation(blocks)
    table = np.full((requests, width), -1, np.int32)
    at = 0
    for r, c in enumerate(cached):
        held = P.blocks(c, bs)
        table[r, :held] = order[at:at + held]
        at += held
    free = list(order[at:])
    capacity = sum(new) + 3
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    stack = np.zeros(blocks, np.int32)
    stack[:len(free)] = free
    lens, fresh, dtable, dfree, count = i32(cached), i32(new), i32(table), i32(stack), i32([len(free)])
    starts, slots, positions, status = i32([0] * (requests + 1)), i32([7] * capacity), i32([7] * capacity), i32([0, 0])
    B.kv4_assign(B.kv4_assign_desc(requests=requests, max_blocks=width, block_size=bs, blocks=blocks, tokens=capacity, cached_lens=lens, new_lens=fresh,
                                   free_blocks=dfree, free_count=count, free_count_out=count, block_table=dtable, total_lens=lens, query_start=starts,
                                   slots=slots, positions=positions, status=status))
    want_slots, want_positions, left = [], [], len(free)
    for r, (c, n) in enumerate(zip(cached, new)):
        for j in range(P.blocks(c, bs), P.blocks(c + n, bs)):
            left -= 1
            table[r, j] = free[left]
        want_positions += range(c, c + n)
        want_slots += [int(table[r, t // bs]) * bs + t % bs for t in range(c, c + n)]
    assert status.cpu().tolist() == [0, 0] and count.item() == left
    assert lens.cpu().tolist() == [c + n for c, n in zip(cached, new)]
    assert (dtable.cpu().numpy() == table).all() and starts.cpu().tolist() == [0] + np.cumsum(new).tolist()
    assert slots.cpu().tolist() == want_slots + [-1] * 3 and positions.cpu().tolist() == want_positions + [-1] * 3
    # half of the requests shrink, some to nothing
    keep = [int(rng.integers(0, n + 1)) if r % 2 else n for r, n in enumerate(lens.cpu().tolist())]
    now = lens.cpu().tolist()
    B.kv4_release(B.kv4_release_desc(requests=requests, max_blocks=width, block_size=bs, blocks=blocks, lens=lens, keep_lens=i32(keep), free_blocks=dfree,
                                     free_count=count, free_count_out=count, block_table=dtable, lens_out=lens, status=status))
    back = [int(table[r, j]) for r in range(requests) for j in range(P.blocks(keep[r], bs), P.blocks(now[r], bs))]
    assert status.cpu().tolist() == [0, 0] and count.item() == left + len(back) and lens.cpu().tolist() == keep
    assert dfree.cpu().tolist()[left:left + len(back)] == back[::-1] and dfree.cpu().tolist()[:left] == [int(f) for f in free[:left]]
