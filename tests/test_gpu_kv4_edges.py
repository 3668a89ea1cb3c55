"""GPU: calls of the 4-bit cache's operators that their documents allow and the other files do not make, with the helpers, plain
forms and limits of tests/test_gpu_kv4.py."""
import ctypes as C
import math

import numpy as np
import pytest

import infer_b200 as B
from tests import kv4_plain as P
from tests.test_gpu_kv4 import KINDS, SCALINGS, attend, dtype_of, half_step, key_rounding, make_rope, same

pytestmark = pytest.mark.gpu


# ---- a value's scale that is no number, beside rows that do not see it ----------------------------------------------------
def spoil_value(token, bs=16):
    def mutate(cache, table, **_):
        cache["v_params"][int(table[0, token // bs]), :, token % bs, 0] = math.nan
    return mutate


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("token,rows", [(31, 12), (31, 16), (30, 5), (33, 7), (0, 12)])
def test_rows_before_a_spoiled_value(cuda, dtype, token, rows):
    """64-wide heads, where a warp takes two groups of 32 tokens of a tile one after the other: the rows before the token keep
    what the first group gave them."""
    attend(cuda, dtype=dtype, lens=[40], new=[rows], hq=1, hk=1, dim=64, bs=16, seed=rows, mutate=spoil_value(token))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,hq", [(2, 1), (2, 4), (5, 2), (16, 1), (150, 1)])
def test_a_spoiled_value_that_only_the_oldest_row_sees(cuda, dtype, dim, rows, hq):
    length, window = 900, 300
    first = length - rows - window + 1   # of the tokens that the oldest row sees
    for token in (first, first + rows - 2):
        attend(cuda, dtype=dtype, lens=[length], new=[rows], hq=hq, hk=1, dim=dim, bs=16, seed=rows, window=window, mutate=spoil_value(token))


@pytest.mark.parametrize("dim,length,rows", [(64, 64, 4), (128, 160, 4), (256, 160, 4), (128, 160, 9), (64, 320, 140)])
def test_large_values_beside_a_spoiled_one(cuda, dim, length, rows):
    """The last 32 tokens' values are 2^14 times as large as the others and the last one is no number: rows that do not see it
    take the others at their size."""
    attend(cuda, dtype="bf16", lens=[length], new=[rows], hq=1, hk=1, dim=dim, bs=16, seed=rows, mutate=spoil_value(length - 1),
           v_gain=lambda torch, n: torch.where(torch.arange(n, device="cuda") >= n - 32, 2.0 ** 14, 1.0))


# ---- rows ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,tokens", [([5, 2, 7], 10), ([5, 2, 7], 6), ([5, 2, 7], 3), ([90, 10, 40], 120), ([90, 10, 40], 70)])
@pytest.mark.parametrize("window", [0, 60])
def test_rows_behind_tokens_are_left_and_the_others_keep_their_positions(cuda, new, tokens, window):
    """query_start goes beyond `tokens`: row i of n stands at total - n + i all the same."""
    torch = cuda
    hq, hk, dim, bs, lens = 8, 2, 128, 16, [300, 50, 129]
    r = attend(torch, dtype="bf16", lens=lens, new=new, hq=hq, hk=hk, dim=dim, bs=bs, seed=1, window=window)
    d = r["desc"]
    d.tokens = tokens
    r["out"].fill_(7.0)
    r["lse"].fill_(7.0)
    B.kv4_attention(d)
    at = 0
    for i, n in enumerate(new):
        kept = max(min(n, tokens - at), 0)
        if kept:
            q = r["q"][at:at + kept].reshape(kept, hq, dim)
            want, want_lse, limit, limit_lse = P.attention(torch, r["cache"], bs, r["table"][i:i + 1], q, [lens[i] - (n - kept)], [kept], hk, d.scale, True,
                                                           window, key_rounding=key_rounding("bf16", d.max_query * hq // hk))
            got = r["out"][at:at + kept].reshape(kept, hq, dim).double()
            assert ((got - want).abs() <= limit + 2.0 ** -8 * want.abs() + 1e-30).all()
            assert ((r["lse"][at:at + kept].double() - want_lse).abs() <= limit_lse).all()
        at += n
    assert (r["out"][tokens:] == 7.0).all() and (r["lse"][tokens:] == 7.0).all()
    assert B.device_status() == 0


# ---- workspaces ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_workspace_of_the_largest_step_serves_smaller_ones(cuda, dim):
    torch = cuda
    big = attend(torch, dtype="bf16", lens=[5000, 90], new=[20, 20], hq=2, hk=2, dim=dim, bs=16, seed=2)
    for rows in (16, 9, 1):
        r = attend(torch, dtype="bf16", lens=[5000, 90], new=[rows, 1], hq=2, hk=2, dim=dim, bs=16, seed=3)
        want = r["out"].clone()
        r["out"].fill_(7.0)
        r["desc"].workspace, r["desc"].workspace_bytes = big["ws"].data_ptr(), big["ws"].numel()
        B.kv4_attention(r["desc"])
        same(r["out"], want)
    assert B.device_status() == 0


# ---- tables -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("requests,width", [(3, 8), (250, 2), (300, 4), (1100, 6), (600, 300)])
@pytest.mark.parametrize("bad", [-1, "blocks", 1 << 30])
def test_release_refuses_a_table_entry_that_is_no_block(cuda, requests, width, bad):
    """One block of few threads, one of many, several blocks, more requests than a block has threads; the entry in the first, the
    last or a middle request, at the begin or the end of what comes back.  The stack keeps its blocks; an entry among the kept
    tokens is not looked at."""
    torch = cuda
    bs, held = 16, width - 1
    blocks = requests * width + 5
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    table[:, :held] = torch.randperm(requests * held, device="cuda").to(torch.int32).view(requests, held)
    good = table.clone()
    spare = blocks - requests * held
    lens, keep = i32([held * bs] * requests), i32([bs // 2] * requests)   # the first block stays
    keep[0] = 0
    status = i32([0, 0])

    def release():
        free = torch.full((blocks,), -7, dtype=torch.int32, device="cuda")
        free[:spare] = torch.arange(requests * held, blocks, device="cuda", dtype=torch.int32)
        count, now = i32([spare]), lens.clone()
        B.kv4_release(B.kv4_release_desc(requests=requests, max_blocks=width, block_size=bs, blocks=blocks, lens=now, keep_lens=keep, free_blocks=free,
                                         free_count=count, free_count_out=count, block_table=table, lens_out=now, status=status))
        return free, count, now
    start = torch.arange(requests * held, blocks, device="cuda", dtype=torch.int32)
    if held > 1:
        for r, j in ((0, 0), (requests - 1, held - 1), (requests // 2, 1)):
            table[r, j] = blocks if bad == "blocks" else bad
            free, count, now = release()
            assert status.cpu().tolist() == [B.KV4_BAD_BLOCK, 0]
            assert count.item() == spare and torch.equal(free[:spare], start) and torch.equal(now, lens)
            table.copy_(good)
    table[requests - 1, 0] = table[requests // 2, held] = -3   # held by the tokens that stay; behind the last token
    free, count, now = release()
    back = torch.cat([good[0, :held], good[1:, 1:held].reshape(-1)])
    assert status.cpu().tolist() == [0, 0] and count.item() == spare + back.numel() and torch.equal(now, keep)
    assert torch.equal(free[:spare], start) and torch.equal(free[spare:spare + back.numel()], back.flip(0))


# ---- storing ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,layout,rotary", [(6, "half", 128), (6, "interleaved", 48), (6, "half", 20), (1301, "half", 128)])
def test_a_negative_position_with_a_slot(cuda, dtype, tokens, layout, rotary):
    """The row is not turned: its key is stored as it is, as by fth_b200_rope in place and fth_b200_kv4_append; q is left."""
    torch = cuda
    hq, hk, dim, bs = 4, 2, 128, 16
    q, k, turns, amplitude = make_rope(torch, dtype, tokens, hq, hk, dim, rotary, layout, SCALINGS[3], None, seed=tokens)
    k[4] = k[4].abs() * (torch.arange(hk * dim, device="cuda") % 3).to(k.dtype) * -0.0   # zeros of both signs: a sign is a byte's too
    k[4, ::2] *= -1.0
    v = torch.randn((tokens, hk, dim), device="cuda").to(k.dtype)
    positions = torch.arange(100, 100 + tokens, device="cuda", dtype=torch.int32)
    positions[1], positions[4], positions[tokens - 1] = -1, -(1 << 31), -77
    slots = torch.arange(3, 3 + tokens, device="cuda", dtype=torch.int32)
    common = dict(dtype=KINDS[dtype], layout=B.ROPE_HALF if layout == "half" else B.ROPE_INTERLEAVED, tokens=tokens, head_dim=dim, rotary_dim=rotary,
                  positions=positions, turns=turns, amplitude=amplitude, q_heads=hq, k_heads=hk, q=q)
    one, two = (P.new_cache(torch, P.blocks(tokens, bs) + 1, hk, bs, dim, seed=1) for _ in range(2))
    qa, qb, kr = torch.full_like(q, 7.0), torch.full_like(q, 7.0), k.clone()
    B.rope(B.rope_desc(q_out=qa, k=kr, k_out=kr, **common))
    assert torch.equal(kr[1], k[1])
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, one, bs), dtype=KINDS[dtype], tokens=tokens, k=kr, v=v, slots=slots))
    B.kv4_append(B.kv4_append_desc(cache=P.bind(B, two, bs), dtype=KINDS[dtype], tokens=tokens, k=k, v=v, slots=slots,
                                   rope=B.rope_desc(q_out=qb, k=k, **common)))
    for n in one:
        same(one[n], two[n])
    same(qa, qb)
    assert (qa[1] == 7.0).all() and B.device_status() == 0


def test_the_status_of_a_bad_slot_is_no_wait_for_a_peer(cuda):
    """Sites 40 and 41 are also those of waits for a rank (detail: the rank, below 2^15); a slot beyond the cache sets bit 15 of the detail."""
    torch = cuda
    cache = P.bind(B, P.new_cache(torch, 2, 1, 16, 64, seed=1), 16)
    k = torch.randn((40003, 1, 64), device="cuda", dtype=torch.bfloat16)
    slots = torch.full((40003,), -1, dtype=torch.int32, device="cuda")
    for token in (0, 1, 40002):
        slots.fill_(-1)
        slots[token] = 32
        B.kv4_append(B.kv4_append_desc(cache=cache, dtype=B.BF16, tokens=40003, k=k, v=k, slots=slots))
        assert B.device_status() == (40 << 16 | 0x8000 | token & 0x7fff)
        B.kv4_gather(B.kv4_gather_desc(cache=cache, dtype=B.BF16, tokens=40003, slots=slots, k_out=k))
        assert B.device_status() == (41 << 16 | 0x8000 | token & 0x7fff)


# ---- scores at the end of the numbers ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,length", [(1, 1), (1, 5000), (12, 3), (200, 1), (200, 5000)])
def test_rows_whose_scores_are_far_below_zero(cuda, dtype, dim, rows, length):
    """All tokens have one key and one value, and the key's product with every row is about -2^105.  FP32 scores of that size are 2^82
    apart, so the weights are whatever the last bit makes them, but the value comes out: FP16 weights or probabilities are off by 2^-12
    each, and values by 2^-12, of |v| <= 5, FP32 sums by 2^-23 * (tokens / 16 + 8) of it.  The lse is off by a score's FP32
    roundings: its two parts (minimum and codes) are up to 15 times as large, and BF16 rows take keys rounded to 2^-12."""
    torch = cuda
    dt, bs = dtype_of(torch, dtype), 64
    blocks = P.blocks(length, bs)
    cache = P.new_cache(torch, blocks, 1, bs, dim, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    key = torch.rand(dim, generator=gen, device="cuda") + 1.0
    k = key.expand(length, 1, dim).to(dt).contiguous()
    v = torch.randn((1, 1, dim), generator=gen, device="cuda").clamp(-5, 5).to(dt).expand(length, 1, dim).contiguous()
    slots = torch.arange(length, device="cuda", dtype=torch.int32)
    P.append(torch, cache, bs, k, v, slots)
    q = -(torch.rand((rows, 1, dim), generator=gen, device="cuda") + 1.0).to(dt)
    scale = 2.0 ** 98
    out, lse = torch.empty_like(q), torch.zeros((rows, 1), device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    d = B.kv4_attention_desc(cache=P.bind(B, cache, bs), dtype=KINDS[dtype], requests=1, tokens=rows, q_heads=1, q=q, out=out,
                             block_table=torch.arange(blocks, device="cuda", dtype=torch.int32)[None], max_blocks=blocks, total_lens=i32([length]),
                             query_start=i32([0, rows]), max_query=rows, scale=scale, causal=False, lse=lse)
    ws = B.kv4_attention_workspace(torch, d)
    B.kv4_attention(d)
    (keys, _), (values, _) = P.read(torch, cache, bs, slots.long())
    want = values[0].expand(rows, dim)
    score = (q[:, 0].double() @ keys[0, 0]) * scale
    assert (score < -1e31).all()
    limit = 5 * (2 * 2.0 ** -12 + 2.0 ** -20 + 2.0 ** -23 * (length / 16 + 8)) + half_step(torch, dt) * want.abs()
    assert not out.isnan().any() and ((out[:, 0].double() - want).abs() <= limit).all()
    assert ((lse[:, 0].double() - score).abs() <= 15 * 2.0 ** -23 * (dim / 16 + 8) * score.abs() + 2.0 ** -12 * (rows > 128) * score.abs()).all()
    assert ws is not None and B.device_status() == 0


# ---- one launch behind another ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_reads_what_the_launch_in_front_stored(cuda, rows, dim):
    """The same slots stored anew and read at once, many times over, eagerly and in a graph: each reading is that of its own storing, to
    the bit.  Every launch may start before the one in front has ended."""
    torch = cuda
    length, bs, hk, times = 1000, 16, 2, 12
    blocks = P.blocks(length, bs)
    cache = B.kv4_new_cache(torch, blocks=blocks, block_size=bs, kv_heads=hk, head_dim=dim)
    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    kv = torch.randn((2, times, length, hk, dim), generator=gen, device="cuda").to(torch.bfloat16)
    q = torch.randn((rows, 2 * hk, dim), generator=gen, device="cuda").to(torch.bfloat16)
    outs = torch.zeros((times, rows, 2 * hk, dim), dtype=torch.bfloat16, device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = torch.arange(length, dtype=torch.int32, device="cuda")
    stores = [B.kv4_append_desc(cache=cache, dtype=B.BF16, tokens=length, k=kv[0, i], v=kv[1, i], slots=slots) for i in range(times)]
    reads = [B.kv4_attention_desc(cache=cache, dtype=B.BF16, requests=1, tokens=rows, q_heads=2 * hk, q=q, out=outs[i],
                                  block_table=torch.arange(blocks, dtype=torch.int32, device="cuda")[None], max_blocks=blocks, total_lens=i32([length]),
                                  query_start=i32([0, rows]), max_query=rows, scale=dim ** -0.5) for i in range(times)]
    ws = B.kv4_attention_workspace(torch, reads[0])
    for r in reads[1:]:
        r.workspace, r.workspace_bytes = ws.data_ptr(), ws.numel()
    for s, r in zip(stores, reads):
        B.kv4_append(s)
        torch.cuda.synchronize()
        B.kv4_attention(r)
        torch.cuda.synchronize()
    want = outs.clone()
    assert not (want[0] == want[1]).all()

    def run():
        for s, r in zip(stores, reads):
            B.kv4_append(s)
            B.kv4_attention(r)
    outs.zero_()
    run()
    same(outs, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        outs.zero_()
        graph.replay()
        same(outs, want)
    assert B.device_status() == 0


# ---- small elements beside large ones -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,rows,exponent", [("fp16", 1, 24), ("fp16", 12, 24), ("fp16", 200, 24), ("bf16", 1, 27), ("bf16", 12, 27), ("bf16", 200, 28)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_small_query_elements_keep_their_bits(cuda, dtype, rows, exponent, dim):
    """One element of a query is 2^exponent times the others; it meets a key element of zero, so only the others make scores.  Keys are
    whole numbers from 0 to 15 (scale 1, minimum 0, exact).  A score is off by the FP32 sum of its products, 2^-23 * (dim / 16 + 8) of
    their sizes' sum A; weights by that, 2^-12 and 2^-20; each moves the result by at most twice that of the largest |v - out|, sums
    by 2^-23 * (tokens / 16 + 8) of |v| + 15 s <= 4 |v|, values of many rows by 2^-12 |v|.  A is some hundreds: a query
    element that lost four of its bits would show."""
    torch = cuda
    dt, bs, length = dtype_of(torch, dtype), 16, 300
    gen = torch.Generator(device="cuda").manual_seed(dim + rows)
    blocks = P.blocks(length, bs)
    cache = P.new_cache(torch, blocks, 1, bs, dim, seed=1)
    k = torch.randint(0, 16, (length, 1, dim), generator=gen, device="cuda").to(dt)
    k[:, 0, 0], k[:, 0, 1] = 0.0, 15.0
    v = torch.randn((length, 1, dim), generator=gen, device="cuda").to(dt)
    slots = torch.arange(length, dtype=torch.int32, device="cuda")
    P.append(torch, cache, bs, k, v, slots)
    bits = 1024 if dtype == "fp16" else 128
    small = (1 + torch.randint(0, bits, (rows, 1, dim), generator=gen, device="cuda") / bits) * (torch.randint(0, 2, (rows, 1, dim), generator=gen, device="cuda") * 2 - 1)
    q = (small * 2.0 ** -12).to(dt)
    assert torch.equal(q.double(), small.double() * 2.0 ** -12)
    q[:, 0, 0] = 2.0 ** (exponent - 12)
    scale = 2.0 ** 12 * 0.125
    out = torch.empty_like(q)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    d = B.kv4_attention_desc(cache=P.bind(B, cache, bs), dtype=KINDS[dtype], requests=1, tokens=rows, q_heads=1, q=q, out=out,
                             block_table=torch.arange(blocks, dtype=torch.int32, device="cuda")[None], max_blocks=blocks, total_lens=i32([length]),
                             query_start=i32([0, rows]), max_query=rows, scale=scale, causal=False)
    ws = B.kv4_attention_workspace(torch, d)
    B.kv4_attention(d)
    (keys, _), (values, _) = P.read(torch, cache, bs, slots.long())
    assert torch.equal(keys, k.double())
    keys, values = keys[:, 0], values[:, 0]
    want = torch.softmax(q[:, 0].double() @ keys.T * scale, dim=-1) @ values
    size = float((q[:, 0, 1:].double().abs() @ keys[:, 1:].T).max()) * scale
    assert 100 < size < 8000
    error = 2.0 ** -23 * (dim / 16 + 8) * size + 2.0 ** -12 + 2.0 ** -20
    spread = values.abs().max() + want.abs().amax(-1, keepdim=True)
    limit = 2 * error * spread + (2.0 ** -23 * (length / 16 + 8) * 4 + 2.0 ** -12 * (rows > 128)) * values.abs().max() + half_step(torch, dt) * want.abs() + 1e-7
    assert ((out[:, 0].double() - want).abs() <= limit).all()
    assert ws is not None and B.device_status() == 0
