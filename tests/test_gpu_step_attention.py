"""GPU: a decoder step with attention over the 4-bit cache (infer_b200/decoder_step.py), as a user runs it: a prompt's rows, then
single tokens, from one AttentionState.

* One layer, step by step: every node that is not new is run again through its own entry point from the step's own buffers and
  gives the step's bytes; what is new (tables, cache contents, attention) is compared with the plain forms of kv4_plain.py.
  A row of attention is off by at most the limit that kv4_plain.attention derives (the kernels' arithmetic), half a BF16 step
  (2^-8 of the value at most) and, with more than 128 rows to a key head, the keys' rounding to FP16.
* Fused calls, node-by-node calls and replays of a captured step give the same bytes."""
import ctypes as C

import numpy as np
import pytest

import infer_b200 as B
from infer_b200.decoder_step import AttentionState, DecoderStep
from tests import kv4_plain as P

pytestmark = pytest.mark.gpu
HIDDEN, INTER = 512, 1024
ACT, OUT = 2.0 ** -9, 2.0 ** -9


def make_layers(torch, count, hq, hk, dim, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = {"q": (HIDDEN, hq * dim), "k": (HIDDEN, hk * dim), "v": (HIDDEN, hk * dim), "o": (hq * dim, HIDDEN), "gate": (HIDDEN, INTER),
              "up": (HIDDEN, INTER), "down": (INTER, HIDDEN)}
    out = []
    for _ in range(count):
        layer = {}
        for name, shape in shapes.items():
            w = torch.randn(shape, generator=gen, device="cuda") * 0.05
            layer[name + "_scale"] = 2.0 ** -16   # 57344 codes reach 0.87: 17 standard deviations
            layer[name] = (w / 2.0 ** -16).to(torch.float8_e5m2).view(torch.uint8)
        for g in ("g1", "g2"):
            layer[g] = (torch.randn(HIDDEN, generator=gen, device="cuda") * 0.1).to(torch.bfloat16).view(torch.int16)
        out.append(layer)
    return out


def bf16(torch, t):
    return t.view(torch.bfloat16)


def linear(torch, a, layer, name, m):
    k, n = layer[name].shape
    out = torch.zeros((m, n), dtype=torch.int16, device="cuda")
    d = B.fp8_linear_desc(dtype=B.E5M2, op=B.OP_MATMUL, m=m, k=k, n=n, a=a, w=layer[name], out=out, a_scale=ACT, w_scale=layer[name + "_scale"],
                          out_scale=OUT, a_dtype=B.BF16, out_dtype=B.BF16)
    ws = B.linear_workspace(torch, d)
    B.fp8_linear(d)
    torch.cuda.synchronize()
    del ws
    return out


def norm(torch, x, g, m):
    out = torch.zeros_like(x)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    B.check(B.lib().fth_b200_qwen_rms_norm(C.c_int32(B.BF16), p(x), C.c_int32(B.BF16), p(g), C.c_float(1.0), C.c_float(1e-6), C.c_int32(B.BF16), p(out),
                                           C.c_int64(m), C.c_int64(HIDDEN), B.current_stream()), "norm")
    return out


def add(torch, a, b):
    out = torch.zeros_like(a)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    B.check(B.lib().fth_b200_binary(C.c_int32(B.BINARY_ADD), C.c_int32(B.BF16), p(a), p(b), p(out), C.c_int64(a.numel()), C.c_int64(0), B.current_stream()),
            "add")
    return out


def make_state(torch, layers, hq, hk, dim, requests, **more):
    state = AttentionState(torch, layers=layers, requests=requests, q_heads=hq, kv_heads=hk, head_dim=dim, blocks=requests * 12, block_size=16,
                           max_blocks=12, **more)
    state.free.copy_(torch.randperm(state.blocks, device="cuda").to(torch.int32))
    return state


@pytest.mark.parametrize("hq,hk,dim,window,layout", [(8, 2, 64, 0, B.ROPE_HALF), (4, 4, 128, 20, B.ROPE_INTERLEAVED), (6, 1, 64, 0, B.ROPE_HALF)])
@pytest.mark.parametrize("fused", [True, False])
def test_steps_of_one_layer(cuda, hq, hk, dim, window, layout, fused):
    torch = cuda
    torch.manual_seed(hq)
    requests, bs = 3, 16
    layer = make_layers(torch, 1, hq, hk, dim, seed=dim)[0]
    state = make_state(torch, 1, hq, hk, dim, requests, window=window, layout=layout, base=500000.0)
    shape = (state.blocks, hk, bs)
    mirror = dict(k_codes=torch.zeros((*shape, dim // 2), dtype=torch.uint8, device="cuda"), v_codes=torch.zeros((*shape, dim // 2), dtype=torch.uint8, device="cuda"),
                  k_params=torch.zeros((*shape, 2), dtype=torch.bfloat16, device="cuda"), v_params=torch.zeros((*shape, 2), dtype=torch.bfloat16, device="cuda"))
    args = dict(hidden=HIDDEN, inter=INTER, act_scale=ACT, out_scale=OUT, attention=state)
    prompt = DecoderStep(torch, [layer], 64, fused=False, **args)   # the fused calls take up to 32 rows
    single = DecoderStep(torch, [layer], requests + 1, max_query=1, fused=fused, **args)
    have = [0] * requests
    for step, grow in ((prompt, [37, 1, 20]), (single, [1, 1, 1]), (single, [1, 0, 1]), (prompt, [2, 33, 0]), (single, [1, 1, 1])):
        rows, m = sum(grow), step.m
        x = torch.randn((m, HIDDEN), device="cuda").to(torch.bfloat16).view(torch.int16)
        step.x.copy_(x)
        step.new_lens.copy_(torch.tensor(grow, dtype=torch.int32))
        step.attended.fill_(0x3f80)
        step.run()
        torch.cuda.synchronize()
        assert B.device_status() == 0
        have = [a + g for a, g in zip(have, grow)]
        assert state.status.cpu().tolist() == [0, 0] and state.lens.cpu().tolist() == have
        assert state.free_count.item() == state.blocks - sum(P.blocks(n, bs) for n in have)
        # the projections in front, from the step's input
        h = norm(torch, x, layer["g1"], m)
        q, k, v = (linear(torch, h, layer, name, m) for name in ("q", "k", "v"))
        assert torch.equal(step.q.view(m, -1), q) and torch.equal(step.k.view(m, -1), k) and torch.equal(step.v.view(m, -1), v)
        # rotary positions: 64 bits, half a BF16 step and the FP32 arithmetic (four roundings of the pair's size)
        positions = torch.cat([torch.arange(a - g, a, device="cuda") for a, g in zip(have, grow)])
        assert torch.equal(step.positions[:rows].long(), positions) and (step.positions[rows:] == -1).all()
        name = "half" if layout == B.ROPE_HALF else "interleaved"
        turned, size = P.rope(torch, bf16(torch, step.q)[:rows], positions, state.turns, state.amplitude, name)
        got = bf16(torch, step.q_turned)[:rows].double()
        assert ((got - turned).abs() <= 2.0 ** -8 * turned.abs() + 2.0 ** -21 * size).all()
        # the cache, from the keys that the framework's own rope gives, and attention over it
        kr = torch.empty_like(step.k)
        B.rope(B.rope_desc(dtype=B.BF16, layout=layout, tokens=m, head_dim=dim, rotary_dim=dim, positions=step.positions, turns=state.turns,
                           amplitude=state.amplitude, k=step.k, k_out=kr, k_heads=hk))
        P.append(torch, mirror, bs, bf16(torch, kr)[:rows], bf16(torch, step.v)[:rows], step.slots[:rows])
        cache = state.caches[0]
        keys, values = (torch.zeros((rows, hk, dim), dtype=torch.float32, device="cuda") for _ in range(2))
        B.kv4_gather(B.kv4_gather_desc(cache=cache, dtype=B.FP32, tokens=rows, slots=step.slots, k_out=keys, v_out=values))
        (want_k, _), (want_v, _) = P.read(torch, mirror, bs, step.slots[:rows].long())
        assert torch.equal(keys, want_k.float()) and torch.equal(values, want_v.float())
        many = step.max_query * (hq // hk) > 128
        want, _, limit, _ = P.attention(torch, mirror, bs, state.table, bf16(torch, step.q_turned)[:rows], have, grow, hk, state.scale, True, window,
                                        key_rounding=2.0 ** -12 if many else 0.0)
        got = bf16(torch, step.attended)[:rows].double()
        assert ((got - want).abs() <= limit + 2.0 ** -8 * want.abs() + 1e-30).all()
        assert (step.attended[rows:] == 0x3f80).all()     # nobody's rows
        # what follows, from the step's attention
        y = add(torch, x, linear(torch, step.attended.view(m, -1), layer, "o", m))
        h = norm(torch, y, layer["g2"], m)
        act = torch.zeros((m, INTER), dtype=torch.int16, device="cuda")
        B.silu_mul(B.BF16, linear(torch, h, layer, "gate", m), linear(torch, h, layer, "up", m), act, m * INTER)
        y = add(torch, y, linear(torch, act, layer, "down", m))
        assert torch.equal(step.result, y)
    # rejected drafts, then everybody done
    keep = [max(n - 18, 0) for n in have]
    for left in (keep, [0] * requests):
        state.keep_lens.copy_(torch.tensor(left, dtype=torch.int32))
        state.release()
        assert state.status.cpu().tolist() == [0, 0] and state.lens.cpu().tolist() == left
        assert state.free_count.item() == state.blocks - sum(P.blocks(n, bs) for n in left)
    assert sorted(state.free.cpu().tolist()) == list(range(state.blocks))


def test_fused_calls_nodes_and_replays_agree(cuda):
    torch = cuda
    hq, hk, dim, requests, count = 8, 2, 64, 2, 2
    layers = make_layers(torch, count, hq, hk, dim, seed=1)
    grows = [[30, 9], [1, 1], [1, 1], [1, 0], [1, 1]]
    inputs = [torch.randn((48 if i == 0 else 2, HIDDEN), device="cuda").to(torch.bfloat16).view(torch.int16) for i in range(len(grows))]
    results = []
    for fused, captured in ((True, False), (False, False), (True, True)):
        state = AttentionState(torch, layers=count, requests=requests, q_heads=hq, kv_heads=hk, head_dim=dim, blocks=24, block_size=16, max_blocks=12)
        args = dict(hidden=HIDDEN, inter=INTER, act_scale=ACT, out_scale=OUT, attention=state)
        prompt, single = DecoderStep(torch, layers, 48, fused=False, **args), DecoderStep(torch, layers, 2, max_query=1, fused=fused, **args)
        assert prompt.launches == 1 + 14 * count and single.launches == 1 + (7 if fused else 14) * count
        graphs = {}
        if captured:
            side = torch.cuda.Stream()
            for step in (prompt, single):
                with torch.cuda.stream(side):
                    step.run()          # no new tokens: nothing is taken or written
                    torch.cuda.synchronize()
                    graphs[step] = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graphs[step], stream=side):
                        step.run()
            assert state.lens.cpu().tolist() == [0, 0]
        outs = []
        for x, grow in zip(inputs, grows):
            step = prompt if x.shape[0] == 48 else single
            step.x.copy_(x)
            step.new_lens.copy_(torch.tensor(grow, dtype=torch.int32))
            torch.cuda.synchronize()
            graphs[step].replay() if captured else step.run()
            torch.cuda.synchronize()
            outs.append(step.result[:sum(grow)].cpu().numpy().copy())
        assert B.device_status() == 0 and state.lens.cpu().tolist() == [34, 12]
        results.append(outs)
        graphs.clear()
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert np.array_equal(a, b)


def test_a_step_that_does_not_fit_changes_nothing(cuda):
    """More tokens than there are blocks: the state says so, and lengths, tables and caches stay as they were."""
    torch = cuda
    layers = make_layers(torch, 1, 8, 2, 64, seed=2)
    state = AttentionState(torch, layers=1, requests=2, q_heads=8, kv_heads=2, head_dim=64, blocks=3, block_size=16)
    step = DecoderStep(torch, layers, 32, HIDDEN, INTER, ACT, OUT, attention=state)
    step.x.copy_(torch.randn((32, HIDDEN), device="cuda").to(torch.bfloat16).view(torch.int16))
    for grow, lens, code in (([20, 10], [20, 10], 0), ([20, 1], [20, 10], 1), ([1, 1], [21, 11], 0)):
        before = [t.clone() for t in (state.table, state.free_count)]
        step.new_lens.copy_(torch.tensor(grow, dtype=torch.int32))
        step.run()
        torch.cuda.synchronize()
        assert state.status[0].item() == code and state.lens.cpu().tolist() == lens
        if code:
            assert torch.equal(before[0], state.table) and torch.equal(before[1], state.free_count)
            assert (step.slots == -1).all()
    assert B.device_status() == 0


def test_wrong_shapes_are_refused(cuda):
    torch = cuda
    layers = make_layers(torch, 1, 8, 2, 64, seed=3)
    with pytest.raises(B.B200Error):
        AttentionState(torch, layers=1, requests=2, q_heads=8, kv_heads=2, head_dim=64, blocks=4, block_size=24)
    state = AttentionState(torch, layers=1, requests=2, q_heads=7, kv_heads=2, head_dim=64, blocks=4, block_size=16)
    with pytest.raises((B.B200Error, ValueError)):
        DecoderStep(torch, layers, 4, HIDDEN, INTER, ACT, OUT, attention=state)
