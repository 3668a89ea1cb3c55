"""One decode / prefill-chunk step of a projection stack, issued as C-ABI calls on one stream.

The layer is the one the synthetic 24-layer configuration uses (hidden H, intermediate I, BF16 residual stream, FP8
projections wrapped in Cast nodes, QwenRmsNorm with weight offset 1, SiLU * Mul between gate / up and down):

    h = QwenRmsNorm(x, g1);  t = o(v(k(q(h))));  x = Add(x, t)
    h = QwenRmsNorm(x, g2);  a = Mul(SiLU(gate(h)), up(h));  x = Add(x, down(a))

`fused=True` issues six launches per layer through fth_b200_fp8_linear_fused — norm + q, k, v, o + residual,
norm + gate | up + SiLU * Mul (one launch, two weights), down + residual — and every launch whose output feeds the next
projection directly also stores the FP8 codes that projection's Cast would make of it (out_codes), so that k, v, o and
down read 8-bit activations and run no Cast of their own; `fused=False` issues every node's own kernel
(twelve launches per layer: fth_b200_qwen_rms_norm, the Cast -> MatMul -> Cast projections, fth_b200_binary,
fth_b200_silu_mul).  Both give the same bytes.  Everything stays on the device; the caller may capture `run` in a CUDA
graph.  torch supplies the device buffers only.

`attention=` (an AttentionState) puts causal attention over a paged 4-bit cache between the projections: q, k and v start
from the normalised input, q and k get their rotary positions, k and v go into the cache, and o projects what attention
gives,

    h = QwenRmsNorm(x, g1);  q, k, v = q(h), k(h), v(h);  x = Add(x, o(attention(rope(q), cache + (rope(k), v))))

with q [H, q_heads * head_dim], k and v [H, kv_heads * head_dim] and o [q_heads * head_dim, H].  The step then begins with
the tables (fth_b200_kv4_assign: blocks, slots and positions of its rows), and a layer's first half is five launches:
norm + q, norm + k | v, rope + append, attention, o + residual.
"""
from __future__ import annotations

import ctypes as C

import infer_b200 as B


class AttentionState:
    """What the requests of a batch hold between steps: one 4-bit cache per layer, and the lengths, the block table and the
    stack of free blocks that the layers share.  Steps of different sizes (a prompt's rows, then one row per request) may use
    the same state one after another."""

    def __init__(self, torch, *, layers, requests, q_heads, kv_heads, head_dim, blocks, block_size=64, max_blocks=None, rotary_dim=None,
                 layout=B.ROPE_HALF, window=0, scale=None, **turns):
        """blocks: of every layer's cache.  max_blocks: of one request (default: all).  turns: base, scaling, ... of rope_turns."""
        self.requests, self.q_heads, self.kv_heads, self.head_dim = requests, q_heads, kv_heads, head_dim
        self.blocks, self.block_size, self.max_blocks = blocks, block_size, max_blocks or blocks
        self.layout, self.window, self.scale = layout, window, head_dim ** -0.5 if scale is None else scale
        self.caches = [B.kv4_new_cache(torch, blocks=blocks, block_size=block_size, kv_heads=kv_heads, head_dim=head_dim) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, **i32)         # tokens held; a step adds its own
        self.keep_lens = torch.zeros(requests, **i32)    # what `release` leaves
        self.table = torch.full((requests, self.max_blocks), -1, **i32)
        self.free = torch.arange(blocks, **i32)
        self.free_count = torch.full((1,), blocks, **i32)
        self.status = torch.zeros(2, **i32)              # [0]: FTH_B200_KV4_* of the last step or release
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        host, self.amplitude = B.rope_turns(self.rotary_dim, **turns)
        self.turns = torch.from_numpy(host).cuda()
        self._release = B.kv4_release_desc(requests=requests, max_blocks=self.max_blocks, block_size=block_size, blocks=blocks, lens=self.lens,
                                           keep_lens=self.keep_lens, free_blocks=self.free, free_count=self.free_count, free_count_out=self.free_count,
                                           block_table=self.table, lens_out=self.lens, status=self.status)
        self.release()   # of nothing: sizes that cannot be are refused here

    def release(self, stream=None):
        """Shrinks every request to keep_lens tokens and gives its other blocks back."""
        B.kv4_release(self._release, stream)


class DecoderStep:
    def __init__(self, torch, layers, m, hidden, inter, act_scale, out_scale, fp8_dtype=None, epsilon=1e-6, fused=True, attention=None,
                 max_query=None):
        """layers: per layer a dict with device tensors q, k, v, o, gate, up, down (FP8 codes, [K,N]) + their scales
        ("q_scale", ...) and g1, g2 (BF16 bits as int16 tensors, [hidden]).
        attention: an AttentionState.  new_lens then says how many of the m rows each request appends, in order; rows behind
        the last one belong to nobody.  max_query: the most rows of one request (default m; 1 for single tokens, which
        have a kernel of their own)."""
        self.torch, self.layers, self.m, self.hidden, self.inter = torch, layers, m, hidden, inter
        self.act_scale, self.out_scale, self.eps, self.fused = act_scale, out_scale, epsilon, fused
        self.dtype = fp8_dtype or B.E5M2
        bf = dict(dtype=torch.int16, device="cuda")
        self.x = torch.zeros((m, hidden), **bf)          # residual stream (input and output of the step)
        self.h = torch.zeros((m, hidden), **bf)
        self.t = [torch.zeros((m, hidden), **bf) for _ in range(2)]
        self.x2 = torch.zeros((m, hidden), **bf)
        self.gate = torch.zeros((m, inter), **bf)
        self.up = torch.zeros((m, inter), **bf)
        self.act = torch.zeros((m, inter), **bf)
        codes = dict(dtype=torch.uint8, device="cuda")
        self.c = [torch.zeros((m, hidden), **codes) for _ in range(2)]   # FP8 codes of t[0] / t[1] for the next projection
        self.act_codes = torch.zeros((m, inter), **codes)
        self.keep = []
        self.calls = []
        self.attention, self.max_query = attention, m if max_query is None else max_query
        if attention is not None:
            self._tables()
        self._build()

    # ---- descriptors -------------------------------------------------------------------------------------------------
    def _proj(self, a, w, w_scale, out, k, n, codes_in=False):
        """codes_in: `a` holds the FP8 codes of the activation already (a producer's out_codes)."""
        d = B.fp8_linear_desc(dtype=self.dtype, op=B.OP_MATMUL, m=self.m, k=k, n=n, a=a, w=w, out=out, a_scale=self.act_scale,
                              w_scale=w_scale, out_scale=self.out_scale, a_dtype=0 if codes_in else B.BF16, out_dtype=B.BF16,
                              weights_static=True)
        self.keep.append(B.linear_workspace(self.torch, d))
        return d

    def _plain(self, d):
        self.calls.append(("linear", d, None))

    def _fused(self, d, **kw):
        f = B.fp8_linear_fusion(**kw)
        rc = B.lib().fth_b200_fp8_linear_fused_supported(C.byref(d), C.byref(f))
        if rc != 0:
            raise B.B200Error(rc, "fth_b200_fp8_linear_fused_supported")
        self.calls.append(("fused", d, f))

    def _tables(self):
        a, m = self.attention, self.m
        i32 = dict(dtype=self.torch.int32, device="cuda")
        self.new_lens = self.torch.zeros(a.requests, **i32)
        self.starts = self.torch.zeros(a.requests + 1, **i32)
        self.slots, self.positions = (self.torch.full((m,), -1, **i32) for _ in range(2))
        wide = lambda heads: self.torch.zeros((m, heads, a.head_dim), dtype=self.torch.int16, device="cuda")  # noqa: E731
        self.q, self.q_turned, self.attended = wide(a.q_heads), wide(a.q_heads), wide(a.q_heads)
        self.k, self.v = wide(a.kv_heads), wide(a.kv_heads)
        self.calls.append(("kv4_assign", B.kv4_assign_desc(
            requests=a.requests, max_blocks=a.max_blocks, block_size=a.block_size, blocks=a.blocks, tokens=m, cached_lens=a.lens, new_lens=self.new_lens,
            free_blocks=a.free, free_count=a.free_count, free_count_out=a.free_count, block_table=a.table, total_lens=a.lens, query_start=self.starts,
            slots=self.slots, positions=self.positions, status=a.status), None))
        self.workspace = None

    def _attend(self, x, nxt, layer, cache):
        a, m, H = self.attention, self.m, self.hidden
        wide, narrow = a.q_heads * a.head_dim, a.kv_heads * a.head_dim
        turn = B.rope_desc(dtype=B.BF16, layout=a.layout, tokens=m, head_dim=a.head_dim, rotary_dim=a.rotary_dim, positions=self.positions, turns=a.turns,
                           amplitude=a.amplitude, q=self.q, q_out=self.q_turned, q_heads=a.q_heads, k=self.k, k_heads=a.kv_heads)
        append = B.kv4_append_desc(cache=cache, dtype=B.BF16, tokens=m, k=self.k, v=self.v, slots=self.slots, rope=turn)
        attend = B.kv4_attention_desc(cache=cache, dtype=B.BF16, requests=a.requests, tokens=m, q_heads=a.q_heads, q=self.q_turned, out=self.attended,
                                      block_table=a.table, max_blocks=a.max_blocks, total_lens=a.lens, query_start=self.starts, max_query=self.max_query,
                                      scale=a.scale, window=a.window)
        if self.workspace is None:   # the layers run one after another
            self.workspace = B.kv4_attention_workspace(self.torch, attend)
        else:
            attend.workspace, attend.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
        if self.fused:
            norm = dict(prologue=B.FUSE_RMS_NORM, norm_weight=layer["g1"], norm_weight_offset=1.0, norm_epsilon=self.eps)
            self._fused(self._proj(x, layer["q"], layer["q_scale"], self.q, H, wide), **norm)
            self._fused(self._proj(x, layer["k"], layer["k_scale"], self.k, H, narrow), w2=layer["v"], w2_scale=layer["v_scale"], out2=self.v, n2=narrow,
                        **norm)
        else:
            self.calls.append(("norm", (x, layer["g1"], self.h), None))
            for name, out, n in (("q", self.q, wide), ("k", self.k, narrow), ("v", self.v, narrow)):
                self._plain(self._proj(self.h, layer[name], layer[name + "_scale"], out, H, n))
        self.calls.append(("kv4_append", append, None))
        self.calls.append(("kv4_attention", attend, None))
        if self.fused:
            self._fused(self._proj(self.attended, layer["o"], layer["o_scale"], nxt, wide, H), residual=x)
        else:
            self._plain(self._proj(self.attended, layer["o"], layer["o_scale"], self.t[1], wide, H))
            self.calls.append(("add", (x, self.t[1], nxt, m * H), None))

    def _build(self):
        H, I, m = self.hidden, self.inter, self.m
        x, nxt = self.x, self.x2
        for index, layer in enumerate(self.layers):
            attend = self.attention is not None
            if attend:
                self._attend(x, nxt, layer, self.attention.caches[index])
                x, nxt = nxt, x
            if self.fused:
                cast = dict(out_codes_scale=self.act_scale)  # the Cast in front of the next projection, run by the producer
                if not attend:
                    self._fused(self._proj(x, layer["q"], layer["q_scale"], self.t[0], H, H), prologue=B.FUSE_RMS_NORM, norm_weight=layer["g1"],
                                norm_weight_offset=1.0, norm_epsilon=self.eps, out_codes=self.c[0], **cast)
                    self._fused(self._proj(self.c[0], layer["k"], layer["k_scale"], self.t[1], H, H, codes_in=True), out_codes=self.c[1], **cast)
                    self._fused(self._proj(self.c[1], layer["v"], layer["v_scale"], self.t[0], H, H, codes_in=True), out_codes=self.c[0], **cast)
                    self._fused(self._proj(self.c[0], layer["o"], layer["o_scale"], nxt, H, H, codes_in=True), residual=x)
                    x, nxt = nxt, x
                self._fused(self._proj(x, layer["gate"], layer["gate_scale"], self.gate, H, I), prologue=B.FUSE_RMS_NORM, norm_weight=layer["g2"],
                            norm_weight_offset=1.0, norm_epsilon=self.eps, w2=layer["up"], w2_scale=layer["up_scale"], n2=I,
                            epilogue=B.FUSE_OUT_SILU_MUL, out_codes=self.act_codes, **cast)
                self._fused(self._proj(self.act_codes, layer["down"], layer["down_scale"], nxt, I, H, codes_in=True), residual=x)
                x, nxt = nxt, x
            else:
                if not attend:
                    self.calls.append(("norm", (x, layer["g1"], self.h), None))
                    self._plain(self._proj(self.h, layer["q"], layer["q_scale"], self.t[0], H, H))
                    self._plain(self._proj(self.t[0], layer["k"], layer["k_scale"], self.t[1], H, H))
                    self._plain(self._proj(self.t[1], layer["v"], layer["v_scale"], self.t[0], H, H))
                    self._plain(self._proj(self.t[0], layer["o"], layer["o_scale"], self.t[1], H, H))
                    self.calls.append(("add", (x, self.t[1], nxt, m * H), None))
                    x, nxt = nxt, x
                self.calls.append(("norm", (x, layer["g2"], self.h), None))
                self._plain(self._proj(self.h, layer["gate"], layer["gate_scale"], self.gate, H, I))
                self._plain(self._proj(self.h, layer["up"], layer["up_scale"], self.up, H, I))
                self.calls.append(("silu_mul", (self.gate, self.up, self.act, m * I), None))
                self._plain(self._proj(self.act, layer["down"], layer["down_scale"], self.t[0], I, H))
                self.calls.append(("add", (x, self.t[0], nxt, m * H), None))
                x, nxt = nxt, x
        self.result = x  # the buffer that holds the final hidden state after run()

    # ---- one step ----------------------------------------------------------------------------------------------------
    def run(self, stream=None):
        """Issues the whole step on `stream` (default: torch's current stream).  self.x holds the input, self.result
        the output (an even number of residual updates brings it back to self.x)."""
        lib = B.lib()
        s = stream or B.current_stream()
        for kind, d, f in self.calls:
            if kind == "linear":
                rc = lib.fth_b200_fp8_linear(C.byref(d), s)
            elif kind.startswith("kv4_"):
                rc = getattr(lib, "fth_b200_" + kind)(C.byref(d), s)
            elif kind == "fused":
                rc = lib.fth_b200_fp8_linear_fused(C.byref(d), C.byref(f), s)
            elif kind == "norm":
                x, g, out = d
                rc = lib.fth_b200_qwen_rms_norm(C.c_int32(B.BF16), C.c_void_p(x.data_ptr()), C.c_int32(B.BF16), C.c_void_p(g.data_ptr()), C.c_float(1.0),
                                                C.c_float(self.eps), C.c_int32(B.BF16), C.c_void_p(out.data_ptr()), C.c_int64(self.m), C.c_int64(self.hidden), s)
            elif kind == "add":
                a, b, out, count = d
                rc = lib.fth_b200_binary(C.c_int32(B.BINARY_ADD), C.c_int32(B.BF16), C.c_void_p(a.data_ptr()), C.c_void_p(b.data_ptr()),
                                         C.c_void_p(out.data_ptr()), C.c_int64(count), C.c_int64(0), s)
            else:
                g, u, out, count = d
                rc = lib.fth_b200_silu_mul(C.c_int32(B.BF16), C.c_void_p(g.data_ptr()), C.c_void_p(u.data_ptr()), C.c_void_p(out.data_ptr()),
                                           C.c_int64(count), s)
            if rc != 0:
                raise B.B200Error(rc, f"decoder step ({kind})")

    @property
    def launches(self):
        return len(self.calls)


def _main():
    """Runs the synthetic stack a few times with random weights and prints the time per step (CUDA events), e.g. as the
    workload of a profiler capture: python -m infer_b200.decoder_step --m 16 --layers 4"""
    import argparse

    import torch

    ap = argparse.ArgumentParser()
    ap.add_argument("--m", type=int, default=1)
    ap.add_argument("--layers", type=int, default=24)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inter", type=int, default=3584)
    ap.add_argument("--steps", type=int, default=3)
    ap.add_argument("--nodes", action="store_true", help="every node as its own launch instead of the fused calls")
    ap.add_argument("--attend", type=int, default=0, help="attention over a 4-bit cache: m requests that hold this many tokens each")
    args = ap.parse_args()
    H, I = args.hidden, args.inter
    D, KV = 128, max(H // 512, 1) * 128   # heads of 128, four query heads to a key head
    narrow = KV if args.attend else H
    shapes = {"q": (H, H), "k": (H, narrow), "v": (H, narrow), "o": (H, H), "gate": (H, I), "up": (H, I), "down": (I, H)}
    gen = torch.Generator(device="cuda").manual_seed(7)
    weights = []
    for _ in range(args.layers):
        layer = {}
        for name, (k, n) in shapes.items():
            layer[name] = torch.randint(0, 120, (k, n), dtype=torch.uint8, device="cuda", generator=gen)
            layer[name + "_scale"] = 2.0 ** -20
        for g in ("g1", "g2"):
            layer[g] = (torch.randn(H, device="cuda", generator=gen) * 0.1).to(torch.bfloat16).view(torch.int16)
        weights.append(layer)
    state = None
    if args.attend:
        per = -(-(args.attend + 2 * args.steps + 8) // 64)
        state = AttentionState(torch, layers=args.layers, requests=args.m, q_heads=H // D, kv_heads=KV // D, head_dim=D, blocks=per * args.m, max_blocks=per)
    step = DecoderStep(torch, weights, args.m, H, I, 2.0 ** -9, 2.0 ** -9, fused=not args.nodes, attention=state, max_query=1)
    if state:   # as if each request held `attend` tokens (of zeros): their blocks are taken from the stack
        step.new_lens.fill_(1)
        held = -(-args.attend // 64)
        state.lens.fill_(args.attend)
        state.table[:, :held] = torch.arange(args.m * held, dtype=torch.int32, device="cuda").view(args.m, held)
        state.free.copy_(torch.arange(per * args.m, dtype=torch.int32, device="cuda").flip(0))
        state.free_count.fill_(per * args.m - args.m * held)
    step.x.copy_(torch.randn((args.m, H), device="cuda", generator=gen).to(torch.bfloat16).view(torch.int16))
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    step.run()
    torch.cuda.synchronize()
    begin.record()
    for _ in range(args.steps):
        step.run()
    end.record()
    torch.cuda.synchronize()
    print(f"m={args.m} layers={args.layers} launches/step={step.launches} {begin.elapsed_time(end) / args.steps * 1e3:.1f} us/step "
          f"(stream launches, no graph) status={B.device_status()}")


if __name__ == "__main__":
    _main()
