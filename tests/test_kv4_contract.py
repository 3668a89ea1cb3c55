"""CPU: what the entry points around the 4-bit cache refuse, the layout of their structs, the host-side table of turns, and
the Python builders' checks.  Nothing is launched."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import infer_b200 as B
from tests import kv4_plain as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"rope_scaling": B.RopeScaling, "rope_desc": B.RopeDesc, "kv4_cache": B.Kv4Cache, "kv4_assign_desc": B.Kv4AssignDesc,
           "kv4_release_desc": B.Kv4ReleaseDesc, "kv4_append_desc": B.Kv4AppendDesc, "kv4_gather_desc": B.Kv4GatherDesc,
           "kv4_attention_desc": B.Kv4AttentionDesc}
A = 1 << 20  # an address that nothing reads here


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines = []
    for name, struct in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof(fth_b200_{name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof(fth_b200_{name}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fth_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    for line in subprocess.check_output([str(exe)], text=True).splitlines():
        key, value = line.split()
        name, _, field = key.partition(".")
        got = getattr(STRUCTS[name], field).offset if field else C.sizeof(STRUCTS[name])
        assert got == int(value), key


# ---- turns --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [2, 10, 64, 128, 256])
@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=3.0),
                                dict(scaling="yarn", factor=8.0, original=4096, fast=32.0, slow=1.0), dict(scaling="yarn", factor=1.0, original=16, fast=2.0, slow=1.0),
                                dict(scaling="banded", factor=8.0, original=8192, fast=4.0, slow=1.0)])
def test_turns(dim, kw):
    if kw.get("scaling") == "ntk" and dim == 2:
        pytest.skip("refused")
    for base in (10000.0, 5e5):
        got, amplitude = B.rope_turns(dim, base=base, **kw)
        want, amp = P.turns(dim, base=base, **kw)
        # pow, log and the products each within a few units in the last place of 64 bits; the ramp divides by its length
        assert np.allclose(got, want, rtol=1e-13, atol=0) and abs(amplitude - amp) <= 2.0 ** -24 * amp


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, base=float("inf")),
                                dict(rotary_dim=8, scaling="linear", factor=0.5), dict(rotary_dim=8, scaling="linear", factor=float("nan")),
                                dict(rotary_dim=2, scaling="ntk", factor=2.0), dict(rotary_dim=8, scaling="yarn", factor=2.0),
                                dict(rotary_dim=8, scaling="banded", factor=2.0, original=100, fast=1.0, slow=1.0)])
def test_turns_refusals(kw):
    with pytest.raises(B.B200Error) as e:
        B.rope_turns(**kw)
    assert e.value.code == B.ERR_INVALID
    with pytest.raises(ValueError):
        B.rope_turns(8, scaling="other")


# ---- refusals -----------------------------------------------------------------------------------------------------------
def refused(fn, desc, code):
    assert getattr(B.lib(), fn)(C.byref(desc) if desc is not None else None, None) == code


def rope_desc(**kw):
    base = dict(dtype=B.BF16, layout=B.ROPE_HALF, tokens=4, head_dim=128, rotary_dim=64, positions=A, turns=A, q=A, q_out=A, q_heads=4, k=A, k_out=A, k_heads=2)
    return B.rope_desc(**{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), B.ERR_INVALID), (dict(rotary_dim=63), B.ERR_INVALID), (dict(rotary_dim=130), B.ERR_INVALID), (dict(rotary_dim=0), B.ERR_INVALID),
    (dict(layout=2), B.ERR_INVALID), (dict(q_heads=-1), B.ERR_INVALID), (dict(q_heads=0, k_heads=0), B.ERR_INVALID), (dict(q=None), B.ERR_INVALID),
    (dict(k_out=None), B.ERR_INVALID), (dict(positions=None), B.ERR_INVALID), (dict(turns=None), B.ERR_INVALID), (dict(ldq=511), B.ERR_INVALID),
    (dict(ldk_out=255), B.ERR_INVALID), (dict(q=A, q_out=A, ldq=512, ldq_out=600), B.ERR_INVALID), (dict(q=A + 1, q_out=A + 1), B.ERR_INVALID),
    (dict(amplitude=float("nan")), B.ERR_INVALID), (dict(dtype=B.INT8), B.ERR_UNSUPPORTED), (dict(tokens=1 << 31), B.ERR_UNSUPPORTED),
    (dict(head_dim=1024, rotary_dim=600), B.ERR_UNSUPPORTED), (dict(head_dim=8192), B.ERR_UNSUPPORTED)])
def test_rope_refusals(kw, code):
    refused("fth_b200_rope", rope_desc(**kw), code)


def test_rope_without_tokens_does_nothing():
    assert B.lib().fth_b200_rope(C.byref(rope_desc(tokens=0)), None) == B.OK
    refused("fth_b200_rope", None, B.ERR_INVALID)


def cache(**kw):
    base = dict(k_codes=A, v_codes=A, k_params=A, v_params=A, blocks=10, block_size=16, kv_heads=2, head_dim=128)
    return B.kv4_cache(**{**base, **kw})


CACHE_REFUSALS = [
    (dict(k_codes=None), B.ERR_INVALID), (dict(v_params=None), B.ERR_INVALID), (dict(blocks=0), B.ERR_INVALID), (dict(block_size=0), B.ERR_INVALID),
    (dict(kv_heads=0), B.ERR_INVALID), (dict(head_dim=-1), B.ERR_INVALID), (dict(k_codes=A + 8), B.ERR_INVALID), (dict(k_params=A + 2), B.ERR_INVALID),
    (dict(block_size=8), B.ERR_UNSUPPORTED), (dict(block_size=48), B.ERR_UNSUPPORTED), (dict(block_size=512), B.ERR_UNSUPPORTED),
    (dict(head_dim=96), B.ERR_UNSUPPORTED), (dict(blocks=1 << 28), B.ERR_UNSUPPORTED), (dict(kv_heads=5000), B.ERR_UNSUPPORTED)]


def append_desc(cache_kw={}, **kw):
    base = dict(dtype=B.BF16, tokens=4, k=A, v=A, slots=A)
    return B.kv4_append_desc(cache=cache(**cache_kw), **{**base, **kw})


def gather_desc(cache_kw={}, **kw):
    base = dict(dtype=B.BF16, tokens=4, k_out=A, v_out=A, slots=A)
    return B.kv4_gather_desc(cache=cache(**cache_kw), **{**base, **kw})


def attention_desc(cache_kw={}, **kw):
    base = dict(dtype=B.BF16, requests=3, tokens=7, q_heads=8, q=A, out=A, block_table=A, max_blocks=5, total_lens=A, scale=0.1, query_start=A, max_query=4,
                workspace=A, workspace_bytes=1 << 30)
    return B.kv4_attention_desc(cache=cache(**cache_kw), **{**base, **kw})


@pytest.mark.parametrize("kw,code", CACHE_REFUSALS)
def test_cache_refusals(kw, code):
    refused("fth_b200_kv4_append", append_desc(kw), code)
    refused("fth_b200_kv4_gather", gather_desc(kw), code)
    refused("fth_b200_kv4_attention", attention_desc(kw), code)
    assert B.lib().fth_b200_kv4_attention_supported(C.byref(attention_desc(kw))) == code
    assert B.lib().fth_b200_kv4_attention_workspace_bytes(C.byref(attention_desc(kw))) == 0


@pytest.mark.parametrize("kw,code", [(dict(tokens=-1), B.ERR_INVALID), (dict(k=None), B.ERR_INVALID), (dict(slots=None), B.ERR_INVALID), (dict(ldk=255), B.ERR_INVALID),
                                     (dict(v=A + 1), B.ERR_INVALID), (dict(dtype=B.E4M3), B.ERR_UNSUPPORTED), (dict(tokens=1 << 31), B.ERR_UNSUPPORTED)])
def test_append_refusals(kw, code):
    refused("fth_b200_kv4_append", append_desc(**kw), code)


@pytest.mark.parametrize("kw", [dict(k_heads=1), dict(k=A + 256), dict(tokens=3), dict(dtype=B.FP16), dict(k_out=A), dict(ldk=300), dict(rotary_dim=5)])
def test_append_refuses_a_rope_of_something_else(kw):
    refused("fth_b200_kv4_append", append_desc(rope=rope_desc(**{**dict(k_out=None), **kw})), B.ERR_INVALID)
    refused("fth_b200_kv4_append", append_desc(rope=rope_desc(k_out=None, head_dim=64)), B.ERR_INVALID)


@pytest.mark.parametrize("kw,code", [(dict(tokens=-1), B.ERR_INVALID), (dict(k_out=None, v_out=None), B.ERR_INVALID), (dict(slots=None), B.ERR_INVALID),
                                     (dict(ldv=255), B.ERR_INVALID), (dict(dtype=B.INT8), B.ERR_UNSUPPORTED)])
def test_gather_refusals(kw, code):
    refused("fth_b200_kv4_gather", gather_desc(**kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(requests=0), B.ERR_INVALID), (dict(tokens=-1), B.ERR_INVALID), (dict(q_heads=0), B.ERR_INVALID), (dict(q_heads=7), B.ERR_INVALID),
    (dict(max_blocks=0), B.ERR_INVALID), (dict(max_query=0), B.ERR_INVALID), (dict(window=-1), B.ERR_INVALID), (dict(scale=float("inf")), B.ERR_INVALID),
    (dict(query_start=None), B.ERR_INVALID), (dict(block_table=None), B.ERR_INVALID), (dict(total_lens=None), B.ERR_INVALID), (dict(q=None), B.ERR_INVALID),
    (dict(ldq=100), B.ERR_INVALID), (dict(workspace=None), B.ERR_INVALID), (dict(workspace_bytes=100), B.ERR_INVALID), (dict(workspace=A + 64), B.ERR_INVALID),
    (dict(dtype=B.FP32), B.ERR_UNSUPPORTED), (dict(max_blocks=1 << 28), B.ERR_UNSUPPORTED)])
def test_attention_refusals(kw, code):
    refused("fth_b200_kv4_attention", attention_desc(**kw), code)


def test_no_tokens_do_nothing():
    assert B.lib().fth_b200_kv4_append(C.byref(append_desc(tokens=0, k=None, v=None, slots=None)), None) == B.OK
    assert B.lib().fth_b200_kv4_gather(C.byref(gather_desc(tokens=0)), None) == B.OK
    assert B.lib().fth_b200_kv4_attention(C.byref(attention_desc(tokens=0)), None) == B.OK


TABLES = dict(requests=3, max_blocks=4, block_size=16, blocks=10, free_blocks=A, free_count=A, free_count_out=A, block_table=A, status=A)
ASSIGN = dict(TABLES, tokens=5, cached_lens=A, new_lens=A, total_lens=A, query_start=A, slots=A, positions=A)
RELEASE = dict(TABLES, lens=A, keep_lens=A, lens_out=A)


@pytest.mark.parametrize("kw,code", [(dict(requests=0), B.ERR_INVALID), (dict(max_blocks=0), B.ERR_INVALID), (dict(blocks=0), B.ERR_INVALID),
                                     (dict(block_size=20), B.ERR_UNSUPPORTED), (dict(max_blocks=1 << 28), B.ERR_UNSUPPORTED), (dict(blocks=1 << 28), B.ERR_UNSUPPORTED)]
                         + [({name: None}, B.ERR_INVALID) for name in TABLES if TABLES[name] is A])
def test_table_refusals(kw, code):
    refused("fth_b200_kv4_assign", B.kv4_assign_desc(**{**ASSIGN, **kw}), code)
    refused("fth_b200_kv4_release", B.kv4_release_desc(**{**RELEASE, **kw}), code)


def test_assign_and_release_refusals():
    for name in ("cached_lens", "new_lens", "total_lens", "query_start", "slots", "positions"):
        refused("fth_b200_kv4_assign", B.kv4_assign_desc(**{**ASSIGN, name: None}), B.ERR_INVALID)
    refused("fth_b200_kv4_assign", B.kv4_assign_desc(**{**ASSIGN, "tokens": -1}), B.ERR_INVALID)
    refused("fth_b200_kv4_assign", B.kv4_assign_desc(**{**ASSIGN, "tokens": 1 << 31}), B.ERR_UNSUPPORTED)
    for name in ("lens", "keep_lens", "lens_out"):
        refused("fth_b200_kv4_release", B.kv4_release_desc(**{**RELEASE, name: None}), B.ERR_INVALID)
    for fn in ("assign", "release", "append", "gather", "attention"):
        refused(f"fth_b200_kv4_{fn}", None, B.ERR_INVALID)


def test_builders_refuse_tensors_that_do_not_fit():
    """Host tensors, wrong element sizes, strides without whole heads, too few elements."""
    import torch
    x = torch.zeros((4, 4, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on a GPU"):
        rope_desc(q=x, q_out=x)
    with pytest.raises(ValueError, match="byte elements"):
        rope_desc(q=x.float(), q_out=x)
    with pytest.raises(ValueError, match="heads 128 apart"):
        rope_desc(q=x.transpose(0, 1), q_out=x)
    with pytest.raises(ValueError, match="heads 128 apart"):
        rope_desc(q=torch.zeros((4, 4, 256), dtype=torch.bfloat16)[:, :, ::2], q_out=x)
    with pytest.raises(ValueError, match="needs 4"):
        rope_desc(positions=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="float64"):
        rope_desc(turns=torch.zeros(32))
    with pytest.raises(ValueError, match="not contiguous"):
        rope_desc(positions=torch.zeros((4, 2), dtype=torch.int32)[:, 0])
    with pytest.raises(ValueError, match="needs"):
        cache(k_codes=torch.zeros(10, dtype=torch.uint8))
    with pytest.raises(ValueError, match="block_table"):
        attention_desc(block_table=torch.zeros(14, dtype=torch.int32))
    with pytest.raises(ValueError, match="slots"):
        append_desc(slots=torch.zeros(4, dtype=torch.int64))


# ---- the plain forms themselves -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_the_plain_quantiser_keeps_its_definition(dtype):
    import torch
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn((300, 64), generator=gen) * torch.exp2(torch.randint(-20, 10, (300, 1), generator=gen))).to(getattr(torch, dtype))
    x[0] = 0
    x[1] = 3.25
    codes, scale, minimum = P.quantise(torch, x)
    y = x.double()
    assert torch.equal(scale.to(torch.bfloat16).double(), scale) and torch.equal(minimum.to(torch.bfloat16).double(), minimum)
    assert (minimum <= y.amin(-1)).all() and (15 * scale >= y.amax(-1) - minimum).all()
    below = scale * (1 - 2.0 ** -8)  # under the next smaller BF16 number's upper neighbour
    assert ((15 * below < (y.amax(-1) - minimum) * (1 + 2.0 ** -7)) | (scale == 2.0 ** -126) | (scale == 0)).all()
    back = minimum[:, None] + scale[:, None] * codes.double()
    assert ((back - y).abs() <= scale[:, None] / 2).all()
