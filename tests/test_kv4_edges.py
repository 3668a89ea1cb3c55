"""CPU: refusals around the 4-bit cache that tests/test_kv4_contract.py does not have.  Nothing is launched."""
import ctypes as C

import pytest
import torch

import infer_b200 as B
from tests.test_kv4_contract import A, ASSIGN, RELEASE, append_desc, attention_desc, cache, gather_desc, refused, rope_desc


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (3, 1), (16, 1)])
def test_a_larger_step_never_needs_a_smaller_workspace(dim, q_heads, kv_heads):
    need = [B.lib().fth_b200_kv4_attention_workspace_bytes(C.byref(attention_desc(dict(head_dim=dim, kv_heads=kv_heads), q_heads=q_heads, max_query=n)))
            for n in range(1, 300)]
    assert need[0] > 0 and need == sorted(need)


def test_builders_refuse_rows_that_a_tensor_does_not_hold():
    """One-dimensional tensors, strides given by hand, rows that repeat (stride 0): the last row has to lie inside the tensor."""
    bf16 = dict(dtype=torch.bfloat16)
    x = torch.zeros((4, 4, 128), **bf16)
    for bad in (torch.zeros(8, **bf16), torch.zeros(4 * 512 - 1, **bf16), torch.zeros((1, 128), **bf16).expand(16, 128).flatten()[:100]):
        with pytest.raises(ValueError, match="elements"):
            rope_desc(q=bad, q_out=x)
    with pytest.raises(ValueError, match="elements"):
        rope_desc(q=x, q_out=x, ldq=513)                     # three strides and a row are one element too many ...
    with pytest.raises(ValueError, match="not on a GPU"):
        rope_desc(q=torch.zeros(3 * 513 + 512, **bf16), q_out=x, ldq=513)   # ... and these hold them
    for name in ("q", "q_out", "k", "k_out"):
        with pytest.raises(ValueError, match=f"{name}: .*elements"):
            rope_desc(**{name: torch.zeros(8, **bf16), "ld" + name: 512})
    for name in ("k", "v"):
        with pytest.raises(ValueError, match=f"{name}: .*elements"):
            append_desc(**{name: torch.zeros(8, **bf16), "ld" + name: 256})
    for name in ("k", "v"):
        with pytest.raises(ValueError, match=f"{name}_out: .*elements"):
            gather_desc(**{name + "_out": torch.zeros(8, **bf16), "ld" + name: 256})
    for name, ld in (("q", "ldq"), ("out", "ldo")):
        with pytest.raises(ValueError, match=f"{name}: .*elements"):
            attention_desc(**{name: torch.zeros(8, **bf16), ld: 1024})
    with pytest.raises(ValueError, match="heads 128 apart"):
        rope_desc(q=torch.zeros((1, 4, 128), **bf16).expand(4, 4, 128), q_out=x)


def test_builders_tell_fp16_from_bf16():
    """Bits in integers are anybody's; numbers have to be of the type that the descriptor names."""
    half, bits = torch.zeros((4, 4, 128), dtype=torch.float16), torch.zeros((4, 4, 128), dtype=torch.int16)
    with pytest.raises(ValueError, match="float16"):
        rope_desc(q=half, q_out=bits)
    with pytest.raises(ValueError, match="bfloat16"):
        rope_desc(dtype=B.FP16, q=half.bfloat16(), q_out=bits)
    with pytest.raises(ValueError, match="not on a GPU"):
        rope_desc(dtype=B.FP16, q=half, q_out=bits)
    with pytest.raises(ValueError, match="not on a GPU"):
        rope_desc(q=bits, q_out=bits)


def test_a_workspace_tensor_is_as_large_as_it_is_said_to_be():
    with pytest.raises(ValueError, match="workspace has"):
        attention_desc(workspace=torch.zeros(100, dtype=torch.uint8), workspace_bytes=101)


@pytest.mark.parametrize("off", [1, 2])
def test_addresses_of_numbers_are_aligned(off):
    """A word read from an odd address would end the context."""
    for name in ("positions", "turns"):
        refused("fth_b200_rope", rope_desc(**{name: A + off}), B.ERR_INVALID)
    refused("fth_b200_rope", rope_desc(turns=A + 4), B.ERR_INVALID)
    refused("fth_b200_kv4_append", append_desc(rope=rope_desc(k_out=None, positions=A + off)), B.ERR_INVALID)
    refused("fth_b200_kv4_append", append_desc(slots=A + off), B.ERR_INVALID)
    refused("fth_b200_kv4_gather", gather_desc(slots=A + off), B.ERR_INVALID)
    for name in ("block_table", "total_lens", "query_start"):
        refused("fth_b200_kv4_attention", attention_desc(**{name: A + off}), B.ERR_INVALID)
    for name in ("cached_lens", "new_lens", "free_blocks", "free_count", "free_count_out", "block_table", "total_lens", "query_start", "slots", "positions",
                 "status"):
        refused("fth_b200_kv4_assign", B.kv4_assign_desc(**{**ASSIGN, name: A + off}), B.ERR_INVALID)
    for name in ("lens", "keep_lens", "free_blocks", "free_count", "free_count_out", "block_table", "lens_out", "status"):
        refused("fth_b200_kv4_release", B.kv4_release_desc(**{**RELEASE, name: A + off}), B.ERR_INVALID)


@pytest.mark.parametrize("block_size,max_blocks", [(16, (1 << 27) - 1), (256, (1 << 23) - 1), (16, (1 << 27) - 31)])
def test_attention_refuses_tables_whose_last_tile_passes_31_bits(block_size, max_blocks):
    d = attention_desc(dict(block_size=block_size), max_blocks=max_blocks)
    assert B.lib().fth_b200_kv4_attention_supported(C.byref(d)) == B.ERR_UNSUPPORTED
    d = attention_desc(dict(block_size=block_size), max_blocks=((1 << 31) - 512) // block_size)
    assert B.lib().fth_b200_kv4_attention_supported(C.byref(d)) == B.OK
