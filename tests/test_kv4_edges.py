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
