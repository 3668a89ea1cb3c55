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
