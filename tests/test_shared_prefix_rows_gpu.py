"""Attention of a batch with a shared prefix: a row's result is made of what that row sees alone, with weights of 32 bits."""
import copy

import pytest
import torch

import shared_prefix as sp
from friday_inference_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
PAGE = sp.PAGE


# ------------------------------------------------------------------ weights
def bound_of_32_bit_weights(b):
    """(result, bound): Batch.reference()'s bound with every sum, score and weight in 32 bits, and the result rounded once.

    A weight may enter the product as two bf16 numbers, itself rounded and what that left rounded, which leaves 2^-8 of 2^-8 of it."""
    c = copy.copy(b)
    c.dtype = F32                                         # (the bound without bf16 weights)
    ref, tol = c.reference()
    c.v_pool = b.v_pool.abs()
    around, _ = c.reference()                             # sum_j w_j |v_j|
    half = sp.HALF[b.dtype]
    return ref, (tol + around * 2.0 ** -16) * (1 + half) + half * ref.abs()


@pytest.mark.parametrize("q_lens,own_lens,prefix,heads,kv_heads,hd,window", [
    ([1] * 4, [1, 40, 17, 33], 500, 14, 2, 64, 0), ([1] * 9, [40 * i + 1 for i in range(9)], 2000, 28, 4, 128, 0), ([30, 1, 90], [30, 3, 200], 300, 28, 4, 128, 0),
    ([30, 1, 90], [30, 3, 200], 300, 8, 8, 80, 77), ([1] * 4, [1, 60, 100, 600], 333, 4, 2, 16, 300), ([1, 3], [5, 70], 130, 2, 2, 20, 0)])
def test_weights_are_not_rounded_to_bf16(q_lens, own_lens, prefix, heads, kv_heads, hd, window):
    b = sp.Batch(BF, q_lens, own_lens, prefix, heads, kv_heads, hd, window=window, seed=hd + prefix)
    ref, bound = bound_of_32_bit_weights(b)
    err = (b.run(ops).double() - ref).abs()
    assert bool((err <= bound).all()), "%d numbers off, the worst by %.3g of the bound" % (int((err > bound).sum()), float((err / bound).max()))


# ------------------------------------------------------------------ windows that reach beyond the tables
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 16), (28, 4, 128), (2, 2, 20)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [1, 3, 40, 2]])
@pytest.mark.parametrize("window", [50, 200])
def test_windows_of_rows_behind_the_tables_end(dtype, heads, kv_heads, hd, q_lens, window):
    """A window ends at its row's position, not at the end of the tables: one that lies partly behind them, and wholly."""
    own = [q + 60 for q in q_lens]
    b = sp.Batch(dtype, q_lens, own, 150, heads, kv_heads, hd, window=window, seed=window)
    b.k_pool.nan_to_num_(0.5)
    b.v_pool.nan_to_num_(0.25)
    room = b.prefix + b.block_table.shape[1] * PAGE
    b.row_pos[0] = room - 1 + window // 3                 # two thirds of its window
    b.row_pos[1] = room - 2 + window                      # the last position alone
    b.row_pos[2] = room - 1 + window                      # nothing
    b.row_pos[-1] = 2000000000
    out = b.run(ops)
    nothing = torch.zeros(len(b.row_pos), dtype=torch.bool, device=DEV)
    nothing[2] = nothing[-1] = True
    assert bool((out[nothing] == 0).all()), "rows that see nothing"
    c = copy.copy(b)                                      # (the definition, for the others)
    c.row_seq = torch.where(nothing, -1, b.row_seq)
    c.check(torch.where(nothing[:, None], 7.25, out.float()).to(dtype), "windows behind the tables' end")
