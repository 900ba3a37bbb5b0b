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


# ------------------------------------------------------------------ values that a row does not see
def seen_places(b):
    """(prefix positions [rows, prefix], own positions [rows, own pages * PAGE]) that each row sees, as truth values."""
    width = b.block_table.shape[1] * PAGE
    j = torch.arange(b.prefix + width, device=DEV)
    pos = b.row_pos.long()[:, None]
    seen = (j <= pos) & (b.row_seq >= 0)[:, None]
    if b.window > 0:
        seen &= j > pos - b.window
    return seen[:, :b.prefix], seen[:, b.prefix:]


SPREAD = [  # q_lens, own_lens, prefix, window, positions of the rows (None: as they are)
    ([1, 1], [1, 1], 600, 32, [40, 290]),                                    # two windows far apart in one tile of the prefix
    ([1] * 6, [200] * 6, 700, 90, [3, 200, 291, 500, 760, 899]),             # some behind the prefix
    ([2, 40], [3, 40], 500, 20, [(37 * i) % 530 for i in range(42)]),        # in no order, near the prefix' end
    ([5, 60], [70, 300], 130, 7, list(range(130, 200, 14)) + [130 + 4 * i for i in range(60)]),        # holes among own keys
    ([1, 30], [1, 90], 300, 0, [5] + list(range(290, 320)))]                 # no window: rows inside the prefix


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 16), (28, 4, 128), (8, 8, 80), (14, 2, 64), (2, 2, 20)])
@pytest.mark.parametrize("shape", range(len(SPREAD)))
def test_places_that_no_row_sees_hold_anything(dtype, heads, kv_heads, hd, shape):
    q_lens, own, prefix, window, positions = SPREAD[shape]
    b = sp.Batch(dtype, q_lens, own, prefix, heads, kv_heads, hd, window=window, seed=90 + shape)
    b.k_pool.nan_to_num_(0.5)
    b.v_pool.nan_to_num_(0.25)
    b.row_pos.copy_(torch.tensor(positions, dtype=torch.int32))
    in_prefix, in_own = seen_places(b)
    j = (~in_prefix.any(0)).nonzero().flatten()
    for pool, bad in ((b.k_pool, float("nan")), (b.v_pool, float("inf"))):
        pool[b.prefix_table.long()[j // PAGE], j % PAGE] = bad
        for s in range(len(q_lens)):
            k = (~in_own[b.row_seq == s].any(0)).nonzero().flatten()
            k = k[b.block_table[s, k // PAGE] >= 0]
            pool[b.block_table[s, k // PAGE].long(), k % PAGE] = bad
    b.check(b.run(ops), "numbers nowhere but where a row looks")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 16), (28, 4, 128), (8, 8, 80), (14, 2, 64), (2, 2, 20)])
@pytest.mark.parametrize("shape", range(len(SPREAD)))
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(dtype, heads, kv_heads, hd, shape):
    """A row's numbers depend on nothing that it does not see, whatever the rows of its tile see."""
    q_lens, own, prefix, window, positions = SPREAD[shape]
    b = sp.Batch(dtype, q_lens, own, prefix, heads, kv_heads, hd, window=window, seed=70 + shape)
    b.k_pool.nan_to_num_(0.5)
    b.v_pool.nan_to_num_(0.25)
    b.row_pos.copy_(torch.tensor(positions, dtype=torch.int32))
    clean = b.v_pool.clone()
    in_prefix, in_own = seen_places(b)
    spoilt = torch.zeros((len(b.row_pos), kv_heads, heads // kv_heads, hd), dtype=torch.bool, device=DEV)
    for n, (j, kvh, c, bad) in enumerate([(38, 0, 3, "inf"), (64, kv_heads - 1, hd - 1, "nan"), (prefix - 1, 0, 5, "-inf"), (290, 0, 2, "inf"), (127, kv_heads - 1, 4, "inf")]):
        if j < prefix:
            b.v_pool[b.prefix_table[j // PAGE].long(), j % PAGE, kvh, c] = float(bad)
            spoilt[:, kvh, :, c] |= in_prefix[:, j, None]
    for s in range(len(q_lens)):
        for k, kvh, c, bad in ((0, 0, 7, "inf"), (own[s] // 2, kv_heads - 1, 1, "nan"), (own[s] - 1, 0, 0, "inf")):
            b.v_pool[b.block_table[s, k // PAGE].long(), k % PAGE, kvh, c] = float(bad)
            spoilt[:, kvh, :, c] |= (in_own[:, k] & (b.row_seq == s))[:, None]
    out = b.run(ops)
    spoilt = spoilt.flatten(1)
    finite = out.isfinite()
    assert bool((finite == ~spoilt).all()), "%d numbers spoilt by what their row does not see, %d clean that should not be" % (
        int((~finite & ~spoilt).sum()), int((finite & spoilt).sum()))
    b.v_pool = clean                                      # (the definition without them, for all other numbers)
    b.check(torch.where(spoilt, b.reference()[0].to(dtype), out), "numbers beside")


# ------------------------------------------------------------------ steps of very unequal sequences
@pytest.mark.parametrize("dtype,heads,kv_heads,hd,window", [(BF, 28, 4, 128, 0), (BF, 4, 2, 16, 333), (F32, 14, 2, 64, 0)])
def test_a_long_prompt_beside_one_token_rows(dtype, heads, kv_heads, hd, window):
    """Most sequences have one row, one has many: most of the jobs that the longest one's tiles give the others have no rows."""
    q_lens = [1] * 20 + [1501] + [1] * 11
    b = sp.Batch(dtype, q_lens, [q + 17 * i for i, q in enumerate(q_lens)], 700, heads, kv_heads, hd, window=window, seed=31)
    b.check(b.run(ops), "a long prompt beside one-token rows")
