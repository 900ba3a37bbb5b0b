"""Rotary positions with several axes, their append to the paged cache, attention of a batch with a shared prefix: against their
definitions in 64-bit, at the sizes, masks and layouts where each can go wrong, and as they are used one after another."""
import ctypes
import threading

import pytest
import torch

import shared_prefix as sp
from friday_inference_engine_b200 import native, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
PAGE = sp.PAGE


def rnd(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def ladder(pairs, theta=10000.0):
    return (theta ** (torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(DEV)


def within(got, ref, err, dtype, what):
    bound = sp.HALF[dtype] * ref.abs() + err * (1 + sp.HALF[dtype]) + 1e-37
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bool(bad.any()), "%s: %d numbers off, the worst by %.3g" % (what, int(bad.sum()), float(((got.double() - ref).abs() / bound).max()))


# ------------------------------------------------------------------ rotation
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,heads,hd,sections,interleaved,neighbours", [
    (1, 1, 2, [1], False, False), (5, 3, 20, [3, 2], False, False), (7, 2, 80, [20, 20], False, False), (33, 32, 80, [20, 20], False, True),
    (1, 28, 128, [16, 24, 24], False, False), (300, 4, 128, [24, 20, 20], True, False), (65, 6, 72, [18, 18], False, False),
    (9, 5, 256, [128], False, False), (9, 5, 256, [64, 32, 32], True, True), (17, 3, 64, [4, 6, 6], False, False),      # dimensions that stay
    (17, 3, 64, [6, 5, 5], True, True), (13, 2, 33, [5, 4, 4], False, False), (4, 7, 16, [2, 2, 2, 2], True, False), (3, 2, 64, [0, 16, 16], False, False)])
def test_rotation(dtype, rows, heads, hd, sections, interleaved, neighbours):
    x = rnd((rows, heads * hd), dtype, 1)
    pos = torch.randint(-50, 40000, (rows, len(sections)), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(DEV)
    denom = ladder(sum(sections), 1e6)
    keep = x.clone()
    out = ops.rotate_axes(x, pos, denom, sections, heads, hd, interleaved=interleaved, neighbours=neighbours)
    ref, err = sp.turned(x.double().view(rows, heads, hd), pos, denom, sections, interleaved, neighbours)
    within(out, ref.flatten(1), err.flatten(1), dtype, "rotation")
    assert torch.equal(x, keep)
    half = sum(sections)
    assert torch.equal(out.view(rows, heads, hd)[..., 2 * half:], x.view(rows, heads, hd)[..., 2 * half:])          # what does not turn stays
    assert ops.rotate_axes(x, pos, denom, sections, heads, hd, interleaved=interleaved, neighbours=neighbours, out=x) is x     # in place
    assert torch.equal(x, out)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rotation_of_columns_of_wider_rows(dtype, offset):
    """Row strides and starts that are no multiple of 16 bytes; columns beside the heads stay; a result in the same rows."""
    rows, heads, hd, sections = 21, 4, 48, [12, 12]
    wide = rnd((rows, offset + 3 * heads * hd + 5), dtype, 3)
    x = wide[:, offset:offset + heads * hd]
    pos = torch.arange(2 * rows, dtype=torch.int32, device=DEV).view(rows, 2)
    denom = ladder(24)
    keep = wide.clone()
    ref, err = sp.turned(x.double().reshape(rows, heads, hd), pos, denom, sections)
    beside = wide[:, offset + heads * hd:offset + 2 * heads * hd]
    ops.rotate_axes(x, pos, denom, sections, heads, hd, out=beside)
    within(beside, ref.flatten(1), err.flatten(1), dtype, "into columns beside")
    assert torch.equal(wide[:, :offset + heads * hd], keep[:, :offset + heads * hd]) and torch.equal(wide[:, offset + 2 * heads * hd:], keep[:, offset + 2 * heads * hd:])
    ops.rotate_axes(x, pos, denom, sections, heads, hd, out=x)
    within(x, ref.flatten(1), err.flatten(1), dtype, "in place")
    ops.rotate_axes(wide, pos, denom, sections, heads, hd, out=torch.empty((rows, heads * hd), dtype=dtype, device=DEV))     # more columns than heads


def test_rotation_at_far_positions():
    """Angles of positions that 32-bit floats cannot hold, and negative ones."""
    sections, hd = [16, 24, 24], 128
    pos = torch.tensor([[0, 1, -1], [1 << 24, (1 << 24) + 1, 1 << 30], [2147483647, -2147483648, 999999937]], dtype=torch.int32, device=DEV)
    x, denom = rnd((3, 2 * hd), F32, 4), ladder(64, 1e6)
    out = ops.rotate_axes(x, pos, denom, sections, 2, hd)
    ref, err = sp.turned(x.double().view(3, 2, hd), pos, denom, sections)
    within(out, ref.flatten(1), err.flatten(1), F32, "far positions")


def test_rotation_of_many_rows():
    rows, heads, hd, sections = 40001, 5, 80, [20, 20]
    x = rnd((rows, heads * hd), BF, 5)
    pos = torch.randint(0, 3000, (rows, 2), generator=torch.Generator().manual_seed(6), dtype=torch.int32).to(DEV)
    out = ops.rotate_axes(x, pos, ladder(40), sections, heads, hd)
    ref, err = sp.turned(x.double().view(rows, heads, hd), pos, ladder(40), sections)
    within(out, ref.flatten(1), err.flatten(1), BF, "many rows")
    assert ops.rotate_axes(x[:0], pos[:0], ladder(40), sections, heads, hd).shape == (0, heads * hd)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,heads,hd,sections,interleaved,neighbours,beside", [
    (3001, 24, 72, [18, 18], False, False, 0), (2500, 24, 72, [16, 12, 8], True, True, 8), (9000, 8, 36, [9, 9], False, False, 0), (9000, 8, 36, [9, 9], False, True, 16),
    (4099, 12, 64, [8, 4, 4], False, False, 0), (1500, 6, 256, [48, 40, 40], True, False, 0), (70000, 1, 32, [16], False, False, 0), (60000, 1, 40, [6, 7], False, True, 0),
    (700, 40, 128, [24, 20, 20], False, False, 24)])
def test_rotation_of_rows_by_the_megabyte(dtype, rows, heads, hd, sections, interleaved, neighbours, beside):
    x = rnd((rows, (heads * hd + beside)), dtype, 45)
    keep = x.clone()
    pos = torch.randint(0, 9000, (rows, len(sections)), generator=torch.Generator().manual_seed(46), dtype=torch.int32).to(DEV)
    denom = ladder(sum(sections))
    out = ops.rotate_axes(x, pos, denom, sections, heads, hd, interleaved=interleaved, neighbours=neighbours)
    ref, err = sp.turned(x[:, :heads * hd].double().reshape(rows, heads, hd), pos, denom, sections, interleaved, neighbours)
    within(out, ref.flatten(1), err.flatten(1), dtype, "many rows")
    half = sum(sections)
    assert torch.equal(out.view(rows, heads, hd)[..., 2 * half:], keep[:, :heads * hd].reshape(rows, heads, hd)[..., 2 * half:])
    ops.rotate_axes(x[:, :heads * hd], pos, denom, sections, heads, hd, interleaved=interleaved, neighbours=neighbours, out=x[:, :heads * hd])
    assert torch.equal(x[:, :heads * hd], out) and torch.equal(x[:, heads * hd:], keep[:, heads * hd:])


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("nq,nkv,hd,sections,neighbours,beside", [(28, 4, 128, [16, 24, 24], False, 0), (3, 1, 32, [4, 4], True, 8), (8, 8, 72, [12, 12, 12], False, 0), (0, 2, 64, [16], False, 0)])
def test_append_of_rows_by_the_megabyte(dtype, nq, nkv, hd, sections, neighbours, beside):
    """Rows without a sequence, places that no page has, and pages in any order among many rows."""
    width = (nq + 2 * nkv) * hd
    rows = (3 << 20) // (width * 2) + 37
    pages = rows // PAGE + 9
    wide = rnd((rows, width + beside), dtype, 47)
    qkv = wide[:, :width]
    g = torch.Generator().manual_seed(48)
    table = torch.randperm(pages, generator=g)[:pages // 2 * 2].to(torch.int32).view(2, -1).contiguous()
    order = torch.randperm(2 * table.shape[1] * PAGE, generator=g)[:rows]
    seq, place = (order % 2).to(torch.int32), (order // 2).to(torch.int32)
    seq[5::97] = -1
    place[7::101] = table.shape[1] * PAGE + 3
    table[1, 1] = -1
    seq, place, table = seq.to(DEV), place.to(DEV), table.to(DEV)
    pos = torch.randint(0, 9000, (rows, len(sections)), generator=g, dtype=torch.int32).to(DEV)
    denom = ladder(sum(sections))
    kp = torch.full((pages, PAGE, nkv, hd), 3.0, dtype=dtype, device=DEV)
    vp = kp.clone()
    q = torch.full((rows, nq * hd), 9.0, dtype=dtype, device=DEV)
    ops.rope_axes_kv_write(qkv, seq, place, pos, denom, sections, nq, nkv, hd, kp, vp, table, PAGE, neighbours=neighbours, q_out=q)
    heads = qkv.double().reshape(rows, nq + 2 * nkv, hd)
    ref, err = sp.turned(heads[:, :nq + nkv], pos, denom, sections, False, neighbours)
    live = seq >= 0
    if nq:
        within(q[live], ref[live][:, :nq].flatten(1), err[live][:, :nq].flatten(1), dtype, "queries")
        assert bool((q[~live] == 9.0).all())
    page = torch.where(live & (place < table.shape[1] * PAGE), table[seq.clamp(min=0).long(), (place // PAGE).clamp(max=table.shape[1] - 1).long()], -1)
    kept = page >= 0
    flat = (page.long() * PAGE + place.long() % PAGE)[kept]
    within(kp.flatten(0, 1)[flat].flatten(1), ref[kept][:, nq:].flatten(1), err[kept][:, nq:].flatten(1), dtype, "keys")
    assert torch.equal(vp.flatten(0, 1)[flat], qkv.reshape(rows, -1, hd)[kept][:, nq + nkv:])
    others = torch.ones(pages * PAGE, dtype=torch.bool, device=DEV)
    others[flat] = False
    assert bool((kp.flatten(0, 1)[others] == 3.0).all()) and bool((vp.flatten(0, 1)[others] == 3.0).all())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("nq,nkv,hd,sections,interleaved,neighbours", [
    (5, 2, 48, [8, 8, 8], False, False), (28, 4, 128, [16, 24, 24], False, False), (40, 8, 128, [24, 20, 20], True, False),
    (3, 1, 32, [4, 4], False, True), (0, 3, 20, [5, 5], False, False), (2, 2, 33, [7], False, False), (4, 4, 72, [10, 8], False, True)])
def test_append(dtype, nq, nkv, hd, sections, interleaved, neighbours):
    rows = 12
    qkv = rnd((rows, (nq + 2 * nkv) * hd), dtype, 7)
    keep = qkv.clone()
    row_seq = torch.tensor([0, 0, 0, 1, 1, -1, 1, 0, 0, 0, 1, 2], dtype=torch.int32, device=DEV)
    row_pos = torch.tensor([62, 63, 64, 0, 1, 0, 2, 65, 127, 200, 64, 5], dtype=torch.int32, device=DEV)       # 1 at 64: a page that it does not hold
    table = torch.tensor([[3, 1, 7, 5], [2, -1, -1, -1], [8, 8, 8, 8]], dtype=torch.int32, device=DEV)         # 2: pages beyond the pool
    pos = torch.randint(0, 5000, (rows, len(sections)), generator=torch.Generator().manual_seed(8), dtype=torch.int32).to(DEV)
    denom = ladder(sum(sections))
    kp = torch.full((8, PAGE, nkv, hd), 3.0, dtype=dtype, device=DEV)
    vp = kp.clone()
    q = torch.full((rows, nq * hd), 9.0, dtype=dtype, device=DEV)
    got = ops.rope_axes_kv_write(qkv, row_seq, row_pos, pos, denom, sections, nq, nkv, hd, kp, vp, table, PAGE, interleaved=interleaved,
                                 neighbours=neighbours, q_out=q)
    assert got is q and torch.equal(qkv, keep)
    heads = qkv.double().view(rows, nq + 2 * nkv, hd)
    ref, err = sp.turned(heads[:, :nq + nkv], pos, denom, sections, interleaved, neighbours)
    live = row_seq >= 0
    if nq:
        within(q[live], ref[live][:, :nq].flatten(1), err[live][:, :nq].flatten(1), dtype, "queries")
        assert bool((q[~live] == 9.0).all())
    written = torch.zeros((8, PAGE), dtype=torch.bool, device=DEV)
    for r in range(rows):
        seq, place = int(row_seq[r]), int(row_pos[r])
        page = int(table[seq, place // PAGE]) if seq >= 0 else -1
        if page < 0 or page >= 8:
            continue
        within(kp[page, place % PAGE], ref[r, nq:], err[r, nq:], dtype, "keys")
        assert torch.equal(vp[page, place % PAGE], qkv[r].view(-1, hd)[nq + nkv:])
        written[page, place % PAGE] = True
    assert int(written.sum()) == 9
    assert bool((kp[~written] == 3.0).all()) and bool((vp[~written] == 3.0).all())
    if nq:              # the queries in their own columns
        ops.rope_axes_kv_write(qkv, row_seq, row_pos, pos, denom, sections, nq, nkv, hd, kp, vp, table, PAGE, interleaved=interleaved,
                               neighbours=neighbours, q_out=qkv[:, :nq * hd])
        assert torch.equal(qkv[live][:, :nq * hd], q[live]) and torch.equal(qkv[:, nq * hd:], keep[:, nq * hd:]) and torch.equal(qkv[~live], keep[~live])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_append_with_equal_positions_agrees_with_the_one_axis_rotation(dtype):
    """Text: all axes have the token's position, which is also its place."""
    nq, nkv, hd, rows = 6, 2, 64, 70
    qkv = rnd((rows, (nq + 2 * nkv) * hd), dtype, 9)
    row_seq = torch.zeros(rows, dtype=torch.int32, device=DEV)
    row_pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    kp, vp = (torch.zeros((2, PAGE, nkv, hd), dtype=dtype, device=DEV) for _ in range(2))
    kp2, vp2 = kp.clone(), vp.clone()
    denom = ladder(32)
    q = ops.rope_axes_kv_write(qkv, row_seq, row_pos, row_pos[:, None].expand(-1, 3).contiguous(), denom, [8, 12, 12], nq, nkv, hd, kp, vp, table, PAGE)
    ops.rope_kv_write(qkv, row_seq, row_pos, denom, hd, nq, nkv, hd, kp2, vp2, table, PAGE)
    step = 2 * sp.HALF[dtype]                              # both are rounded once; their angles differ by parts of 2^-24 * 70
    for a, b in ((q, qkv[:, :nq * hd]), (kp, kp2)):
        assert bool(((a.double() - b.double()).abs() <= step * b.double().abs() + 70 * 2.0 ** -22).all())
    assert torch.equal(vp, vp2)


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_append_between_tensors_side_by_side_in_memory(rows):
    """Rows and turned queries that touch, and turned queries in columns behind the rows' own, are not on one another."""
    nq, nkv, hd = 6, 2, 32
    width = (nq + 2 * nkv) * hd
    buf = rnd((rows * (width + nq * hd),), BF, 44)
    seq, place = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.arange(rows, dtype=torch.int32, device=DEV)
    pos = torch.stack((place + 3, place), 1).contiguous()
    kp, vp = (torch.zeros((2, PAGE, nkv, hd), dtype=BF, device=DEV) for _ in range(2))
    args = (seq, place, pos, ladder(16), [8, 8], nq, nkv, hd, kp, vp, torch.tensor([[1]], dtype=torch.int32, device=DEV), PAGE)
    apart, touching = buf[:rows * width].view(rows, width), buf[rows * width:].view(rows, nq * hd)
    want = ops.rope_axes_kv_write(apart.clone(), *args)
    assert torch.equal(ops.rope_axes_kv_write(apart, *args, q_out=touching), want)
    wide = torch.cat((apart, torch.zeros((rows, nq * hd), dtype=BF, device=DEV)), 1)
    assert torch.equal(ops.rope_axes_kv_write(wide[:, :width], *args, q_out=wide[:, width:]), want)


def test_append_of_many_rows_far_into_a_large_pool():
    """Places whose element numbers pass 2^31."""
    nq, nkv, hd, pages = 2, 8, 128, 33000
    kp = torch.empty((pages, PAGE, nkv, hd), dtype=BF, device=DEV)                     # 2.16e9 numbers
    vp = torch.empty_like(kp)
    rows = 3000
    table = torch.arange(pages - 1, pages - 48, -1, dtype=torch.int32, device=DEV).view(1, -1)
    qkv = rnd((rows, (nq + 2 * nkv) * hd), BF, 10)
    seq, place = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.arange(rows, dtype=torch.int32, device=DEV)
    pos = torch.stack((place, place // 7, place % 7), 1).contiguous()
    q = ops.rope_axes_kv_write(qkv, seq, place, pos, ladder(64), [16, 24, 24], nq, nkv, hd, kp, vp, table, PAGE)
    ref, err = sp.turned(qkv.double().view(rows, -1, hd)[:, :nq + nkv], pos, ladder(64), [16, 24, 24])
    within(q, ref[:, :nq].flatten(1), err[:, :nq].flatten(1), BF, "queries")
    flat = table[0, (place // PAGE).long()].long() * PAGE + (place % PAGE).long()
    within(kp.flatten(0, 1)[flat], ref[:, nq:], err[:, nq:], BF, "keys")
    assert torch.equal(vp.flatten(0, 1)[flat], qkv.view(rows, -1, hd)[:, nq + nkv:])


# ------------------------------------------------------------------ attention
LAYOUTS = [(4, 2, 16), (3, 1, 32), (28, 4, 128), (6, 2, 48), (8, 8, 80), (14, 2, 64), (16, 2, 112)]
OTHER_LAYOUTS = [(2, 2, 20), (5, 5, 256), (4, 1, 160), (1, 1, 1)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS + OTHER_LAYOUTS)
def test_one_token_steps(dtype, heads, kv_heads, hd):
    b = sp.Batch(dtype, [1] * 5, [1, 64, 65, 130, 7], 301, heads, kv_heads, hd, seed=hd)
    b.check(b.run(ops), "one-token step")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127, 128, 129, 1000])
def test_prefixes_that_end_anywhere(dtype, prefix):
    b = sp.Batch(dtype, [1, 3, 1, 2], [1, 3, 128, 66], prefix, 14, 2, 64, seed=prefix, wider=2)
    b.check(b.run(ops), "prefix of %d" % prefix)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 16), (28, 4, 128), (8, 8, 80), (14, 2, 64), (2, 2, 20)])
@pytest.mark.parametrize("window", [0, 5, 90, 400])
def test_prompts_of_unequal_lengths(dtype, heads, kv_heads, hd, window):
    b = sp.Batch(dtype, [37, 1, 100, 64, 5], [37, 1, 150, 64, 261], 200, heads, kv_heads, hd, window=window, seed=hd + window)
    b.check(b.run(ops), "prompts, window %d" % window)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("window", [1, 63, 64, 100, 128, 700])
def test_windows_of_one_token_steps(dtype, window):
    b = sp.Batch(dtype, [1] * 4, [1, 60, 100, 600], 333, 28, 4, 128, window=window, seed=window)
    b.check(b.run(ops), "window %d" % window)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_long_prefix_of_many_sequences(dtype):
    b = sp.Batch(dtype, [1] * 40, [17 * i % 200 + 1 for i in range(40)], 5003, 14, 2, 64, seed=3)
    b.check(b.run(ops), "long prefix")


def test_long_prefix_at_the_7b_shape():
    b = sp.Batch(BF, [1] * 33, [29 * i % 300 + 1 for i in range(33)], 9001, 28, 4, 128, seed=4)
    b.check(b.run(ops), "decode")
    b = sp.Batch(BF, [200, 1, 90], [230, 3, 90], 3003, 28, 4, 128, seed=5)
    b.check(b.run(ops), "prompts")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (40, 1), (64, 1), (128, 1), (129, 1), (100, 2)])
def test_many_heads_on_one_kv_head(dtype, heads, kv_heads):
    b = sp.Batch(dtype, [1, 2, 1], [5, 70, 1], 150, heads, kv_heads, 64, seed=heads)
    b.check(b.run(ops), "%d heads on %d" % (heads, kv_heads))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("page", [1, 16, 48, 96])
def test_pages_of_other_sizes(dtype, page):
    b = sp.Batch(dtype, [1, 3, 1], [1, 70, 200], 130, 14, 2, 64, seed=page, page=page)
    b.check(b.run(ops), "pages of %d" % page)
    b = sp.Batch(dtype, [1, 30, 1], [1, 70, 20], 90, 4, 2, 16, window=50, seed=page, page=page)
    b.check(b.run(ops), "pages of %d, a window" % page)


@pytest.mark.parametrize("window", [0, 300])
def test_more_jobs_than_the_device_takes_at_once(window):
    """A CTA takes several shares one after another: of unequal lengths, some without keys, some without rows."""
    lens = [(37 * i * i) % 700 + 1 for i in range(100)]
    b = sp.Batch(BF, [1] * 100, lens, 2500, 28, 4, 128, window=window, seed=50)
    b.row_seq[7::13] = -1
    b.row_pos[3::17] = 100                 # inside the prefix: nothing of their own
    b.check(b.run(ops), "a hundred sequences")
    first = b.run(ops).clone()
    for _ in range(10):
        b.out.fill_(7.25)
        assert torch.equal(b.run(ops), first)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 16), (28, 4, 128), (14, 2, 64), (8, 8, 80), (70, 70, 32), (12, 4, 96)])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 7])
def test_few_sequences(dtype, heads, kv_heads, hd, n):
    """One token each, and two for some; rows without a sequence, rows that
    see nothing, windows, the same bits every time."""
    b = sp.Batch(dtype, [1] * n, [33 * i + 1 for i in range(n)], 500, heads, kv_heads, hd, seed=60 + n)
    b.check(b.run(ops), "%d sequences" % n)
    first = b.run(ops).clone()
    for _ in range(5):
        b.out.fill_(7.25)
        assert torch.equal(b.run(ops), first)
    b = sp.Batch(dtype, [1 + i % 2 for i in range(n)], [70 * i + 2 for i in range(n)], 129, heads, kv_heads, hd, window=150, seed=70 + n)
    b.check(b.run(ops), "%d sequences, a window" % n)
    b.row_seq[0] = -1
    b.row_pos[-1] = -1
    b.out.fill_(7.25)
    b.check(b.run(ops), "%d sequences, rows left out" % n)


def test_hundreds_of_sequences():
    b = sp.Batch(BF, [1] * 333, [i % 90 + 1 for i in range(333)], 400, 6, 3, 16, seed=51)
    b.check(b.run(ops), "hundreds of sequences")
    b = sp.Batch(BF, [1 + i % 3 for i in range(250)], [3 + i % 70 for i in range(250)], 65, 8, 8, 32, seed=52)
    b.check(b.run(ops), "hundreds of short ones")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,hd", [(28, 4, 128), (14, 2, 64), (2, 2, 20)])
def test_a_prefix_that_is_still_being_filled(dtype, heads, kv_heads, hd):
    """Rows inside the prefix, behind which the prefix' pages hold no numbers yet."""
    for q_lens in ([1, 1, 1], [5, 40, 1]):
        b = sp.Batch(dtype, q_lens, [q + 3 for q in q_lens], 300, heads, kv_heads, hd, seed=53)
        far = 205
        b.row_pos.copy_(torch.arange(len(b.row_pos), device=DEV) * 4 % far)
        b.row_pos[0] = far
        flat = torch.arange(far + 1, 300, device=DEV)
        for pool in (b.k_pool, b.v_pool):
            pool[b.prefix_table.long()[flat // PAGE], flat % PAGE] = float("nan")
        b.check(b.run(ops), "half a prefix")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_that_see_nothing_rows_without_a_sequence_and_pages_left_out(dtype):
    b = sp.Batch(dtype, [1, 4, 1, 3, 1], [30, 10, 1, 200, 64], 140, 14, 2, 64, seed=6)
    b.row_seq[0] = -1
    b.row_seq[5] = -1
    b.row_pos[2] = -1                      # sees nothing: zeros
    b.row_pos[3] = 70                      # inside the prefix
    b.row_pos[9] = 139                     # the whole prefix and nothing of its own
    b.block_table[3, 1] = -1
    b.block_table[3, 2] = b.k_pool.shape[0] + 5
    b.prefix_table[1] = -1
    out = b.run(ops)
    b.check(out, "left out")
    assert bool((out[2] == 0).all())
    b.prefix_table[1] = 1 << 30
    b.out.fill_(7.25)
    b.check(b.run(ops), "beyond the pool")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_positions_beyond_the_tables_see_what_there_is(dtype):
    b = sp.Batch(dtype, [1, 2], [64, 128], 70, 4, 2, 16, seed=7)
    b.row_pos[0] = 2000000000
    b.block_table[0, 1] = 0
    b.k_pool.nan_to_num_(0.5)
    b.v_pool.nan_to_num_(0.25)
    b.check(b.run(ops), "far position")


def test_without_pages_of_their_own():
    b = sp.Batch(BF, [1, 1], [1, 1], 300, 28, 4, 128, seed=8)
    b.block_table = b.block_table[:, :0].contiguous()
    b.row_pos.fill_(299)
    b.check(b.run(ops), "prefix alone")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("beside", [8, 3])
def test_queries_within_wider_rows(dtype, beside):
    for q_lens, own in ([1, 1, 1], [4, 90, 1]), ([40, 3], [60, 3]):
        b = sp.Batch(dtype, q_lens, own, 129, 14, 2, 64, seed=beside, beside=beside)
        b.check(b.run(ops), "queries beside other columns")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_scores_far_apart(dtype):
    """A softmax whose maximum lies in one part alone, below it by more than an exponential reaches elsewhere; infinite scores."""
    for spread in (30.0, 300.0):
        b = sp.Batch(dtype, [1, 5, 1], [70, 5, 300], 500, 14, 2, 64, seed=9, spread=spread)
        b.check(b.run(ops), "spread %g" % spread)
    b = sp.Batch(dtype, [1, 1], [10, 80], 200, 4, 2, 16, seed=10)
    b.q[0, :16] = float("nan")                            # one head of one row: nothing else is touched
    out = b.run(ops)
    assert bool(out[0, :16].isnan().all())
    b.q[0, :16] = 0.0
    clean = torch.empty_like(out)
    b.run(ops, clean)
    assert torch.equal(out[:, 16:], clean[:, 16:])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("most_rows,most_keys", [(1 << 30, 2), (2147483647, 2147483647), (7, 1)])
def test_bounds_far_from_what_there_is(dtype, most_rows, most_keys):
    """A bound on a sequence's rows far above the step's, bounds on the positions above and below them: the same results."""
    b = sp.Batch(dtype, [1, 3, 7, 1], [1, 200, 90, 65], 300, 14, 2, 64, seed=49)
    b.geometry.max_q_len, b.geometry.max_kv_len = most_rows, most_keys
    b.check(b.run(ops), "bounds")


def test_same_bits_every_time():
    for dtype in (F32, BF):
        b = sp.Batch(dtype, [1] * 9 + [30], [40 * i + 1 for i in range(9)] + [90], 2000, 28, 4, 128, seed=11)
        first = b.run(ops).clone()
        for _ in range(5):
            b.out.fill_(7.25)
            assert torch.equal(b.run(ops), first)


def test_a_pool_whose_offsets_pass_32_bits():
    b = sp.Batch(BF, [1, 1, 20], [70, 1, 20], 700, 40, 8, 128, seed=12)
    pages = 33000
    shift = pages - b.k_pool.shape[0]
    big_k = torch.empty((pages, PAGE, 8, 128), dtype=BF, device=DEV)
    big_v = torch.empty_like(big_k)
    big_k[shift:], big_v[shift:] = b.k_pool, b.v_pool
    want = b.run(ops).clone()
    b.k_pool, b.v_pool = big_k, big_v
    b.prefix_table += shift
    b.block_table += shift * (b.block_table >= 0)
    b.out.zero_()
    assert torch.equal(b.run(ops), want)


# ------------------------------------------------------------------ streams, graphs, threads
def test_on_a_stream_of_its_own_and_captured():
    side = torch.cuda.Stream()
    b = sp.Batch(BF, [1] * 6, [20, 1, 77, 130, 64, 2], 900, 28, 4, 128, seed=13)
    want = b.run(ops).clone()
    x = rnd((50, 256), BF, 14)
    pos = torch.arange(100, dtype=torch.int32, device=DEV).view(50, 2)
    denom = ladder(64)
    want_x = ops.rotate_axes(x, pos, denom, [32, 32], 2, 128)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty_like(want)
        b.run(ops, out)
        got_x = ops.rotate_axes(x, pos, denom, [32, 32], 2, 128)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(got_x, want_x)
    graphs, outs = [], []
    for _ in range(2):                                    # two graphs of the same call: each has scratch of its own
        g = torch.cuda.CUDAGraph()
        o = torch.zeros_like(want)
        with torch.cuda.graph(g):
            b.run(ops, o)
            y = ops.rotate_axes(x, pos, denom, [32, 32], 2, 128)
        graphs.append(g)
        outs.append((o, y))
    # other calls, larger ones too, between capture and replay
    big = sp.Batch(BF, [1] * 30, [300] * 30, 2000, 28, 4, 128, seed=15)
    big.run(ops)
    b.q.mul_(0.5)
    b.row_pos[1] += 0
    b.out.fill_(7.25)
    want2 = b.run(ops).clone()
    assert not torch.equal(want2, want)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, y in outs:
            assert torch.equal(o, want2) and torch.equal(y, want_x)
            o.zero_()
    b.check(want2, "after the graphs")


def test_positions_that_move_between_replays():
    """What a captured step reads from the device may change: the rows' positions grow."""
    b = sp.Batch(BF, [1, 1, 1], [200, 130, 70], 333, 14, 2, 64, seed=16)
    last = b.row_pos.clone()
    b.row_pos -= 60
    out = torch.zeros_like(b.out)
    g = torch.cuda.CUDAGraph()
    b.run(ops)
    with torch.cuda.graph(g):
        b.run(ops, out)
    for back in (60, 30, 1, 0):
        b.row_pos.copy_(last - back)
        g.replay()
        b.check(out, "replayed, %d before the end" % back)


def test_calls_from_several_threads():
    batches = [sp.Batch(BF if i % 2 else F32, [1] * (3 + i), [50 * (i + 1)] * (3 + i), 700 + 100 * i, 14, 2, 64, seed=20 + i) for i in range(4)]
    want = [b.run(ops).clone() for b in batches]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = torch.empty_like(want[i])
            for _ in range(50):
                out.zero_()
                batches[i].run(ops, out)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------ all of them, as they are used
@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_document_and_questions_to_it(dtype):
    """A prefix goes into the cache, then questions of unequal lengths behind it, then one-token steps: every row's attention is that
    of its sequence alone, written and read by the operators of one position per token."""
    nq, nkv, hd, prefix, sections = 14, 2, 64, 150, [8, 12, 12]
    asks, steps = [5, 70, 1], 3
    denom = ladder(32)
    n = len(asks)
    g = torch.Generator().manual_seed(30)
    total = [prefix + a + steps for a in asks]
    rows_of = [torch.randn((t, (nq + 2 * nkv) * hd), generator=g).to(dtype).to(DEV) for t in total]
    for r in rows_of[1:]:
        r[:prefix] = rows_of[0][:prefix]
    places = [torch.arange(t, dtype=torch.int32, device=DEV) for t in total]
    positions = [torch.stack((p // 12, p % 12, p % 5), 1).contiguous() for p in places]
    # each sequence alone: its own pages for everything, the plain definition of both operators
    def alone(s):
        q, _ = sp.turned(rows_of[s].double().view(-1, nq + 2 * nkv, hd)[:, :nq + nkv], positions[s], denom, sections)
        return q
    pages = 40
    kp, vp = (torch.full((pages, PAGE, nkv, hd), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    prefix_table = torch.tensor([7, 3, 11], dtype=torch.int32, device=DEV)
    own_table = torch.tensor([[20, 21], [2, 30], [25, 0]], dtype=torch.int32, device=DEV)
    zeros = torch.zeros(prefix, dtype=torch.int32, device=DEV)
    ops.rope_axes_kv_write(rows_of[0][:prefix], zeros, places[0][:prefix], positions[0][:prefix].contiguous(), denom, sections, nq, nkv, hd, kp, vp,
                           prefix_table.view(1, -1), PAGE)

    def step(begin, counts):
        """The next counts[s] tokens of every sequence (begin: how many it has behind the prefix)."""
        idx = [slice(prefix + b, prefix + b + c) for b, c in zip(begin, counts)]
        qkv = torch.cat([r[i] for r, i in zip(rows_of, idx)])
        seq = torch.tensor([s for s, c in enumerate(counts) for _ in range(c)], dtype=torch.int32, device=DEV)
        place = torch.cat([p[i] for p, i in zip(places, idx)])
        pos = torch.cat([p[i] for p, i in zip(positions, idx)]).contiguous()
        q = ops.rope_axes_kv_write(qkv, seq, place - prefix, pos, denom, sections, nq, nkv, hd, kp, vp, own_table, PAGE)
        b = sp.Batch.__new__(sp.Batch)
        b.dtype, b.heads, b.kv_heads, b.hd, b.window, b.prefix, b.device = dtype, nq, nkv, hd, 0, prefix, DEV
        b.page, b.k_pool, b.v_pool, b.prefix_table, b.block_table, b.q, b.wide = PAGE, kp, vp, prefix_table, own_table, q, q
        b.row_seq, b.row_pos, b.scale = seq, place, hd ** -0.5
        b.geometry = sp.Geometry([sum(counts[:s]) for s in range(n)], counts, prefix + max(b0 + c for b0, c in zip(begin, counts)), DEV)
        b.out = torch.full((len(seq), nq * hd), 7.25, dtype=dtype, device=DEV)
        b.check(b.run(ops), "step of %s tokens" % (counts,))
        # the same keys in the sequence's own pages, read by attention()
        for s in range(n):
            length = prefix + begin[s] + counts[s]
            count = -(-length // PAGE)
            k1, v1 = (torch.zeros((count, PAGE, nkv, hd), dtype=dtype, device=DEV) for _ in range(2))
            for pool, mine in ((kp, k1), (vp, v1)):
                flat = torch.cat((pool[prefix_table.long()].flatten(0, 1)[:prefix], pool[own_table[s].long()].flatten(0, 1)[:length - prefix]))
                mine.flatten(0, 1)[:length] = flat
            here = (seq == s).nonzero().flatten()
            geo = sp.Geometry([0], [counts[s]], length, DEV)
            geo.seq_pos0 = torch.tensor([length - counts[s]], dtype=torch.int32, device=DEV)
            one = torch.empty((counts[s], nq * hd), dtype=dtype, device=DEV)
            ops.attention(q[here].contiguous(), nq * hd, one, k1, v1, torch.arange(count, dtype=torch.int32, device=DEV).view(1, -1), PAGE,
                          torch.zeros(counts[s], dtype=torch.int32, device=DEV), place[here].contiguous(), nq, nkv, hd, 0, hd ** -0.5, geo)
            ref, tol = b.reference()
            assert bool(((one.double() - b.out[here].double()).abs() <= 2 * tol[here]).all())
        return q

    q = step([0] * n, asks)
    want = torch.cat([alone(s)[prefix:prefix + asks[s], :nq] for s in range(n)]).flatten(1)
    assert bool(((q.double() - want).abs() <= 2 * sp.HALF[dtype] * want.abs() + 1e-5).all())
    for t in range(steps):
        step([a + t for a in asks], [1] * n)


# ------------------------------------------------------------------ refusals
def test_rows_without_an_address_are_refused():
    lib, backend = native.lib(), ops.backend()
    P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
    x, one = torch.zeros((2, 64), device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    ones, pool = torch.ones(32, device=DEV), torch.zeros((1, PAGE, 1, 64), device=DEV)
    at = [P(t.data_ptr()) for t in (x, one, ones, pool)]
    sections, h = (I * 1)(32), P(backend._h.value)
    rotate, append, shared = (getattr(lib, "friday_ops_" + n) for n in ("rotate_axes", "rope_axes_kv_write", "attention_shared"))
    for a, b in ((None, at[0]), (at[0], None)):
        assert rotate(h, a, L(2), L(64), L(64), b, L(2), L(64), L(64), I(0), at[1], at[2], sections, I(1), I(0), I(0), I(1), I(64), None) != 0
        assert shared(h, a, L(2), L(64), L(64), b, L(2), L(64), I(0), at[3], at[3], I(1), I(PAGE), None, I(0), at[1], I(1), I(1), at[1], at[1], at[1], at[1],
                      I(2), I(2), I(1), I(1), I(64), I(0), F(0.1), None, L(0), None) != 0
    assert append(h, None, L(2), L(192), L(192), at[0], L(2), L(64), L(64), I(0), at[1], at[1], at[1], at[2], sections, I(1), I(0), I(0), I(1), I(1),
                  I(64), at[3], at[3], I(1), I(PAGE), at[1], I(1), I(1), None) != 0
    backend.check_status()


def test_refusals():
    b = sp.Batch(BF, [1, 1], [4, 5], 70, 14, 2, 64, seed=40)
    args = dict(q=b.q, q_stride=b.wide.stride(0), out=b.out, k_pool=b.k_pool, v_pool=b.v_pool, prefix_table=b.prefix_table, prefix_len=70,
                block_table=b.block_table, page_size=PAGE, row_seq=b.row_seq, row_pos=b.row_pos, n_heads=14, n_kv_heads=2, head_dim=64,
                window=0, scale=b.scale, geometry=b.geometry)
    ops.attention_shared(**args)
    wrong = [dict(q=b.q.float()), dict(out=b.out[:, :-64]), dict(out=b.q), dict(prefix_len=-1), dict(prefix_len=129), dict(prefix_table=None),
             dict(prefix_table=b.prefix_table.long()), dict(block_table=b.block_table[:1]), dict(page_size=32), dict(row_seq=b.row_seq[:1]),
             dict(row_pos=b.row_pos.float()), dict(n_heads=13), dict(n_kv_heads=1), dict(head_dim=32), dict(scale=0.0), dict(scale=float("nan")),
             dict(scale=float("inf")), dict(window=-3), dict(q_stride=64), dict(k_pool=b.k_pool.cpu()), dict(v_pool=b.k_pool), dict(q=b.q[:, :64]),
             dict(k_pool=b.k_pool.half(), v_pool=b.v_pool.half()), dict(k_pool=b.k_pool.transpose(1, 2))]
    for w in wrong:
        with pytest.raises(native.KernelError):
            ops.attention_shared(**{**args, **w})
    x = rnd((6, 128), BF, 41)
    pos = torch.zeros((6, 2), dtype=torch.int32, device=DEV)
    args = dict(x=x, positions=pos, denom=ladder(32), sections=[16, 16], heads=2, head_dim=64)
    ops.rotate_axes(**args)
    wrong = [dict(heads=3), dict(heads=0), dict(head_dim=32), dict(sections=[16, 17]), dict(sections=[]), dict(sections=[8] * 5), dict(sections=[40, -8]),
             dict(sections="ab"), dict(positions=pos[:5]), dict(positions=pos.long()), dict(positions=pos[:, :1].contiguous()), dict(positions=pos.t().contiguous()),
             dict(denom=ladder(31)), dict(denom=ladder(32).double()), dict(x=x.half()), dict(x=x.t()), dict(x=x.cpu()), dict(out=x[:, :64]),
             dict(out=torch.empty((6, 128), dtype=F32, device=DEV)), dict(out=torch.empty((5, 128), dtype=BF, device=DEV)),
             dict(sections=[10, 22], interleaved=True)]
    for w in wrong:
        with pytest.raises(native.KernelError):
            ops.rotate_axes(**{**args, **w})
    wide = rnd((6, 256), BF, 42)
    with pytest.raises(native.KernelError):               # a result that lies partly on what is turned
        ops.rotate_axes(wide[:, :128], pos, ladder(32), [16, 16], 2, 64, out=wide[:, 64:192])
    kp, vp = (torch.zeros((3, PAGE, 2, 64), dtype=BF, device=DEV) for _ in range(2))
    seq = torch.zeros(6, dtype=torch.int32, device=DEV)
    args = dict(qkv=rnd((6, 8 * 64), BF, 43), row_seq=seq, row_pos=torch.arange(6, dtype=torch.int32, device=DEV), positions=pos, denom=ladder(32),
                sections=[16, 16], n_heads=4, n_kv_heads=2, head_dim=64, k_pool=kp, v_pool=vp, block_table=seq[:1].view(1, 1), page_size=PAGE)
    ops.rope_axes_kv_write(**args)
    wrong = [dict(n_heads=5), dict(n_kv_heads=3), dict(n_kv_heads=0), dict(k_pool=kp.float()), dict(v_pool=kp), dict(k_pool=kp[:, :, :1]), dict(page_size=16),
             dict(block_table=seq[:1].view(1, 1).long()), dict(block_table=seq[:1]), dict(row_seq=seq[:3]), dict(q_out=args["qkv"][:, 64:320]),
             dict(q_out=torch.empty((6, 4 * 64), dtype=F32, device=DEV)), dict(qkv=args["qkv"][:, :-1]), dict(positions=pos.cpu()),
             dict(block_table=torch.empty((1, 0), dtype=torch.int32, device=DEV))]
    for w in wrong:
        with pytest.raises(native.KernelError):
            ops.rope_axes_kv_write(**{**args, **w})
