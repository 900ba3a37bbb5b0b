"""The operators of a shared prefix where there is no GPU: the module that takes torch tensors is made and loads, and what it and the
kernels' launchers refuse before anything is launched."""
import ctypes

import pytest
import torch

from friday_inference_engine_b200 import native, ops
from friday_inference_engine_b200.ops import lib

P, I, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


def binding():
    try:
        return ops._torch_ops()
    except native.BuildError as e:
        pytest.skip("the binding cannot be built here: %s" % e)


def family(name):
    try:
        return lib.family(name)
    except Exception as e:           # no compiler, or no CUDA runtime library to load against
        pytest.skip("the %s library is not available here: %s" % (name, e))


def test_tensors_of_another_device_are_refused():
    b = binding()
    x, pos, denom = torch.zeros((4, 8)), torch.zeros((4, 1), dtype=torch.int32), torch.ones(4)
    with pytest.raises(native.KernelError, match="rotate_axes: x is on cpu, these operations are cuda:0's"):
        b.rotate_axes(0, 0, x, 1, 8, pos, denom, [4], False, False, None)
    with pytest.raises(native.KernelError, match="rope_axes_kv_write: qkv is on cpu"):
        b.rope_axes_kv_write(0, 0, x, 1, 1, 2, pos, denom, [1], False, False, pos, pos, x, x, pos, 64, None)
    with pytest.raises(native.KernelError, match="attention_shared: q is on cpu"):
        b.attention_shared(0, 0, x, 8, x, 1, 1, 8, x, x, pos, 64, None, 0, pos, pos, 0, 1.0, 1, 1, 1, pos, pos)
    for bad in ((), (0,), (0, 0), (0, "a"), (0, 0, 3), (1 << 70, 0)):
        for f in (b.rotate_axes, b.rope_axes_kv_write, b.attention_shared):
            with pytest.raises(native.KernelError):
                f(*bad)


def rotate(rows=3, heads=2, hd=8, sections=(2, 2), interleaved=0, dtype=0):
    fam = family("rope_axes")
    fn = fam.declare("rope_axes_rotate", [P, L, P, L, I, I, I, P, I, P, P, I, I, P, I, P])
    return fn(None, heads * hd, None, heads * hd, rows, heads, hd, None, len(sections), None, (I * len(sections))(*sections), interleaved, 0, None, dtype, None)


@pytest.mark.parametrize("wrong", [dict(dtype=2), dict(heads=0), dict(hd=0), dict(sections=(3, 2)), dict(sections=(0, 0)), dict(sections=(-1, 4)),
                                   dict(sections=(1, 1, 1, 1, 0)), dict(sections=(1, 3), interleaved=1), dict(hd=512, sections=(100, 100))])
def test_sizes_that_a_rotation_refuses(wrong):
    assert rotate(**wrong) == 1
    assert rotate(rows=0) == 0                            # nothing to do is no error


def shared(rows=2, n_seqs=2, page=64, prefix=70, nq=4, nkv=2, hd=64, window=0, scale=0.1, floats=0, dtype=1, pool_pages=3, width=1, aligned=16):
    fam = family("attention_shared")
    fn = fam.declare("attention_shared", [P, L, P, P, P, I, I, P, I, P, I, I, P, P, P, P, I, I, I, I, I, I, I, ctypes.c_float, P, L, P, I, P, P])
    launches = I(7)
    rc = fn(aligned, nq * hd, aligned, aligned, aligned, pool_pages, page, None, prefix, None, n_seqs, width, None, None, None, None, rows, 1, prefix + 30, nq, nkv, hd,
            window, scale, None, floats, 16, dtype, ctypes.byref(launches), None)
    assert launches.value == 0
    return rc


@pytest.mark.parametrize("wrong", [dict(dtype=2), dict(nq=3), dict(nkv=0), dict(hd=0), dict(hd=257), dict(page=0), dict(prefix=-1), dict(window=-1), dict(scale=0.0),
                                   dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(pool_pages=0), dict(width=-1),
                                   dict(floats=10, prefix=20000), dict(floats=10, prefix=20000, dtype=0), dict(floats=10, hd=20)])
def test_sizes_that_attention_refuses(wrong):
    assert shared(**wrong) == 1
    assert shared(rows=0) == 0 and shared(n_seqs=0) == 0


def test_working_memory_that_is_missing_or_begins_anywhere_is_refused():
    fam = family("attention_shared")
    fn = fam.declare("attention_shared", [P, L, P, P, P, I, I, P, I, P, I, I, P, P, P, P, I, I, I, I, I, I, I, ctypes.c_float, P, L, P, I, P, P])
    for scratch in (None, 4, 8, 20):
        for hd in (64, 20):
            launches = I(7)
            assert fn(16, 4 * hd, 16, 16, 16, 3, 64, None, 20000, None, 2, 1, None, None, None, None, 2, 1, 20030, 4, 2, hd, 0, 0.1, scratch, 1 << 30,
                      16, 1, ctypes.byref(launches), None) == 1
            assert launches.value == 0


def floats_of(rows, n_seqs, max_q, max_kv, prefix, nq, nkv, hd, page=64, window=0, dtype=1):
    fam = family("attention_shared")
    fn = fam.declare("attention_shared_floats", [I] * 11, ctypes.c_longlong)
    return fn(rows, n_seqs, max_q, max_kv, prefix, nq, nkv, hd, page, window, dtype)


def parts_of(rows, nq, hd, floats):
    return 1 if floats == 0 else (floats - 1) // (rows * nq * (hd + 2))


def test_working_memory():
    # one-token steps behind a long prefix go in parts, prompts of many rows do not; nothing for nothing
    assert floats_of(0, 1, 1, 1, 0, 4, 2, 64) == 0 and floats_of(4, 0, 1, 1, 0, 4, 2, 64) == 0
    assert parts_of(64, 28, 128, floats_of(64, 64, 1, 17001, 16001, 28, 4, 128)) >= 4
    assert parts_of(1, 28, 128, floats_of(1, 1, 1, 32001, 32000, 28, 4, 128)) >= 16
    assert floats_of(2188, 16, 257, 8257, 8000, 28, 4, 128) <= 2188 * 28 * 130 + 1          # (the single rows' kernel: one part)
    # at most 64 parts of a row and head, whatever the sizes
    for rows, seqs, prefix, layout in ((1, 1, 2000000, (28, 4, 128)), (1, 1, 2000000, (2, 2, 20)), (3, 3, 100000, (3, 1, 32)), (1, 1, 1000000, (128, 1, 64))):
        for dtype in (0, 1):
            assert parts_of(rows, layout[0], layout[2], floats_of(rows, seqs, 1, prefix + 500, prefix, *layout, dtype=dtype)) <= 64
