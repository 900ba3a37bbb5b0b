"""Failures of the operators of a shared prefix: who is told, and as what.  Kernels whose bounded waits gave up: the failure is made on the
host, a code is copied to where a kernel would leave it, no kernel is made to wait."""
import ctypes

import numpy as np
import pytest
import torch

import shared_prefix as sp
from friday_inference_engine_b200 import native, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def cudart():
    try:
        from cuda.bindings import runtime
    except ImportError:
        from cuda import cudart as runtime
    return runtime


def word_of(stream):
    word = ctypes.c_void_p()
    native.call("friday_ops_stream_status", ops.backend()._h, stream.cuda_stream, ctypes.byref(word))
    return word.value


def leave(code, stream):
    """What a kernel that gives up does, behind the work that the stream has."""
    rt = cudart()
    number = torch.tensor([code], dtype=torch.int32).pin_memory()
    (err,) = rt.cudaMemcpyAsync(word_of(stream), number.data_ptr(), 4, rt.cudaMemcpyKind.cudaMemcpyHostToDevice, stream.cuda_stream)
    assert int(err) == 0
    return number


def test_a_failure_reaches_who_asks_about_its_stream_and_nobody_else():
    be = ops.backend()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x, pos = torch.ones((3, 8), device=DEV), torch.zeros((3, 1), dtype=torch.int32, device=DEV)
    denom = torch.ones(4, device=DEV)
    torch.cuda.synchronize()
    for s in (a, b):
        with torch.cuda.stream(s):
            ops.rotate_axes(x, pos, denom, [4], 1, 8)
        be.check_status(s)                                # nothing has happened
    assert len({word_of(a), word_of(b), be.info()["status_word"]}) == 3
    with torch.cuda.stream(a):
        torch.cuda._sleep(200_000_000)                    # a tenth of a second: who does not wait for the stream sees nothing
        held = leave(35, a)
    be.check_status(b)
    be.check_status()                                     # the default stream's
    with pytest.raises(native.KernelError, match=r"code 35.*attention_shared\.cu"):
        be.check_status(a)
    be.check_status(a)                                    # cleared
    with torch.cuda.stream(b):
        held = leave(41, b)
        with pytest.raises(native.KernelError, match=r"code 41.*rope_axes\.cu"):
            be.check_status()                             # torch's current stream
        be.check_status()
    del held


def test_the_default_streams_word_is_the_backends_own():
    be = ops.backend()
    assert word_of(torch.cuda.default_stream()) == be.info()["status_word"]
    held = leave(38, torch.cuda.default_stream())
    with pytest.raises(native.KernelError, match="code 38"):
        be.check_status(torch.cuda.Stream())              # (the backend's own is always asked about)
    be.check_status()
    del held


def test_a_captured_call_reports_to_the_stream_of_its_capture():
    be = ops.backend()
    b = sp.Batch(torch.bfloat16, [1] * 3, [20, 1, 77], 300, 14, 2, 64, seed=13)
    want = b.run(ops).clone()
    side, out = torch.cuda.Stream(), torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.run(ops, out)
        with pytest.raises(native.KernelError, match="while it is being captured"):
            native.call("friday_ops_check_stream", be._h, side.cuda_stream)
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        g.replay()
    other.synchronize()
    assert torch.equal(out, want)
    held = leave(31, side)
    be.check_status(other)
    with pytest.raises(native.KernelError, match="code 31"):
        be.check_status(side)
    del held


def test_more_streams_than_words():
    """Past the last word of their own, streams share the backend's: nothing is out of range, nothing is lost."""
    handle = ctypes.c_void_p()
    native.call("friday_ops_new", 0, None, ctypes.byref(handle))
    try:
        words = []
        for n in range(300):                              # (names of streams only: nothing runs on them)
            word = ctypes.c_void_p()
            native.call("friday_ops_stream_status", handle, 4096 + 64 * n, ctypes.byref(word))
            words.append(word.value)
        own = native.call_json("friday_ops_info", handle)["status_word"]
        assert len(set(words[:252])) == 252 and own not in words[:252] and set(words[252:]) == {own}
        assert np.ptp(np.array(words[:252])) == 4 * 251
        again = ctypes.c_void_p()
        native.call("friday_ops_stream_status", handle, 4096 + 64 * 7, ctypes.byref(again))
        assert again.value == words[7]
    finally:
        native.lib().friday_ops_free(handle)


def test_no_memory_for_a_result_is_torchs_own_error():
    x = torch.zeros((1 << 16, 256), device=DEV)
    pos, denom = torch.zeros((1 << 16, 1), dtype=torch.int32, device=DEV), torch.ones(64, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    room = (torch.cuda.memory_reserved(0) + (8 << 20)) / torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction(room)      # (of this process alone)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            ops.rotate_axes(x, pos, denom, [64], 2, 128)          # a result of 64 MB
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert ops.rotate_axes(x, pos, denom, [64], 2, 128).shape == x.shape


@pytest.mark.parametrize("shape", [(0, 3), (0, 0), (2, 0)])
def test_an_append_without_a_table_is_refused(shape):
    """(It used to hand back queries that nothing had written.)"""
    qkv, pos = torch.ones((2, 3 * 16), device=DEV), torch.zeros((2, 1), dtype=torch.int32, device=DEV)
    rows, table = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(shape, dtype=torch.int32, device=DEV)
    kp, vp = torch.zeros((1, 64, 1, 16), device=DEV), torch.zeros((1, 64, 1, 16), device=DEV)
    with pytest.raises(native.KernelError, match="block table is empty"):
        ops.rope_axes_kv_write(qkv, rows, rows, pos, torch.ones(8, device=DEV), [8], 1, 1, 16, kp, vp, table, 64)
    assert ops.rope_axes_kv_write(qkv[:0], rows[:0], rows[:0], pos[:0], torch.ones(8, device=DEV), [8], 1, 1, 16, kp, vp, table, 64).shape == (0, 16)
