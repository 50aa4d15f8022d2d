"""Calls of 4-bit attention whose launches have too many threads are refused, and kernels that
are none (no kernel is launched: the device handle is a block of zeros, which sizing such a
call only reads)."""
import ctypes as C

import pytest

import opure_hip as H


def reserve(heads, n_kv, hd, batch, rows, max_ctx):
    zeros = C.create_string_buffer(8192)
    m = H.Model()
    m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = 1, heads, n_kv, hd, H.A_F16
    kv = H.KV(1 << 40, 4, H.PAGE_SIZE, 1 << 41, 4)
    a = H.AttnKv4Args(C.pointer(m), C.pointer(kv), 0, batch, rows, None, max_ctx, 0, 0, None, None)
    return H.lib().opure_attn_kv4_reserve((C.addressof(zeros) + 255) // 256 * 256, C.byref(a))


@pytest.mark.parametrize("heads,hd,batch,fits", [(1 << 16, 64, 64, False), (1 << 16, 64, 63, True), (1 << 16, 128, 128, False), (1 << 16, 128, 127, True)])
def test_threads_of_one_launch(heads, hd, batch, fits):
    """A workgroup a sequence and KV head, 16 waves up to 64 channels, 8 past them: 2^32 threads are too many."""
    rc = reserve(heads, heads, hd, batch, 1, 1)
    assert (rc == H.E_CAPACITY) != fits                     # one that fits goes on to ask the device for its workspace
    if not fits:
        assert b"workgroups" in H.lib().opure_last_error()


def test_kernels_that_are_none():
    L, zeros, n = H.lib(), C.create_string_buffer(8192), C.c_uint32()
    dev = (C.addressof(zeros) + 255) // 256 * 256
    assert L.opure_debug_set_kv4_kernels(None, H.KV4_ONE) == H.E_INVALID
    assert L.opure_debug_set_kv4_kernels(dev, H.KV4_ROWS + 1) == H.E_INVALID
    a = H.AttnKv4Args()
    for args in ((None, C.byref(a), C.byref(n), C.byref(n)), (dev, None, C.byref(n), C.byref(n)), (dev, C.byref(a), None, C.byref(n)), (dev, C.byref(a), C.byref(n), None),
                 (dev, C.byref(a), C.byref(n), C.byref(n))):
        assert L.opure_debug_kv4_kernels(*args) == H.E_INVALID
