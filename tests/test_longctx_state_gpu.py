"""What the long-context handles keep between calls: error words, tickets, set-up on the GPU."""
import ctypes

import numpy as np
import pytest

from ligguf_b200 import _lib
from test_longctx_gpu import F32, close, decode_case, decode_ref, make_cache, run_decode

pytestmark = pytest.mark.gpu


class Kv4Handle(ctypes.Structure):
    """Mirror of struct ligguf_kv4 (ligguf_b200/csrc/longctx_api.cu)."""

    _fields_ = [("cfg", _lib.Kv4Cfg), ("nrep", ctypes.c_int), ("tiles_per_head", ctypes.c_longlong),
                ("tile_bytes", ctypes.c_size_t), ("tiles", ctypes.c_void_p), ("turns", ctypes.c_void_p),
                ("gammas", ctypes.c_void_p), ("norm_set", ctypes.c_void_p), ("parts", ctypes.c_void_p),
                ("tickets", ctypes.c_void_p), ("num_sms", ctypes.c_int), ("h_err", ctypes.POINTER(ctypes.c_int)),
                ("d_err", ctypes.c_void_p)]


def device_ints(address, n):
    """n ints of device memory that the library owns, as a tensor."""
    import torch

    class Memory:
        __cuda_array_interface__ = {"shape": (n,), "typestr": "<i4", "data": (address, False), "version": 3}
    return torch.as_tensor(Memory(), device="cuda")


@pytest.mark.parametrize("position_too", [False, True])
def test_kv4_decode_recovers_from_a_wait_that_gave_up(gpu, position_too):
    """What a launch leaves behind when a wait in it gives up (its word and tickets of items that blocks share), put
    there by the host; then, with position_too, a decode that meets a position beyond the context.  The status call
    reports the wait whatever came later, and the next decode is right."""
    import torch
    from ligguf_b200 import LigGufAttnError
    rng = np.random.default_rng(1)
    n = 3000
    c = make_cache(128, 2, 4, n_context=n, n_seqs=2)
    h = ctypes.cast(c.handle, ctypes.POINTER(Kv4Handle)).contents
    assert (h.cfg.n_context, h.nrep, h.tile_bytes) == (n, 4, 18 * 128) and h.num_sms > 0 and not any(h.h_err[:2])
    pos = [n - 1, n - 5]
    kb, vb, qkv, d = decode_case(rng, c, pos, F32)
    if position_too:
        run_decode(c, d, [-1, n], F32)  # (no shared items)
        torch.cuda.synchronize()
    h.h_err[0] = 1  # KERR_TIMEOUT_FULL
    tickets = device_ints(h.tickets, 4)
    assert not tickets.any()
    tickets.copy_(torch.tensor([1, 0, 3, 2], dtype=torch.int32))
    with pytest.raises(LigGufAttnError) as e:
        c.status()
    assert e.value.status == _lib.ETIMEDOUT
    c.status()  # reported once
    for _ in range(2):
        out, _, _ = run_decode(c, d, pos, F32)
        want = decode_ref(c, kb, vb, qkv, pos)
        close(out, want, 2e-5 * np.abs(want).max())
    c.status()
