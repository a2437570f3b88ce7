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


def test_window_entries_after_more_than_two_seconds_of_work(gpu):
    """Entry 0: 2^19 tokens without a window, so that none of its key tiles has rows to be hidden, about three seconds
    of work; entry 1: 200 keys, with such rows.  The kernel's waits are bounded to two seconds each, and none of them
    may count the time before its own item.  Rows of both entries against 64 bits; bound: see
    test_longctx_accuracy_gpu.py (equal values keep entry 0's sums, of half a million keys, apart from the cut)."""
    import torch
    from ligguf_b200 import WindowAttention, WindowConfig
    g = torch.Generator(device="cuda").manual_seed(5)
    B, n, H, dim, short = 2, 1 << 19, 48, 64, 200
    q = torch.randn(B, n, H * dim, generator=g, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(B, n, dim, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    v[0] = v[0, 0]
    out = torch.full_like(q, float("nan"))
    h = WindowAttention(WindowConfig(H, 1, dim))
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    h.attn_async(B, n, n, q, k, v, out, d_pos0=torch.zeros(2, dtype=torch.int32, device="cuda"),
                 d_lens=torch.tensor([n, short], dtype=torch.int32, device="cuda"))
    end.record()
    h.status()
    assert begin.elapsed_time(end) > 2100, "too little work for what this test is about"
    assert not torch.isnan(out).any()
    for b, rows in ((0, (0, 1, 127, 128, 4000)), (1, (0, 63, 127, 128, 199, 200, 5000, n - 1))):
        for i in rows:
            seen = min(i + 1, n if b == 0 else short)
            s = q[b, i].double().view(H, dim) @ k[b, :seen].double().T * dim ** -0.5
            want = torch.softmax(s, -1) @ v[b, :seen].double()
            close(out[b, i].double().view(H, dim).cpu().numpy(), want.cpu().numpy(), 5e-5 * float(v[b].abs().max()), 2.0 ** -8)
    last = out[0, -1].double().view(H, dim).cpu().numpy()
    close(last, np.broadcast_to(v[0, 0].double().cpu().numpy(), last.shape), 0.0, 2.0 ** -8 + 2.0 ** -8)


@pytest.mark.parametrize("rope_dim", [0, 128])
def test_kv4_cache_is_ready_for_any_stream(gpu, rope_dim):
    """A cache of 9.7 GB, whose zeroing takes the GPU some milliseconds, then at once a load on a stream that does not
    wait for the legacy stream: what was loaded stays, the rest is zeros.  The norm weights are there as well."""
    import torch
    import longctx_ref as ref
    n, Hk, last = 1 << 20, 8, 7
    kb, vb = (torch.randint(0, 256, (1, 64, Hk * 4, 18), dtype=torch.uint8, device="cuda") for _ in range(2))
    q, k, v = (torch.randn(1, w, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") for w in (1024,) * 3)
    got = [torch.full_like(kb, 7) for _ in range(2)]
    rows = [torch.full((1, 1024), float("nan"), device="cuda") for _ in range(3)]
    before = [torch.full_like(kb, 7) for _ in range(2)]
    g = (1 + 0.1 * np.random.default_rng(3).standard_normal((2, 128))).astype(np.float32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c = make_cache(128, Hk, 1, n_context=n, n_layers=last + 1, rope_dim=rope_dim, qk_norm=True, rows_type=F32)
    with torch.cuda.stream(side):
        c.load_async(last, 0, 1, n - 64, 64, kb, vb)
        c.set_qk_norm(last, g[0], g[1])
        c.append_async(last, 0, 0, 1, q, k, v, rows[0], rows[1], rows[2])
        c.store_async(last, 0, 1, n - 64, 64, *got)
        c.store_async(last, 0, 1, n - 128, 64, *before)
    torch.cuda.synchronize()
    assert torch.equal(got[0], kb) and torch.equal(got[1], vb)
    assert not any(x.any() for x in before)
    want = ref.rms(q.cpu().numpy().reshape(1, 8, 128), g[0], 1e-6)  # (position 0: no rotation)
    close(rows[0].cpu().numpy().reshape(1, 8, 128), want, 1e-5 * np.abs(want).max())
    c.status(stream=side)
