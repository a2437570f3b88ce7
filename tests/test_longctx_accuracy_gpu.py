"""How exact the long-context operators are, against plain numpy in 64 bits.

Windowed attention in its ordinary form: scores are sums of exact products; with scores below 10 they and their
exponentials are off by some 5e-6; a weight is held to 2^-17 (bf16: two halves of 8 bits) or 2^-22 (fp16), and fp16
weights below 2^-21 of the largest to 2^-33 of it; a sum over the keys cuts off at most 2^-23 of itself for every
16 keys and half.  So a result is within 5e-6 + 2^-17 + keys * (2^-26 + 2^-33) of the largest value, before it is
rounded to its type.
"""
import numpy as np
import pytest

import longctx_ref as ref
from test_longctx_gpu import (BF16, F16, F32, HALF_ULP, close, dev, make_cache, rounded, run_window, store,
                              window_tol)

pytestmark = pytest.mark.gpu

SHAPES = [(1, 300, 40, 4), (5, 2000, 0, 0), (16, 700, 0, 0), (130, 130, 1, 0), (257, 300, 64, 3), (300, 300, 128, 130),
          (33, 1500, 700, 20)]


def case(kin, dim, H, Hk, n, m):
    rng = np.random.default_rng(n + m + dim)
    q, dq = rounded(rng.standard_normal((1, n, H, dim)), kin)
    k, dk = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    v, dv = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    return (q, k, v), (dq, dk, dv)


@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("dim,H,Hk", [(64, 4, 2), (128, 3, 1)])
@pytest.mark.parametrize("n,m,window,sinks", SHAPES)
def test_window_weights_are_not_rounded_to_16_bits(gpu, kin, dim, H, Hk, n, m, window, sinks):
    from ligguf_b200 import WindowConfig
    (q, k, v), d = case(kin, dim, H, Hk, n, m)
    out = run_window(WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=F32), *d, None, None, 1, n, m)
    want = ref.window_attention(q, k, v, [m - n], [m], window, sinks, dim ** -0.5)
    tol = (5e-6 + 2.0 ** -17 + m * (2.0 ** -26 + 2.0 ** -33)) * np.abs(v).max()
    close(out, want, tol)
    # and with 16-bit results, nothing but their own rounding on top
    out = run_window(WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=kin), *d, None, None, 1, n, m)
    close(out, want, tol, 1.01 * HALF_ULP[kin])


@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("kout", [F32, None])
@pytest.mark.parametrize("n,m,window,sinks", SHAPES)
def test_window_rounded_weights_when_asked_for(gpu, kin, kout, n, m, window, sinks):
    from ligguf_b200 import WindowConfig
    kout = kin if kout is None else kout
    (q, k, v), d = case(kin, 64, 4, 2, n, m)
    cfg = WindowConfig(4, 2, 64, window, sinks, in_type=kin, out_type=kout, round_weights=True)
    out = run_window(cfg, *d, None, None, 1, n, m)
    want = ref.window_attention(q, k, v, [m - n], [m], window, sinks, 64 ** -0.5)
    close(out, want, *window_tol(kin, kout, v))


@pytest.mark.parametrize("round_weights", [False, True])
@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("n", [2, 200])
def test_window_many_small_weights_add_up(gpu, kin, n, round_weights):
    """One key of weight 1 and value 0 before 4000 of weight e^-18 (2^-26, below fp16's range as it is) and value 1.
    A half of 2^-26 * 2^7 has five bits: within 2^-5.  (So many heads that no head's keys are split.)"""
    from ligguf_b200 import WindowConfig
    m, H, dim = 4001 + n, 300, 64
    q, k, v = np.zeros((1, n, H, dim)), np.zeros((1, m, H, dim)), np.ones((1, m, H, dim))
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 16.0, 1.125, 0.0
    cfg = WindowConfig(H, H, dim, scale=1.0, in_type=kin, out_type=F32, round_weights=round_weights)
    out = run_window(cfg, *(dev(x.astype(np.float32), kin) for x in (q, k, v)), None, None, 1, n, m)
    small = np.exp(-18.0) * (m - n + np.arange(n))
    want = np.broadcast_to((small / (1 + small))[None, :, None, None], out.shape)
    close(out, want, 0, 2.0 ** -5)


@pytest.mark.parametrize("kin", [F32, F16, BF16])
@pytest.mark.parametrize("dim,rope_dim,layout", [(128, 128, "adjacent"), (128, 128, "halves"), (64, 64, "halves"),
                                                 (128, 96, "halves"), (64, 20, "halves"), (64, 0, "adjacent")])
def test_token_is_held_alike_whichever_call_brought_it(gpu, kin, dim, rope_dim, layout):
    """A token's key and value are the same in the cache, bit for bit, whether append or decode wrote them."""
    import torch
    rng = np.random.default_rng(dim + rope_dim)
    n, Hk, nrep, pos0 = 300, 3, 2, 1000
    kw = dict(n_context=pos0 + n, rope_dim=rope_dim, layout=layout, qk_norm=True, in_type=kin, rows_type=F32)
    g = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    a, b = make_cache(dim, Hk, nrep, **kw), make_cache(dim, Hk, nrep, n_seqs=n, **kw)
    a.set_qk_norm(0, g[0], g[1])
    b.set_qk_norm(0, g[0], g[1])
    q, k, v = (rounded(rng.standard_normal((n, h * dim)) * 2, kin)[1] for h in (Hk * nrep, Hk, Hk))
    a.append_async(0, 0, pos0, n, None, k, v)
    out = torch.empty_like(q)
    b.decode_async(0, n, q, k, v, out, d_pos=torch.arange(pos0, pos0 + n, dtype=torch.int32, device="cuda"))
    ka, va = store(a, 0, 0, 1, pos0, n)
    kb, vb = store(b, 0, 0, n, pos0, n)
    each = np.arange(n)
    assert np.array_equal(va[0], vb[each, each]) and np.array_equal(ka[0], kb[each, each])
