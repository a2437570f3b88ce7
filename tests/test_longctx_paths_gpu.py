"""Paths of the long-context kernels that only large or many-sided calls reach, against 64 bits."""
import numpy as np
import pytest

import longctx_ref as ref
from test_longctx_gpu import F32, close, dev, host, make_cache, rounded, store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers,seqs", [(18, 1), (1, 18), (3, 6)])
def test_kv4_offsets_past_2_to_the_32(gpu, layers, seqs):
    """The last layer and sequence of a cache of 5.4 GB, at the end of a context of 2^18: its tiles lie past 2^32 bytes,
    by the layers, by the sequences or by both."""
    import torch
    rng = np.random.default_rng(12)
    n, Hk, dim, g = 1 << 18, 8, 128, 300
    layer, seq, first = layers - 1, seqs - 1, n - g
    assert ((layer * seqs + seq) * Hk * (n // 16) + first // 16) * 18 * dim > 1 << 32
    c = make_cache(dim, Hk, 1, n_context=n, n_layers=layers, n_seqs=seqs, window=200, sinks=3, rows_type=F32)
    kb, vb = (ref.q40(rng.standard_normal((1, g, Hk * dim))) for _ in range(2))
    c.load_async(layer, seq, 1, first, g, dev(kb), dev(vb))
    got = store(c, layer, seq, 1, first, g)
    assert np.array_equal(got[0], kb) and np.array_equal(got[1], vb)
    rows = [torch.empty(g, Hk * dim, device="cuda") for _ in range(2)]
    c.read_async(layer, seq, first, g, *rows)
    assert np.array_equal(host(rows[0]), ref.q40_values(kb)[0]) and np.array_equal(host(rows[1]), ref.q40_values(vb)[0])
    # One token of the last sequence (the others idle), then the cache as it left it.
    q, dq = rounded(rng.standard_normal((seqs, Hk, dim)), F32)
    k, dk = rounded(rng.standard_normal((seqs, Hk, dim)), F32)
    v, dv = rounded(rng.standard_normal((seqs, Hk, dim)), F32)
    out = torch.empty(seqs, Hk * dim, device="cuda")
    pos = np.full(seqs, -1, np.int32)
    pos[seq] = n - 1
    c.decode_async(layer, seqs, dq, dk, dv, out, d_pos=dev(pos))
    freq = ref.frequencies(dim, 1e4)
    qr, kr = (ref.rotate(x[seq:], [n - 1], freq, "adjacent") for x in (q, k))
    keys = ref.seen(n - 1, n - 1, 200, 0)  # the first tokens are zeros: keys of score 0, values of 0
    kk, vv = (ref.q40_values(b[0, keys - first]).reshape(-1, Hk, dim) for b in (kb, vb))
    zero = np.zeros((3, dim))
    want = np.stack([ref.attend(qr[0, h], np.concatenate([zero, kk[:, h], kr[0, h][None]]),
                                np.concatenate([zero, vv[:, h], v[seq, h][None]]), dim ** -0.5) for h in range(Hk)])
    close(host(out)[seq].reshape(Hk, dim), want, 2e-5 * np.abs(want).max())
    after = store(c, layer, seq, 1, first, g)
    assert np.array_equal(after[1][0, :-1], vb[0, :-1])
    assert np.array_equal(after[1][0, -1], ref.q40(v[seq].reshape(-1)))
    # An append there, across the end of a tile.
    kx, dk = rounded(rng.standard_normal((9, Hk * dim)), F32)
    c.append_async(layer, seq, n - 20, 9, None, dk, dk)
    assert np.array_equal(store(c, layer, seq, 1, n - 20, 9)[1][0], ref.q40(kx))
