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


def window_ref(q, k, v, pos0, lens, window, sinks):
    """ref.window_attention with torch on the GPU, an entry at a time: q [B, n, H, D], k, v [B, m, Hk, D]."""
    import torch
    B, n, H, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    keys = torch.arange(k.shape[1], device="cuda")
    for b in range(B):
        at = pos0[b] + torch.arange(n, device="cuda")[:, None]
        seen = (keys <= at) & (keys < lens[b])
        if window:
            seen &= (keys > at - window) | (keys < sinks)
        kk, vv = (x[b].double().repeat_interleave(H // k.shape[2], 1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q[b].double(), kk) * D ** -0.5
        w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).masked_fill(~seen.any(-1)[:, None], 0.0)
        out[b] = torch.einsum("hij,jhd->ihd", w, vv)
    return out


def poisoned(x, pos0, lens, n, window, sinks, value):
    """x [B, m, ..] with `value` in every row that no query of its entry sees."""
    import torch
    y = x.clone()
    keys = torch.arange(x.shape[1], device="cuda")
    for b in range(x.shape[0]):
        at = pos0[b] + torch.arange(n, device="cuda")[:, None]
        seen = (keys <= at) & (keys < lens[b])
        if window:
            seen &= (keys > at - window) | (keys < sinks)
        y[b, ~seen.any(0)] = value
    return y


def check_window(B, n, m, H, Hk, dim, window, sinks, pos0, lens, kin, round_weights, seed):
    import torch
    from ligguf_b200 import KV_BF16, KV_F16, WindowAttention, WindowConfig
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.bfloat16 if kin == "bf16" else torch.float16
    kind = KV_BF16 if kin == "bf16" else KV_F16
    q = torch.randn(B, n, H, dim, generator=g, device="cuda").to(t)
    k, v = (torch.randn(B, m, Hk, dim, generator=g, device="cuda").to(t) for _ in range(2))
    want = window_ref(q, k, v, pos0, lens, window, sinks)
    k2 = poisoned(k, pos0, lens, n, window, sinks, float("nan"))
    v2 = poisoned(v, pos0, lens, n, window, sinks, float("inf"))
    h = WindowAttention(WindowConfig(H, Hk, dim, window, sinks, in_type=kind, out_type=F32, round_weights=round_weights))
    out = torch.full((B, n, H, dim), float("nan"), device="cuda")
    d = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (pos0, lens)]
    h.attn_async(B, n, m, q, k2, v2, out, *d)
    h.status()
    again = torch.full_like(out, float("nan"))
    h.attn_async(B, n, m, q, k2, v2, again, *d)
    h.status()
    assert torch.equal(out, again)
    # test_longctx_accuracy_gpu.py's bound, or test_longctx_gpu.py's for rounded weights
    top = float(v.abs().max())
    ulp = 2.0 ** -8 if kin == "bf16" else 2.0 ** -11
    tol = 1.1e-4 + 1.05 * ulp if round_weights else 5e-6 + 2.0 ** -17 + m * (2.0 ** -26 + 2.0 ** -33)
    close(out.double().cpu().numpy(), want.cpu().numpy(), tol * top + 1e-6)


@pytest.mark.parametrize("round_weights", [False, True])
@pytest.mark.parametrize("kin", ["bf16", "f16"])
@pytest.mark.parametrize("dim,H,Hk", [(64, 8, 2), (128, 6, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3), (128, 200), (1, 0)])
def test_window_many_items_a_cta(gpu, window, sinks, kin, dim, H, Hk, round_weights):
    """Several items a CTA, one after another: entries without keys, with one, with whole key tiles and with parts of
    them; queries before the first key, at the end and far past it; unseen rows of k and v poisoned.  (Fewer than 1024
    keys and more than 64 rows a KV head, so that the tensor-core form takes them.)"""
    import torch
    B, n, m = 60, 150, 700
    rng = np.random.default_rng(window + dim)
    lens = [0, 1, 128, 127, 129, 256, 384, 700, 640, 333] + rng.integers(0, m + 1, B - 10).tolist()
    rng.shuffle(lens)
    pos0 = [int(rng.choice([x - n, 0, x, rng.integers(-n - 5, m + 300)])) for x in lens]
    items = H * 2 * B
    assert items > 4 * torch.cuda.get_device_properties(0).multi_processor_count
    check_window(B, n, m, H, Hk, dim, window, sinks, pos0, lens, kin, round_weights, 7)


@pytest.mark.parametrize("kin,dim", [("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
def test_window_more_items_than_a_cta_works_out_ahead(gpu, window, sinks, kin, dim):
    """More than 64 items a CTA: those from the 65th on are worked out by each role."""
    import torch
    B, n, m, H = 160, 2, 150, 64
    assert B * H > 64 * torch.cuda.get_device_properties(0).multi_processor_count
    rng = np.random.default_rng(window)
    lens = rng.integers(0, m + 1, B).tolist()
    pos0 = [int(rng.choice([x - n, 0, x, rng.integers(-5, m + 50)])) for x in lens]
    check_window(B, n, m, H, 1, dim, window, sinks, pos0, lens, kin, False, 8)


@pytest.mark.parametrize("dim,nrep", [(128, 4), (64, 1), (64, 8), (128, 8), (128, 2)])
def test_kv4_decode_one_head_over_more_than_64_blocks(gpu, dim, nrep):
    """One KV head, whose item more blocks share than the join holds factors of in registers (two a lane): about 2100
    units (an item's 56, its 2048 tiles and the token), at least 16 a block."""
    from test_longctx_gpu import decode_case, decode_ref, run_decode
    rng = np.random.default_rng(dim + nrep)
    n = 32768
    assert (56 + n // 16 + 1) / 16 > 2 * 64
    c = make_cache(dim, 1, nrep, n_context=n + 1)
    kb, vb, qkv, d = decode_case(rng, c, [n], F32)
    out, _, _ = run_decode(c, d, [n], F32)
    want = decode_ref(c, kb, vb, qkv, [n])
    close(out, want, 2e-5 * np.abs(want).max())
    assert np.linalg.norm(out - want) <= 2e-6 * np.linalg.norm(want)
    again, _, _ = run_decode(c, d, [n], F32)
    assert np.array_equal(out, again)
    c.status()
