"""The long-context operators on the GPU against plain numpy in 64 bits: norms and rotation, the 4-bit
cache, its decode, windowed attention.

Tolerances, from the arithmetic (eps32 = 2^-24, half an ulp):
  rotation   the sum of D squares is off by at most D eps32, its root by half of that, a product and a
             rotation by about six roundings: below 1e-5 of the largest element at D = 128
  16 bits    one rounding more: 2^-11 (fp16) or 2^-8 (bf16) of the element
  decode     scores of magnitude S are off by a few S eps32 sqrt(D), so weights by about 1e-6 S; S < 10
             here: 2e-5 of the largest value
  window     weights are rounded to the operands' type once (relative 2^-11 / 2^-8), scores come from
             exact products; their exponentials are within 1.1e-4: (1.1e-4 + 2^-11 or 2^-8) of the largest
             value, and the output's own rounding
"""
import numpy as np
import pytest

import longctx_ref as ref
from ligguf_b200 import _lib

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _lib.KV_F32, _lib.KV_F16, _lib.KV_BF16
HALF_ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def tt(kind):
    import torch
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[kind]


def dev(x, kind=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if kind is None else t.to(tt(kind))


def host(t):
    return t.double().cpu().numpy()


def rounded(x, kind):
    """x as the type holds it, in 64 bits, and on the device."""
    t = dev(np.asarray(x, np.float32), kind)
    return host(t), t


def close(got, want, atol, rtol=0.0):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    bad = np.abs(got - want) - (atol + rtol * np.abs(want))
    assert bad.max(initial=-1.0) <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


# ------------------------------------------------------------------------------- norms and rotation
@pytest.mark.parametrize("n", [1, 3, 300])
@pytest.mark.parametrize("dim,rope_dim,layout", [(128, 128, "adjacent"), (128, 128, "halves"), (64, 64, "halves"),
                                                 (128, 96, "halves"), (64, 20, "halves"), (64, 2, "halves"),
                                                 (128, 126, "adjacent"), (64, 0, "adjacent"), (128, 62, "halves")])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_matches_formula(gpu, n, dim, rope_dim, layout, norm):
    from ligguf_b200 import QkRope, QkRopeConfig, RopeConfig
    import torch
    rng = np.random.default_rng(n + dim + rope_dim)
    H, Hk = 6, 3
    q, dq = rounded(rng.standard_normal((n, H, dim)) * 2, F32)
    k, dk = rounded(rng.standard_normal((n, Hk, dim)), F32)
    g = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    dg = dev(g)
    h = QkRope(QkRopeConfig(rope=RopeConfig(dim, rope_dim, layout, base=1e5), n_heads=H, n_kv_heads=Hk, qk_norm=norm))
    qo, ko = torch.full_like(dq, float("nan")), torch.full_like(dk, float("nan"))
    pos0 = 777
    h.run_async(n, dq, dk, qo, ko, pos0=pos0, q_gamma=dg[0] if norm else None, k_gamma=dg[1] if norm else None)
    freq = ref.frequencies(rope_dim, 1e5)
    for x, out, gm in ((q, qo, g[0]), (k, ko, g[1])):
        y = ref.rms(x, gm, 1e-6) if norm else x
        y = ref.rotate(y, pos0 + np.arange(n), freq, layout)
        close(host(out), y, 1e-5 * np.abs(y).max())


@pytest.mark.parametrize("scaling,factor,magnitude", [("linear", 4.0, 0.0), ("blend", 8.0, 1.2079), ("none", 1.0, 0.5)])
@pytest.mark.parametrize("layout", ["adjacent", "halves"])
def test_rope_scaled_far_positions(gpu, scaling, factor, magnitude, layout):
    """Positions up to 2^30 keep fp32 accuracy: the angle is formed in 64 bits."""
    from ligguf_b200 import QkRope, QkRopeConfig, RopeConfig
    import torch
    rng = np.random.default_rng(5)
    n, H, dim = 40, 4, 128
    pos = np.concatenate([[0, 1, 4095, 131071, 1 << 30], rng.integers(0, 1 << 21, n - 5)]).astype(np.int32)
    q, dq = rounded(rng.standard_normal((n, H, dim)), F32)
    rope = RopeConfig(dim, dim, layout, base=5e5, scaling=scaling, factor=factor, orig_context=8192, low=1.0, high=4.0,
                      magnitude=magnitude)
    h = QkRope(QkRopeConfig(rope=rope, n_heads=H, n_kv_heads=0))
    out = torch.empty_like(dq)
    h.run_async(n, dq, None, out, None, d_pos=dev(pos))
    y = ref.rotate(q, pos, ref.frequencies(dim, 5e5, scaling, factor, 8192), layout, magnitude or 1.0)
    close(host(out), y, 1e-5 * np.abs(y).max())


@pytest.mark.parametrize("kin", [F32, F16, BF16])
@pytest.mark.parametrize("kout", [F32, F16, BF16])
def test_rope_types_strides_in_place_and_stream(gpu, kin, kout):
    from ligguf_b200 import QkRope, QkRopeConfig, RopeConfig
    import torch
    rng = np.random.default_rng(11)
    n, H, Hk, dim = 37, 8, 2, 64
    wide = (H + 2 * Hk) * dim + 16
    x, dx = rounded(rng.standard_normal((n, wide)), kin)
    freq = np.abs(rng.standard_normal(16)).astype(np.float32)
    same = kin == kout
    rope = RopeConfig(dim, 32, "halves", freq=freq)
    cfg = QkRopeConfig(rope=rope, n_heads=H, n_kv_heads=Hk, in_type=kin, out_type=kout, q_stride=wide, k_stride=wide,
                       q_out_stride=wide if same else 0, k_out_stride=wide if same else 0)
    h = QkRope(cfg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        if same:  # in place, the rest of the rows untouched
            qo, ko = dx[:, :H * dim], dx[:, H * dim:(H + Hk) * dim]
        else:
            qo = torch.empty(n, H * dim, dtype=tt(kout), device="cuda")
            ko = torch.empty(n, Hk * dim, dtype=tt(kout), device="cuda")
        h.run_async(n, dx, dx[:, H * dim:], qo, ko, pos0=9)
    side.synchronize()
    for out, lo, heads in ((qo, 0, H), (ko, H * dim, Hk)):
        y = ref.rotate(x[:, lo:lo + heads * dim].reshape(n, heads, dim), 9 + np.arange(n), freq.astype(np.float64), "halves")
        close(host(out).reshape(y.shape), y, 1e-5 * np.abs(y).max(), HALF_ULP[kout])
    if same:
        assert np.array_equal(host(dx)[:, (H + Hk) * dim:], x[:, (H + Hk) * dim:])


# ------------------------------------------------------------------------------- 4-bit cache
def make_cache(dim=128, Hk=2, nrep=4, n_context=100, n_seqs=1, n_layers=1, rope_dim=None, **kw):
    from ligguf_b200 import Kv4Cache, Kv4Config, RopeConfig
    rope = RopeConfig(dim, dim if rope_dim is None else rope_dim, kw.pop("layout", "adjacent"), base=1e4)
    return Kv4Cache(Kv4Config(rope=rope, n_layers=n_layers, n_seqs=n_seqs, n_context=n_context, n_heads=Hk * nrep,
                              n_kv_heads=Hk, **kw))


def store(c, layer, seq, n_seqs, pos0, n):
    import torch
    G = c.cfg.n_kv_heads * c.cfg.rope.head_dim // 32
    kb, vb = (torch.zeros(n_seqs, n, G, 18, dtype=torch.uint8, device="cuda") for _ in range(2))
    c.store_async(layer, seq, n_seqs, pos0, n, kb, vb)
    return kb.cpu().numpy(), vb.cpu().numpy()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,pos0", [(1, 0), (5, 14), (16, 16), (45, 3)])
def test_kv4_blocks_round_trip_and_read(gpu, dim, n, pos0):
    import torch
    rng = np.random.default_rng(dim + n)
    c = make_cache(dim, Hk=3, nrep=1, n_context=48, n_seqs=3, n_layers=2, rows_type=F32)
    kb, vb = (ref.q40(rng.standard_normal((2, n, 3 * dim)) * s) for s in (1.0, 30.0))
    c.load_async(1, 1, 2, pos0, n, dev(kb), dev(vb))
    got = store(c, 1, 1, 2, pos0, n)
    assert np.array_equal(got[0], kb) and np.array_equal(got[1], vb)
    k, v = (torch.empty(n, 3 * dim, device="cuda") for _ in range(2))
    c.read_async(1, 2, pos0, n, k, v)
    # the value is a product of a 4-bit and an 11-bit number: exact in fp32
    assert np.array_equal(host(k), ref.q40_values(kb)[1]) and np.array_equal(host(v), ref.q40_values(vb)[1])
    everything = store(c, 1, 0, 3, 0, 48)
    for x in everything:  # nothing else was touched
        x[1:, pos0:pos0 + n] = 0
        assert not x.any()
    assert not any(x.any() for x in store(c, 0, 0, 3, 0, 48))


@pytest.mark.parametrize("dim,layout", [(64, "halves"), (128, "adjacent")])
@pytest.mark.parametrize("kin,rows", [(F32, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("n,pos0", [(1, 0), (2, 15), (61, 21), (300, 7)])
def test_kv4_append(gpu, dim, layout, kin, rows, n, pos0):
    """Values land as the definition's fp32 arithmetic has them, bit for bit; keys, whose norm and rotation
    may differ in the last place, within half a step of the exact ones."""
    import torch
    rng = np.random.default_rng(n)
    Hk, nrep = 2, 4
    c = make_cache(dim, Hk, nrep, n_context=320, n_seqs=2, qk_norm=True, in_type=kin, rows_type=rows, layout=layout)
    g = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    c.set_qk_norm(0, g[0], g[1])
    q, dq = rounded(rng.standard_normal((n, Hk * nrep, dim)) * 3, kin)
    k, dk = rounded(rng.standard_normal((n, Hk, dim)) * 2, kin)
    v, dv = rounded(rng.standard_normal((n, Hk, dim)) * rng.choice([1e-4, 1.0, 300.0], (n, Hk, 1)), kin)
    qo = torch.full((n, Hk * nrep * dim), float("nan"), dtype=tt(rows), device="cuda")
    kr, vr = (torch.full((n, Hk * dim), float("nan"), dtype=tt(rows), device="cuda") for _ in range(2))
    c.append_async(0, 1, pos0, n, dq, dk, dv, qo, kr, vr)
    freq = ref.frequencies(dim, 1e4)
    at = pos0 + np.arange(n)
    yq, yk = (ref.rotate(ref.rms(x, gm, 1e-6), at, freq, layout) for x, gm in ((q, g[0]), (k, g[1])))
    close(host(qo).reshape(yq.shape), yq, 1e-5 * np.abs(yq).max(), HALF_ULP[rows])
    kb, vb = store(c, 0, 1, 1, pos0, n)
    assert np.array_equal(vb[0], ref.q40(v.reshape(n, -1)))
    yk = yk.reshape(n, -1, 32)
    scale = np.ascontiguousarray(kb[0, ..., :2]).view(np.float16).astype(np.float64)
    m = np.where(yk.max(-1) >= -yk.min(-1), yk.max(-1), yk.min(-1))
    close(scale[..., 0], m / -8, 0, 1.01 * 2.0 ** -11 + 1e-5)
    held = ref.q40_values(kb[0]).reshape(yk.shape)
    top = np.concatenate([kb[0, ..., 2:] & 15, kb[0, ..., 2:] >> 4], -1) == 15  # clamped at 7 steps: off by up to one
    assert (np.abs(held - yk) <= np.abs(scale) * np.where(top, 1.01, 0.505)).all()
    for rr, bb in ((kr, kb), (vr, vb)):
        want = ref.q40_values(bb[0])
        close(host(rr), want, 1e-12, HALF_ULP[rows])
    # the other positions and the other sequence are untouched
    every = store(c, 0, 0, 2, 0, 320)
    for x in every:
        x[1, pos0:pos0 + n] = 0
        assert not x.any()


def test_kv4_append_odd_values(gpu):
    """Zeros, equal magnitudes of both signs, tiny and huge blocks, infinities and NaN."""
    dim = 64
    c = make_cache(dim, 1, 1, n_context=16, rope_dim=0, rows_type=F32)
    x = np.zeros((9, dim), np.float32)
    x[1, :32], x[1, 3], x[1, 9] = 0.25, -2.0, 2.0         # a tie: the positive one
    x[2] = np.linspace(-1e-7, 1e-7, dim)                    # the scale is a subnormal half
    x[3] = 1e-12                                            # the scale rounds to zero
    x[4] = np.linspace(-1e9, 1e9, dim)                      # it saturates
    x[5, 7] = np.inf
    x[6, 40] = np.nan
    x[7] = -np.abs(np.linspace(0, 4, dim))
    x[8, ::2] = 65504 * 8
    d = dev(x)
    c.append_async(0, 0, 2, 9, None, d, d)
    kb, vb = store(c, 0, 0, 1, 2, 9)
    assert np.array_equal(kb, vb)
    whole = [0, 1, 2, 3, 4, 7, 8]
    assert np.array_equal(kb[0][whole], ref.q40(x[whole]))
    held = ref.q40_values(kb[0])
    assert np.isnan(held[5, :32]).all() and not held[5, 32:].any()
    assert np.isnan(held[6, 32:]).all() and not held[6, :32].any()
    assert held[1, 9] == 2.0 and held[1, 3] == -1.75


def decode_case(rng, c, pos, kin, spread=1.0):
    """Fills the cache with random blocks and returns the inputs of one decode, on both sides."""
    cfg = c.cfg
    dim, Hk, H, R = cfg.rope.head_dim, cfg.n_kv_heads, cfg.n_heads, len(pos)
    n = cfg.n_context
    kb = ref.q40(rng.standard_normal((cfg.n_seqs, n, Hk * dim)))
    vb = ref.q40(rng.standard_normal((cfg.n_seqs, n, Hk * dim)) * spread)
    c.load_async(0, 0, cfg.n_seqs, 0, n, dev(kb), dev(vb))
    q, dq = rounded(rng.standard_normal((R, H, dim)), kin)
    k, dk = rounded(rng.standard_normal((R, Hk, dim)), kin)
    v, dv = rounded(rng.standard_normal((R, Hk, dim)) * (spread if np.isscalar(spread) else 1.0), kin)
    return kb, vb, (q, k, v), (dq, dk, dv)


def decode_ref(c, kb, vb, qkv, pos, gammas=None):
    cfg = c.cfg
    dim, Hk, H = cfg.rope.head_dim, cfg.n_kv_heads, cfg.n_heads
    q, k, v = qkv
    if gammas is not None:
        q, k = ref.rms(q, gammas[0], 1e-6), ref.rms(k, gammas[1], 1e-6)
    at = np.maximum(pos, 0)
    freq = ref.frequencies(cfg.rope.rope_dim, 1e4)
    q, k = ref.rotate(q, at, freq, cfg.rope.layout), ref.rotate(k, at, freq, cfg.rope.layout)
    out = np.zeros(q.shape)
    for r, p in enumerate(pos):
        if p < 0 or p >= cfg.n_context:
            continue
        keys = ref.seen(p, p, cfg.window, cfg.sinks)
        kk = ref.q40_values(kb[r, keys]).reshape(len(keys), Hk, dim)
        vv = ref.q40_values(vb[r, keys]).reshape(len(keys), Hk, dim)
        for h in range(H):
            g = h // (H // Hk)
            out[r, h] = ref.attend(q[r, h], np.concatenate([kk[:, g], k[r, g][None]]),
                                   np.concatenate([vv[:, g], v[r, g][None]]), cfg.scale or dim ** -0.5)
    return out


def run_decode(c, d, pos, kin, device_pos=True):
    import torch
    R = len(pos)
    w = c.cfg.n_kv_heads * c.cfg.rope.head_dim
    out = torch.full((R, c.cfg.n_heads * c.cfg.rope.head_dim), float("nan"), dtype=tt(kin), device="cuda")
    kr, vr = (torch.full((R, w), float("nan"), dtype=tt(c.cfg.rows_type), device="cuda") for _ in range(2))
    if device_pos:
        c.decode_async(0, R, *d, out, d_pos=dev(np.asarray(pos, np.int32)), k_rows=kr, v_rows=vr)
    else:
        c.decode_async(0, R, *d, out, pos=int(pos[0]), k_rows=kr, v_rows=vr)
    return host(out).reshape(R, c.cfg.n_heads, -1), host(kr), host(vr)


def check_rows(c, pos, kr, vr):
    """k_rows and v_rows are what the cache now holds; an idle row's are zeros."""
    for r, p in enumerate(pos):
        if 0 <= p < c.cfg.n_context:
            kb, vb = store(c, 0, r, 1, p, 1)
            ulp = HALF_ULP[c.cfg.rows_type]
            close(kr[r], ref.q40_values(kb[0, 0]), 1e-12, ulp)
            close(vr[r], ref.q40_values(vb[0, 0]), 1e-12, ulp)
        else:
            assert not kr[r].any() and not vr[r].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nrep", [1, 2, 4, 8])
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 17, 128, 1000])
def test_kv4_decode_single(gpu, dim, nrep, pos):
    rng = np.random.default_rng(pos + nrep)
    c = make_cache(dim, 2, nrep, n_context=1001, qk_norm=True, layout="halves")
    g = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    c.set_qk_norm(0, g[0], g[1])
    kb, vb, qkv, d = decode_case(rng, c, [pos], F32)
    out, kr, vr = run_decode(c, d, [pos], F32, device_pos=False)
    want = decode_ref(c, kb, vb, qkv, [pos], g)
    close(out, want, 2e-5 * np.abs(want).max())
    check_rows(c, [pos], kr, vr)
    c.status()


@pytest.mark.parametrize("kin", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 0), (33, 1), (100, 40), (5000, 3), (64, 200)])
def test_kv4_decode_batch_masks(gpu, kin, window, sinks):
    rng = np.random.default_rng(window)
    pos = np.array([0, 700, -1, 33, 32, 699, -5, 1, 100, 15, 16, 250])
    c = make_cache(128, 3, 4, n_context=701, n_seqs=len(pos), window=window, sinks=sinks, in_type=kin, rows_type=F32)
    kb, vb, qkv, d = decode_case(rng, c, pos, kin)
    out, kr, vr = run_decode(c, d, pos, kin)
    want = decode_ref(c, kb, vb, qkv, pos)
    close(out, want, 2e-5 * np.abs(want).max(), HALF_ULP[kin])
    assert not out[pos < 0].any()
    check_rows(c, pos, kr, vr)
    # what was there before the token is there still
    for r, p in enumerate(pos):
        now = store(c, 0, r, 1, 0, 701)
        for x, was in zip(now, (kb, vb)):
            keep = np.arange(701) != p
            assert np.array_equal(x[0, keep], was[r, keep])
    c.status()


@pytest.mark.parametrize("spread", [1e-5, 3e4])
def test_kv4_decode_value_magnitudes(gpu, spread):
    """Very small and very large values: the weights that multiply the codes carry the values' scales."""
    rng = np.random.default_rng(3)
    c = make_cache(128, 2, 4, n_context=513)
    kb, vb, qkv, d = decode_case(rng, c, [512], F32, spread)
    out, _, _ = run_decode(c, d, [512], F32)
    want = decode_ref(c, kb, vb, qkv, [512])
    close(out, want, 2e-5 * np.abs(want).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nrep", [1, 2, 4, 8])
@pytest.mark.parametrize("n", [15, 600, 5000])
def test_kv4_decode_holds_fp32_accuracy_with_unlike_weights(gpu, dim, nrep, n):
    """Scores spread over twenty powers of two: the halves that the tensor cores multiply together hold the
    queries and the weights to 2^-22, so the relative error (2-norm) stays within that of fp32 scores of this
    size: 20 * 2^-24 * ln 2 a weight, and as much again for the sums: 2e-6."""
    rng = np.random.default_rng(n + nrep)
    c = make_cache(dim, 2, nrep, n_context=n + 1, rope_dim=0)
    kb, vb, qkv, d = decode_case(rng, c, [n], F32)
    q = (qkv[0] * 3).astype(np.float32)
    out, _, _ = run_decode(c, (dev(q), d[1], d[2]), [n], F32)
    want = decode_ref(c, kb, vb, (q, qkv[1], qkv[2]), [n])
    assert np.linalg.norm(out - want) <= 2e-6 * np.linalg.norm(want)


def test_kv4_decode_mixed_value_magnitudes_and_large_scores(gpu):
    """Keys of very different scores and rows of very different values: a row of large values that gets a
    tiny weight, and one of tiny values that gets nearly all."""
    rng = np.random.default_rng(4)
    n = 777
    spread = 10.0 ** rng.integers(-4, 4, (1, n, 1))
    c = make_cache(64, 2, 8, n_context=n, scale=1.0)
    kb, vb, qkv, d = decode_case(rng, c, [n - 1], F32, spread)
    out, _, _ = run_decode(c, d, [n - 1], F32)
    want = decode_ref(c, kb, vb, qkv, [n - 1])
    # scores reach 40 here: weights within 4e-5, of values up to 4e3
    close(out, want, 1e-4 * np.abs(want).max())


@pytest.mark.parametrize("rows,dim,Hk,nrep", [(33, 64, 1, 2), (100, 128, 2, 4), (7, 64, 40, 1), (40, 64, 33, 2)])
def test_kv4_decode_many_rows_and_heads(gpu, rows, dim, Hk, nrep):
    """More sequences and KV heads than a warp has lanes, idle ones among them; from the device and, with one position
    for all, from the host."""
    rng = np.random.default_rng(rows)
    pos = rng.integers(-2, 150, rows)
    c = make_cache(dim, Hk, nrep, n_context=150, n_seqs=rows, window=70, sinks=2)
    kb, vb, qkv, d = decode_case(rng, c, pos, F32)
    out, kr, vr = run_decode(c, d, pos, F32)
    want = decode_ref(c, kb, vb, qkv, pos)
    close(out, want, 2e-5 * np.abs(want).max())
    assert not out[pos < 0].any()
    check_rows(c, pos[:40], kr, vr)
    c.load_async(0, 0, rows, 0, 150, dev(kb), dev(vb))
    pos = np.full(rows, 149)
    out, _, _ = run_decode(c, d, pos, F32, device_pos=False)
    want = decode_ref(c, kb, vb, qkv, pos)
    close(out, want, 2e-5 * np.abs(want).max())


@pytest.mark.parametrize("rope_dim,layout", [(20, "halves"), (48, "halves"), (62, "adjacent"), (2, "halves")])
@pytest.mark.parametrize("n", [3, 200])
def test_kv4_partly_rotated_heads(gpu, rope_dim, layout, n):
    """Rotated parts that are not whole units of eight elements, appended and decoded."""
    import torch
    rng = np.random.default_rng(rope_dim)
    c = make_cache(64, 2, 2, n_context=n + 1, rope_dim=rope_dim, layout=layout, rows_type=F32)
    x, dx = rounded(rng.standard_normal((n, 8 * 64)), F32)
    q, k, v = (x[:, a:b].reshape(n, -1, 64) for a, b in ((0, 256), (256, 384), (384, 512)))
    qo, kr, vr = (torch.empty(n, w, device="cuda") for w in (256, 128, 128))
    c.append_async(0, 0, 0, n, *(dx[:, a:b].contiguous() for a, b in ((0, 256), (256, 384), (384, 512))), qo, kr, vr)
    freq = ref.frequencies(rope_dim, 1e4)
    want = ref.rotate(q, np.arange(n), freq, layout)
    close(host(qo).reshape(want.shape), want, 1e-5 * np.abs(want).max())
    kb, vb = store(c, 0, 0, 1, 0, n)
    yk = ref.rotate(k, np.arange(n), freq, layout).reshape(n, -1, 32)
    d = np.abs(np.ascontiguousarray(kb[0, ..., :2]).view(np.float16).astype(np.float64))
    top = np.concatenate([kb[0, ..., 2:] & 15, kb[0, ..., 2:] >> 4], -1) == 15
    assert (np.abs(ref.q40_values(kb[0]).reshape(yk.shape) - yk) <= d * np.where(top, 1.01, 0.505)).all()
    assert np.array_equal(vb[0], ref.q40(v.reshape(n, -1)))
    kb, vb = (np.concatenate([b, np.zeros((1, 1) + b.shape[2:], np.uint8)], 1) for b in (kb, vb))
    qkv = [x for x in (rng.standard_normal((1, 4, 64)), rng.standard_normal((1, 2, 64)), rng.standard_normal((1, 2, 64)))]
    qkv, dd = zip(*(rounded(x, F32) for x in qkv))
    out, _, _ = run_decode(c, dd, [n], F32)
    want = decode_ref(c, kb, vb, qkv, [n])
    close(out, want, 2e-5 * np.abs(want).max())


def test_kv4_decode_poisoned_unseen_rows(gpu):
    """NaN in rows that the window hides, beyond the position, and in the token's own old row."""
    rng = np.random.default_rng(6)
    n, pos = 400, 301
    c = make_cache(128, 2, 4, n_context=n, window=70, sinks=5)
    kb, vb, qkv, d = decode_case(rng, c, [pos], F32)
    want = decode_ref(c, kb, vb, qkv, [pos])
    hidden = np.setdiff1d(np.arange(n), ref.seen(pos, pos, 70, 5))
    for b in (kb, vb):
        b[0, hidden, :, :2] = np.array([np.nan], np.float16).view(np.uint8)
    c.load_async(0, 0, 1, 0, n, dev(kb), dev(vb))
    out, kr, vr = run_decode(c, d, [pos], F32)
    close(out, want, 2e-5 * np.abs(want).max())
    assert np.isfinite(kr).all() and np.isfinite(vr).all()


def test_kv4_decode_nan_in_a_seen_row_reaches_its_heads_only(gpu):
    rng = np.random.default_rng(7)
    c = make_cache(64, 2, 2, n_context=64)
    kb, vb, qkv, d = decode_case(rng, c, [50], F32)
    vb[0, 20, 0, :2] = np.array([np.nan], np.float16).view(np.uint8)  # head 0, elements 0..31
    c.load_async(0, 0, 1, 0, 64, dev(kb), dev(vb))
    out, _, _ = run_decode(c, d, [50], F32)
    assert np.isnan(out[0, :2, :32]).all() and np.isfinite(out[0, 2:]).all()


def test_kv4_decode_position_beyond_context_is_reported(gpu):
    from ligguf_b200 import LigGufAttnError
    rng = np.random.default_rng(8)
    pos = np.array([40, 64, 2 ** 31 - 1])
    c = make_cache(128, 1, 4, n_context=64, n_seqs=3)
    kb, vb, qkv, d = decode_case(rng, c, pos, F32)
    out, kr, vr = run_decode(c, d, pos, F32)
    want = decode_ref(c, kb, vb, qkv, pos)
    close(out, want, 2e-5 * np.abs(want).max())
    assert not out[1:].any() and not kr[1:].any() and not vr[1:].any()
    with pytest.raises(LigGufAttnError, match="n_context"):
        c.status()
    c.status()  # reported once


def test_kv4_decode_repeats_bit_for_bit_and_replays_in_a_graph(gpu):
    import torch
    rng = np.random.default_rng(9)
    pos = np.array([1999, 30, -1, 700])
    c = make_cache(128, 4, 4, n_context=2000, n_seqs=4)
    kb, vb, qkv, d = decode_case(rng, c, pos, F32)
    dpos = dev(pos.astype(np.int32))
    outs = [torch.empty(4, 16 * 128, device="cuda") for _ in range(4)]
    for o in outs[:3]:
        c.decode_async(0, 4, *d, o, d_pos=dpos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.decode_async(0, 4, *d, outs[3], d_pos=dpos)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    # positions move on the device between replays
    dpos.copy_(dev(np.array([100, 29, 5, -1], np.int32)))
    graph.replay()
    out = host(outs[3]).reshape(4, 16, 128)
    want = decode_ref(c, kb, vb, qkv, [100, 29, 5, -1])
    close(out, want, 2e-5 * np.abs(want).max())


# ------------------------------------------------------------------------------- windowed attention
def window_tol(kin, kout, v):
    return (1.1e-4 + 1.05 * HALF_ULP[kin]) * np.abs(v).max() + 1e-6, HALF_ULP[kout]


def run_window(cfg, q, k, v, pos0, lens, batch, n, m, stream=None):
    import torch
    from ligguf_b200 import WindowAttention
    h = WindowAttention(cfg)
    out = torch.full((batch, n, cfg.n_heads * cfg.head_dim), float("nan"), dtype=tt(cfg.out_type), device="cuda")
    h.attn_async(batch, n, m, q, k, v, out, None if pos0 is None else dev(np.asarray(pos0, np.int32)),
                 None if lens is None else dev(np.asarray(lens, np.int32)))
    h.status()
    return host(out).reshape(batch, n, cfg.n_heads, cfg.head_dim)


@pytest.mark.parametrize("kin,kout", [(BF16, BF16), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("dim,H,Hk", [(64, 4, 2), (128, 3, 1), (128, 4, 4)])
@pytest.mark.parametrize("n,m,window,sinks", [(1, 1, 0, 0), (1, 300, 40, 4), (5, 300, 0, 0), (130, 130, 1, 0),
                                              (257, 300, 64, 3), (300, 300, 128, 130), (140, 140, 1000, 2),
                                              (33, 513, 129, 0)])
def test_window_matches_formula(gpu, kin, kout, dim, H, Hk, n, m, window, sinks):
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(n + m + window)
    q, dq = rounded(rng.standard_normal((1, n, H, dim)), kin)
    k, dk = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    v, dv = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    cfg = WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=kout)
    out = run_window(cfg, dq, dk, dv, None, None, 1, n, m)
    want = ref.window_attention(q, k, v, [m - n], [m], window, sinks, dim ** -0.5)
    close(out, want, *window_tol(kin, kout, v))


@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 0), (150, 6)])
@pytest.mark.parametrize("n", [3, 150])
def test_window_ragged_batch_empty_rows_and_poison(gpu, kin, window, sinks, n):
    """Lengths from none to all, queries before the first key and far past the last (rows that see
    nothing), rows of k and v past each length and outside the window poisoned."""
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(n)
    B, m, H, Hk, dim = 6, 200, 4, 2, 64
    lens = [200, 0, 1, 77, 130, 200]
    pos0 = [200 - n, 0, 0, -4, 400, 20]
    q, dq = rounded(rng.standard_normal((B, n, H, dim)), kin)
    k = rng.standard_normal((B, m, Hk, dim)).astype(np.float32)
    v = rng.standard_normal((B, m, Hk, dim)).astype(np.float32)
    clean, _ = rounded(v, kin)
    for b in range(B):
        used = set()
        for i in range(n):
            used |= set(ref.seen(pos0[b] + i, lens[b], window, sinks).tolist())
        hide = [j for j in range(m) if j not in used]
        k[b, hide], v[b, hide] = np.nan, np.inf
    kx, dk = rounded(k, kin)
    vx, dv = rounded(v, kin)
    cfg = WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=kin)
    out = run_window(cfg, dq, dk, dv, pos0, lens, B, n, m)
    want = ref.window_attention(q, kx, vx, pos0, lens, window, sinks, dim ** -0.5)
    close(out, want, *window_tol(kin, kin, clean))
    assert not out[1].any()


def test_window_strides_of_a_fused_row_and_batches(gpu):
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(2)
    B, n, H, Hk, dim = 2, 70, 4, 2, 128
    wide = (H + 2 * Hk) * dim + 8
    x, dx = rounded(rng.standard_normal((B, n + 3, wide)), BF16)
    nq, nk = H * dim, Hk * dim
    cfg = WindowConfig(H, Hk, dim, 20, 2, q_stride=wide, k_stride=wide, v_stride=wide,
                       q_batch_stride=(n + 3) * wide, k_batch_stride=(n + 3) * wide, v_batch_stride=(n + 3) * wide)
    out = run_window(cfg, dx, dx[..., nq:], dx[..., nq + nk:], None, None, B, n, n)
    q, k, v = (x[:, :n, lo:lo + w].reshape(B, n, -1, dim) for lo, w in ((0, nq), (nq, nk), (nq + nk, nk)))
    want = ref.window_attention(q, k, v, [0, 0], [n, n], 20, 2, dim ** -0.5)
    close(out, want, *window_tol(BF16, BF16, v))


@pytest.mark.parametrize("n", [2, 200])
def test_window_values_one_for_all_and_large_scores(gpu, n):
    """Equal values come back whatever the weights; scores of hundreds do not overflow."""
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(1)
    m, H, dim = 500, 2, 128
    _, dq = rounded(rng.standard_normal((1, n, H, dim)) * 20, F16)
    _, dk = rounded(rng.standard_normal((1, m, H, dim)) * 20, F16)
    _, dv = rounded(np.full((1, m, H, dim), 1.5), F16)
    out = run_window(WindowConfig(H, H, dim, 100, 4, in_type=F16, out_type=F32), dq, dk, dv, None, None, 1, n, m)
    close(out, np.full(out.shape, 1.5), (1.1e-4 + 1.05 * HALF_ULP[F16]) * 1.5)


def test_window_repeats_bit_for_bit(gpu):
    import torch
    from ligguf_b200 import WindowAttention, WindowConfig
    g = torch.Generator(device="cuda").manual_seed(3)
    for n, m in ((2, 9000), (700, 700)):
        q, k, v = (torch.randn(1, r, 8 * 128, generator=g, device="cuda").bfloat16() for r in (n, m, m))
        h = WindowAttention(WindowConfig(8, 8, 128, 4000, 4))
        outs = [torch.empty_like(q) for _ in range(3)]
        for o in outs:
            h.attn_async(1, n, m, q, k, v, o)
        h.status()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("kin,kout", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("dim,H,Hk", [(64, 2, 2), (128, 6, 2), (64, 8, 1), (128, 64, 1)])
@pytest.mark.parametrize("n,m,window,sinks", [(65, 1024, 0, 0), (23, 1100, 1000, 4), (33, 1500, 1, 1100), (37, 2050, 0, 0)])
def test_window_some_tokens_against_long_contexts(gpu, kin, kout, dim, H, Hk, n, m, window, sinks):
    """More rows of a KV head than one block holds, last blocks with few of them."""
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(n + m + window + H)
    q, dq = rounded(rng.standard_normal((1, n, H, dim)), kin)
    k, dk = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    v, dv = rounded(rng.standard_normal((1, m, Hk, dim)), kin)
    cfg = WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=kout)
    out = run_window(cfg, dq, dk, dv, None, None, 1, n, m)
    want = ref.window_attention(q, k, v, [m - n], [m], window, sinks, dim ** -0.5)
    close(out, want, *window_tol(kin, kout, v))
    assert np.array_equal(out, run_window(cfg, dq, dk, dv, None, None, 1, n, m))


@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1000, 6), (30, 1000)])
def test_window_some_tokens_ragged_batch_and_poison(gpu, kin, window, sinks):
    """As the ragged batch above, with blocks of one entry on both sides of its first key, its last
    key and its window."""
    from ligguf_b200 import WindowConfig
    rng = np.random.default_rng(window)
    B, n, m, H, Hk, dim = 5, 70, 1200, 4, 2, 64
    lens = [1200, 0, 33, 1130, 1200]
    pos0 = [1130, 0, -40, 1110, 2160]
    q, dq = rounded(rng.standard_normal((B, n, H, dim)), kin)
    k = rng.standard_normal((B, m, Hk, dim)).astype(np.float32)
    v = rng.standard_normal((B, m, Hk, dim)).astype(np.float32)
    clean, _ = rounded(v, kin)
    for b in range(B):
        used = set()
        for i in range(n):
            used |= set(ref.seen(pos0[b] + i, lens[b], window, sinks).tolist())
        hide = [j for j in range(m) if j not in used]
        k[b, hide], v[b, hide] = np.nan, np.inf
    kx, dk = rounded(k, kin)
    vx, dv = rounded(v, kin)
    cfg = WindowConfig(H, Hk, dim, window, sinks, in_type=kin, out_type=kin)
    out = run_window(cfg, dq, dk, dv, pos0, lens, B, n, m)
    want = ref.window_attention(q, kx, vx, pos0, lens, window, sinks, dim ** -0.5)
    close(out, want, *window_tol(kin, kin, clean))
    assert not out[1].any() and not out[2, :40].any()


def test_empty_calls_do_nothing(gpu):
    import torch
    from ligguf_b200 import QkRope, QkRopeConfig, RopeConfig, WindowAttention, WindowConfig
    QkRope(QkRopeConfig(rope=RopeConfig(64, 64), n_heads=1, n_kv_heads=1)).run_async(0, None, None, None, None)
    c = make_cache(64, 1, 1, n_context=16)
    c.append_async(0, 0, 16, 0, None, None, None)
    c.decode_async(0, 0, None, None, None, None)
    h = WindowAttention(WindowConfig(1, 1, 64))
    h.attn_async(0, 5, 5, None, None, None, None)
    h.attn_async(5, 0, 5, None, None, None, None)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, float("nan"))
    h.attn_async(1, 2, 0, q, None, None, out)  # no keys at all: zeros
    h.status()
    assert not out.any()


# ------------------------------------------------------------------------------- calls that are refused
def test_calls_with_bad_arguments_are_refused(gpu):
    """Each of these returns before anything is launched."""
    import torch
    from ligguf_b200 import LigGufAttnError, QkRope, QkRopeConfig, RopeConfig, WindowAttention, WindowConfig
    x = torch.zeros(4096, device="cuda")
    h = x.half()
    odd = x[1:]  # 4 bytes past an aligned address
    rope = RopeConfig(64, 64)
    r = QkRope(QkRopeConfig(rope=rope, n_heads=1, n_kv_heads=1, qk_norm=True))
    c = make_cache(64, 1, 1, n_context=16, n_seqs=2, qk_norm=True)
    w = WindowAttention(WindowConfig(1, 1, 64, in_type=F16, out_type=F16))

    def refused(status, word, f, *a, **k):
        with pytest.raises(LigGufAttnError, match=word) as e:
            f(*a, **k)
        assert e.value.status == status

    bad, state = _lib.EINVAL, _lib.ESTATE
    refused(bad, "tokens", r.run_async, -1, x, x, x, x)
    refused(bad, "tokens", r.run_async, 2, x, x, x, x, pos0=2 ** 31 - 2)
    refused(bad, "null", r.run_async, 1, None, x, x, x)
    refused(bad, "null", r.run_async, 1, x, x, x, None)
    refused(bad, "norm weights", r.run_async, 1, x, x, x, x, q_gamma=x)
    refused(bad, "aligned", r.run_async, 1, odd, x, x, x, q_gamma=x, k_gamma=x)
    refused(state, "were not set", c.append_async, 0, 0, 0, 1, None, x, x)
    refused(state, "were not set", c.decode_async, 0, 1, x, x, x, x)
    g = np.ones(64, np.float32)
    with pytest.raises(ValueError):
        c.set_qk_norm(0, g[:32], g)
    refused(bad, "layer", c.set_qk_norm, 1, g, g)
    c.set_qk_norm(0, g, g)
    refused(bad, "layer", c.append_async, -1, 0, 0, 1, None, x, x)
    refused(bad, "sequences", c.append_async, 0, 2, 0, 1, None, x, x)
    refused(bad, "positions", c.append_async, 0, 0, 15, 2, None, x, x)
    refused(bad, "positions", c.append_async, 0, 0, 0, -1, None, x, x)
    refused(bad, "null", c.append_async, 0, 0, 0, 1, None, x, None)
    refused(bad, "null", c.append_async, 0, 0, 0, 1, None, x, x, x)  # queries wanted, none given
    refused(bad, "aligned", c.append_async, 0, 0, 0, 1, None, odd, x)
    refused(bad, "sequences", c.decode_async, 0, 3, x, x, x, x)
    refused(bad, "pos", c.decode_async, 0, 1, x, x, x, x, pos=16)
    refused(bad, "pos", c.decode_async, 0, 1, x, x, x, x, pos=-1)
    refused(bad, "null", c.decode_async, 0, 1, x, x, None, x)
    refused(bad, "aligned", c.decode_async, 0, 1, x, x, x, odd)
    refused(bad, "positions", c.read_async, 0, 0, 10, 7, x, x)
    refused(bad, "sequences", c.load_async, 0, 1, 2, 0, 1, x, x)
    refused(bad, "null", c.store_async, 0, 0, 1, 0, 1, x, None)
    refused(bad, "batch", w.attn_async, -1, 1, 1, h, h, h, h)
    refused(bad, "batch", w.attn_async, 1, 1, 1 << 30, h, h, h, h)
    refused(bad, "null", w.attn_async, 1, 1, 1, h, None, h, h)
    refused(bad, "aligned", w.attn_async, 1, 1, 1, h, h[1:], h, h)
    c.status()
    w.status()


def test_cache_beyond_the_memory_is_refused(gpu):
    from ligguf_b200 import LigGufAttnError
    for seqs, status in ((2048, _lib.ENOMEM), (65535, _lib.EUNSUPPORTED)):
        with pytest.raises(LigGufAttnError) as e:
            make_cache(128, 8, 4, n_context=1 << 20, n_seqs=seqs, n_layers=64)
        assert e.value.status == status


def test_kv4_offsets_beyond_32_bits(gpu):
    """The last layer of a cache of 5.7 GB: tiles past 2^32 bytes, and the last positions of a context of 2^18."""
    rng = np.random.default_rng(12)
    n = 1 << 18
    c = make_cache(128, 8, 1, n_context=n, n_layers=9, window=200, sinks=3, rows_type=F32)
    g = 300
    kb, vb = (ref.q40(rng.standard_normal((1, g, 8 * 128))) for _ in range(2))
    first = n - g
    c.load_async(8, 0, 1, first, g, dev(kb), dev(vb))
    assert np.array_equal(store(c, 8, 0, 1, first, g)[1], vb)
    q, dq = rounded(rng.standard_normal((1, 8, 128)), F32)
    k, dk = rounded(rng.standard_normal((1, 8, 128)), F32)
    v, dv = rounded(rng.standard_normal((1, 8, 128)), F32)
    import torch
    out = torch.empty(1, 8 * 128, device="cuda")
    c.decode_async(8, 1, dq, dk, dv, out, pos=n - 1)
    freq = ref.frequencies(128, 1e4)
    qr, kr = (ref.rotate(x, [n - 1], freq, "adjacent") for x in (q, k))
    keys = ref.seen(n - 1, n - 1, 200, 0)  # the first tokens are zeros: keys of score 0, values of 0
    want = np.zeros((8, 128))
    kk = ref.q40_values(kb[0, keys - first]).reshape(-1, 8, 128)
    vv = ref.q40_values(vb[0, keys - first]).reshape(-1, 8, 128)
    for h in range(8):
        zero = np.zeros((3, 128))
        want[h] = ref.attend(qr[0, h], np.concatenate([zero, kk[:, h], kr[0, h][None]]),
                             np.concatenate([zero, vv[:, h], v[0, h][None]]), 128 ** -0.5)
    close(host(out).reshape(8, 128), want, 2e-5 * np.abs(want).max())


def test_example_runs_the_operators_together(gpu):
    """examples/long_context.py: prompt and draft within the operands' rounding (2^-8 of bf16, weights and exponentials
    as for windowed attention: 1.1e-4 + 2^-8 of the largest value, twice for values and result of unlike size), single
    tokens within fp32's."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "long_context.py")
    spec = importlib.util.spec_from_file_location("long_context", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    e = m.run(prompt=1300, chunk=555, tokens=3, window=400)
    assert e["prompt"] <= 1e-2 and e["draft"] <= 1e-2 and e["tokens"] <= 2e-5, e
