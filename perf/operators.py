"""The long-context operators of this package as measurable cases, with their plain forms.

Four operators that a serving engine runs one after another on long contexts:

  rope     the RMS norm of every query and key head and the rotation by position, in one pass
  append   the same, and a prompt's keys and values quantized to the 4-bit cache
  decode   one token of each sequence: norm, rotation, append, attention over the 4-bit cache
  window   causal attention with a sliding window and visible first tokens over 16-bit rows

``run(state)`` makes one pass: with ``own`` false in elementary torch operations in 32 bits, with
``own`` true through the package's public calls.  ``exact`` gives the same outputs in 64 bits, from the
definitions.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # The 32 query and 8 key heads of one decoded token, straight from the fp32 projections.
        dict(name="rope token f32", op="rope", n=1, heads=32, kv_heads=8, dim=128, rope_dim=128, layout="adjacent",
             norm=True, base=1e6, scaling="none", factor=1.0, pos0=32768, scattered=False, strided=False, type="f32",
             out="f32"),
        # A prompt of 7777 tokens packed from sequences at different places (so with a position array), read
        # from rows that hold q, k and v side by side; three quarters of the head rotated, frequencies
        # blended for a context eight times the trained one.
        dict(name="rope packed prompt f16", op="rope", n=7777, heads=32, kv_heads=8, dim=128, rope_dim=96,
             layout="halves", norm=True, base=1e6, scaling="blend", factor=8.0, pos0=0, scattered=True, strided=True,
             type="f16", out="f16"),
        # A prompt of 2048 tokens into one layer's cache, from fp32 projections, with the rotated queries and
        # the rows as the cache holds them for the prompt's attention.
        dict(name="append prompt 2048 f32", op="append", n=2048, heads=32, kv_heads=8, dim=128, rope_dim=128,
             layout="adjacent", norm=True, base=1e6, scaling="none", factor=1.0, pos0=0, strided=False, type="f32",
             out="bf16"),
        # A short turn appended in the middle of a conversation (odd length and place), small heads.
        dict(name="append turn 333 bf16", op="append", n=333, heads=32, kv_heads=4, dim=64, rope_dim=64,
             layout="halves", norm=False, base=1e4, scaling="linear", factor=4.0, pos0=1717, strided=True,
             type="bf16", out="bf16"),
        # One token of a chat on a small model: 512 cached positions, where latency counts.
        dict(name="decode 512 f32", op="decode", rows=1, heads=32, kv_heads=4, dim=64, rope_dim=64,
             layout="adjacent", norm=False, base=1e4, scaling="none", factor=1.0, low=512, high=512, idle=0,
             window=0, sinks=0, type="f32", out="f16"),
        # One token at the end of a context of 32768, the whole of it read.
        dict(name="decode 32768 f32", op="decode", rows=1, heads=32, kv_heads=8, dim=128, rope_dim=128,
             layout="adjacent", norm=True, base=1e6, scaling="none", factor=1.0, low=32768, high=32768, idle=0,
             window=0, sinks=0, type="f32", out="f16"),
        # A batch of 24 sequences of all lengths up to 8192, three of its slots idle.
        dict(name="decode batch 24 bf16", op="decode", rows=24, heads=32, kv_heads=8, dim=128, rope_dim=128,
             layout="halves", norm=True, base=1e6, scaling="blend", factor=4.0, low=1, high=8191, idle=3, window=0,
             sinks=0, type="bf16", out="bf16"),
        # Sixteen long streams that keep their first 4 tokens and the last 4096.
        dict(name="decode streams 16 f16", op="decode", rows=16, heads=32, kv_heads=8, dim=128, rope_dim=128,
             layout="halves", norm=False, base=1e6, scaling="none", factor=1.0, low=100, high=16000, idle=0,
             window=4096, sinks=4, type="f16", out="f16"),
        # A prompt of 2048 tokens through a layer with a window of 512.
        dict(name="window prompt 2048 bf16", op="window", batch=1, n=2048, m=2048, heads=32, kv_heads=8, dim=128,
             window=512, sinks=4, ragged=False, strided=False, type="bf16"),
        # A long prompt, q, k and v side by side in one row, a window of 4096.
        dict(name="window prompt 8192 f16", op="window", batch=1, n=8192, m=8192, heads=32, kv_heads=8, dim=128,
             window=4096, sinks=16, ragged=False, strided=True, type="f16"),
        # Five conversations of different lengths that go on by up to 777 tokens, one of them empty.
        dict(name="window ragged 5 bf16", op="window", batch=5, n=777, m=1500, heads=32, kv_heads=4, dim=64,
             window=300, sinks=1, ragged=True, strided=False, type="bf16"),
        # Four new tokens (a checked draft) at the end of a 16-bit cache of 32768.
        dict(name="window 4 tokens bf16", op="window", batch=1, n=4, m=32768, heads=32, kv_heads=8, dim=128,
             window=16384, sinks=64, ragged=False, strided=False, type="bf16"),
    ]


def _between(rng, low, high):
    """A whole number, its logarithm spread evenly."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "decode", "decode", "window", "window"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    c = dict(op=op, heads=kv * rng.choice([1, 2, 4, 4, 8] if kv < 8 else [1, 2, 4]), kv_heads=kv, dim=dim)
    if op != "window":
        c |= dict(rope_dim=rng.choice([dim, dim, dim * 3 // 4, dim // 2]), layout=rng.choice(["adjacent", "halves"]),
                  norm=rng.random() < 0.6, base=rng.choice([1e4, 1e6]), scaling=rng.choice(["none", "linear", "blend"]))
        c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0])
    if op == "rope":
        c |= dict(n=_between(rng, 1, 7777), pos0=_between(rng, 1, 100000), scattered=rng.random() < 0.5,
                  strided=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]))
        c["out"] = rng.choice([c["type"], "bf16", "f16"])
    elif op == "append":
        c |= dict(n=_between(rng, 1, 2048), pos0=_between(rng, 1, 4000), strided=rng.random() < 0.5,
                  type=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f16", "bf16"]))
    elif op == "decode":
        rows = _between(rng, 1, 24)
        high = _between(rng, 64, 32768 if rows < 4 else 8192)
        c |= dict(rows=rows, low=rng.choice([1, high // 2, high]), high=high, idle=rows // 8,
                  window=rng.choice([0, 0, _between(rng, 16, 4096)]), type=rng.choice(["f32", "f16", "bf16"]),
                  out=rng.choice(["f16", "bf16"]))
        c["sinks"] = rng.choice([0, 1, 4, 64]) if c["window"] else 0
    else:
        few = rng.random() < 0.35
        n = rng.randint(1, 8) if few else _between(rng, 32, 4096)
        c |= dict(batch=1 if few or n > 1000 else rng.randint(1, 5), n=n,
                  m=_between(rng, 256, 32768) if few else n + rng.choice([0, rng.randint(1, 700)]),
                  window=rng.choice([0, _between(rng, 16, 4096)]), type=rng.choice(["f16", "bf16"]))
        c["sinks"] = rng.choice([0, 1, 4, 64]) if c["window"] else 0
        c["ragged"] = not few and rng.random() < 0.4
        c["strided"] = c["n"] == c["m"] and rng.random() < 0.5
    return c


# ---------------------------------------------------------------------------------------- the inputs
def _positions(c):
    """Decode positions of the case's rows (-1: idle), spread over [low, high]; by the case alone."""
    rng = random.Random(c["rows"] * 7919 + c["high"])
    at = [c["high"] if r == 0 else rng.randint(c["low"], c["high"]) for r in range(c["rows"])]
    for r in range(c["idle"]):
        at[(2 * r + 1) % c["rows"]] = -1
    return at


def _spans(c):
    """(first query's position, keys) of each batch entry of a window case; by the case alone."""
    n, m = c["n"], c["m"]
    if not c["ragged"]:
        return [m - n] * c["batch"], [m] * c["batch"]
    rng = random.Random(n * 31 + m)
    lens = [0 if b == 1 else rng.randint(max(1, m // 3), m) for b in range(c["batch"])]
    return [max(0, x - n) for x in lens], lens


def _context(c):
    return (c["high"] if c["op"] == "decode" else c["pos0"] + c["n"]) + 1


def _sizes(c):
    return c["heads"] * c["dim"], c["kv_heads"] * c["dim"]


def _frequencies(c):
    """Rotations per position of each pair, in radians, float64."""
    rd = c["rope_dim"]
    f = c["base"] ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    elif c["scaling"] == "blend":  # a trained context of 8192; 1 rotation in it and fewer scaled, 4 and more kept
        keep = ((8192 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / c["factor"])
    return f


def _q40(x):
    """Rows of floats as 4-bit blocks: [..., D] -> [..., D/32, 18] bytes (a half, then 32 codes in 16 bytes)."""
    x = x.float().unflatten(-1, (-1, 32))
    top, low = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    d = (torch.where(top >= -low, top, low) / -8.0).clamp(-65504.0, 65504.0).half()
    inv = torch.where(d == 0, torch.zeros_like(top), 1.0 / d.float())
    code = ((x * inv).round() + 8.0).clamp(0, 15).to(torch.uint8)
    return torch.cat([d.view(torch.uint8), code[..., :16] | (code[..., 16:] << 4)], -1)


def _values(blocks):
    """The values of 4-bit blocks, in 32 bits: [..., D/32, 18] bytes -> [..., D]."""
    d = blocks[..., :2].contiguous().view(torch.float16).float()
    codes = torch.cat([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], -1).float() - 8.0
    return (codes * d).flatten(-2)


def _inputs(c, seed):
    """Everything of a case that is drawn from the seed, on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[c["type"]]
    nq, nk = _sizes(c)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = {}
    if c["op"] == "window":
        b, n, m = c["batch"], c["n"], c["m"]
        if c["strided"]:
            row = normal(b, n, nq + 2 * nk).to(t)
            s["q"], s["k"], s["v"] = row[..., :nq], row[..., nq:nq + nk], row[..., nq + nk:]
        else:
            s["q"], s["k"], s["v"] = (normal(b, r, w).to(t) for r, w in ((n, nq), (m, nk), (m, nk)))
        return s
    n = c["rows"] if c["op"] == "decode" else c["n"]
    # Projections as a layer's normed input gives them: queries and keys of unlike size before their norm.
    parts = [2.0 * normal(n, nq), 1.5 * normal(n, nk), normal(n, nk)]
    if c.get("strided"):
        row = torch.cat(parts, -1).to(t)
        s["q"], s["k"], s["v"] = row[:, :nq], row[:, nq:nq + nk], row[:, nq + nk:]
    else:
        s["q"], s["k"], s["v"] = (p.to(t) for p in parts)
    if c["norm"]:
        s["q_gamma"], s["k_gamma"] = (1.0 + 0.02 * normal(c["dim"]) for _ in range(2))
    if c.get("scattered"):
        s["pos"] = torch.randint(0, 131072, (n,), generator=g, device=DEV, dtype=torch.int32)
    if c["op"] == "decode":
        shape = (n, _context(c), c["kv_heads"], c["dim"])
        s["k_blocks"], s["v_blocks"] = _q40(normal(*shape)), _q40(normal(*shape))
    return s


def prepare(case, seed):
    c = dict(case)
    s = {"case": c} | _inputs(c, seed)
    n, (nq, nk) = c.get("rows") or c["n"], _sizes(c)
    if c["op"] == "window":
        pos0, lens = _spans(c)
        s["pos0"], s["lens"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (pos0, lens))
        s["out"] = torch.empty(c["batch"], n, nq, dtype=TYPES[c["type"]], device=DEV)
    else:
        if c["op"] == "decode":
            s["pos"] = torch.tensor(_positions(c), dtype=torch.int32, device=DEV)
        elif "pos" not in s:
            s["pos"] = torch.arange(c["pos0"], c["pos0"] + n, dtype=torch.int32, device=DEV)
        # The rotation of every position of the context, which a program makes once.
        places = torch.arange(131072 if c.get("scattered") else _context(c), dtype=torch.float64, device=DEV)
        turn = places[:, None] * _frequencies(c).to(DEV)
        s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
        out = TYPES[c["out"]]
        s["q_out"] = torch.empty(n, nq, dtype=TYPES[c["type"]] if c["op"] == "decode" else out, device=DEV)
        s["k_rows"], s["v_rows"] = (torch.empty(n, nk, dtype=out, device=DEV) for _ in range(2))
    if own:
        s["plan"] = _plan(c, s)
    return s


def _plan(c, s):
    """The package's handle for a case, with the cache of a decode case in it."""
    from ligguf_b200 import (KV_BF16, KV_F16, KV_F32, Kv4Cache, Kv4Config, QkRope, QkRopeConfig, RopeConfig,
                             WindowAttention, WindowConfig)
    kinds = {"f32": KV_F32, "f16": KV_F16, "bf16": KV_BF16}
    nq, nk = _sizes(c)
    heads = dict(n_heads=c["heads"], n_kv_heads=c["kv_heads"])
    row = nq + 2 * nk if c.get("strided") else 0
    if c["op"] == "window":
        return WindowAttention(WindowConfig(**heads, head_dim=c["dim"], window=c["window"], sinks=c["sinks"],
                                            in_type=kinds[c["type"]], out_type=kinds[c["type"]], q_stride=row,
                                            k_stride=row, v_stride=row))
    rope = RopeConfig(head_dim=c["dim"], rope_dim=c["rope_dim"], layout=c["layout"], base=c["base"],
                      scaling=c["scaling"], factor=c["factor"], orig_context=8192, low=1.0, high=4.0)
    if c["op"] == "rope":
        return QkRope(QkRopeConfig(rope=rope, **heads, qk_norm=c["norm"], in_type=kinds[c["type"]],
                                   out_type=kinds[c["out"]], q_stride=row, k_stride=row))
    n_seqs = c["rows"] if c["op"] == "decode" else 1
    cache = Kv4Cache(Kv4Config(rope=rope, **heads, n_layers=1, n_seqs=n_seqs, n_context=_context(c),
                               qk_norm=c["norm"], window=c.get("window", 0), sinks=c.get("sinks", 0),
                               in_type=kinds[c["type"]], rows_type=kinds[c["out"]], q_stride=row, k_stride=row,
                               v_stride=row))
    if c["norm"]:
        cache.set_qk_norm(0, s["q_gamma"].cpu().numpy(), s["k_gamma"].cpu().numpy())
    if c["op"] == "decode":
        cache.load_async(0, 0, n_seqs, 0, _context(c), s["k_blocks"], s["v_blocks"])
    return cache


# ---------------------------------------------------------------------------------------- plain forms
def _rms(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gamma


def _turn(x, cos, sin, c):
    """The leading rope_dim elements of every head rotated: x [n, heads, dim], cos and sin [n, rope_dim / 2]."""
    rd, (cos, sin) = c["rope_dim"], (cos[:, None], sin[:, None])
    y = x.clone()
    one, two = ((slice(0, rd // 2), slice(rd // 2, rd)) if c["layout"] == "halves" else
                (slice(0, rd, 2), slice(1, rd, 2)))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * cos - b * sin, a * sin + b * cos
    return y


def _heads(s, c):
    """Normed and rotated queries and keys, and the values, of a call's tokens: [n, heads, dim] in 32 bits."""
    q, k, v = (s[x].float().unflatten(-1, (-1, c["dim"])) for x in ("q", "k", "v"))
    if c["norm"]:
        q, k = _rms(q, s["q_gamma"]), _rms(k, s["k_gamma"])
    at = s["pos"].long().clamp(min=0)
    cos, sin = s["cos"][at], s["sin"][at]
    return _turn(q, cos, sin, c), _turn(k, cos, sin, c), v


def _softmax_sum(score, seen, v, eq):
    """Softmax over the last axis of the seen scores (a row that sees nothing gives zeros), times v."""
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.einsum(eq, p / torch.where(total == 0, 1.0, total), v)


def _plain_decode(s, c):
    q, k, v = _heads(s, c)
    out = TYPES[c["out"]]
    live = s["pos"] >= 0
    keys = torch.arange(_context(c), device=q.device)
    pos = s["pos"].long()[:, None]
    seen = (keys < pos) & ((keys > pos - c["window"]) | (keys < c["sinks"]) if c["window"] else (keys >= 0))
    q = q.unflatten(1, (c["kv_heads"], -1)) / math.sqrt(c["dim"])
    past = torch.einsum("rhgd,rjhd->rhgj", q, _values(s["k_blocks"]))
    score = torch.cat([past, torch.einsum("rhgd,rhd->rhg", q, k)[..., None]], -1)
    seen = torch.cat([seen, live[:, None]], -1)[:, None, None]
    o = _softmax_sum(score, seen, torch.cat([_values(s["v_blocks"]), v[:, None]], 1), "rhgj,rjhd->rhgd")
    rows = [torch.where(live[:, None, None], _values(_q40(x)), 0.0).flatten(1).to(out) for x in (k, v)]
    return {"out": o.flatten(1).to(TYPES[c["type"]]), "k_rows": rows[0], "v_rows": rows[1]}


def _plain_window(s, c):
    q, k, v = (s[x].float().unflatten(-1, (-1, c["dim"])) for x in ("q", "k", "v"))
    at = s["pos0"].long()[:, None, None] + torch.arange(c["n"], device=q.device)[:, None]
    keys = torch.arange(c["m"], device=q.device)
    seen = (keys <= at) & (keys < s["lens"].long()[:, None, None])
    if c["window"]:
        seen &= (keys > at - c["window"]) | (keys < c["sinks"])
    q = q.unflatten(2, (c["kv_heads"], -1)) / math.sqrt(c["dim"])
    score = torch.einsum("bihgd,bjhd->bhgij", q, k)
    o = _softmax_sum(score, seen[:, None, None], v, "bhgij,bjhd->bihgd")
    return o.flatten(2).to(TYPES[c["type"]])


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        return _run_own(s, c, op)
    if op == "window":
        return _plain_window(s, c)
    if op == "decode":
        return _plain_decode(s, c)
    q, k, v = _heads(s, c)
    out = TYPES[c["out"]]
    if op == "rope":
        return {"q": q.flatten(1).to(out), "k": k.flatten(1).to(out)}
    return {"q": q.flatten(1).to(out), "k_rows": _values(_q40(k)).flatten(1).to(out),
            "v_rows": _values(_q40(v)).flatten(1).to(out)}


def _run_own(s, c, op):
    plan = s["plan"]
    if op == "window":
        plan.attn_async(c["batch"], c["n"], c["m"], s["q"], s["k"], s["v"], s["out"], d_pos0=s["pos0"],
                        d_lens=s["lens"])
        return s["out"]
    if op == "decode":
        plan.decode_async(0, c["rows"], s["q"], s["k"], s["v"], s["q_out"], d_pos=s["pos"], k_rows=s["k_rows"],
                          v_rows=s["v_rows"])
        return {"out": s["q_out"], "k_rows": s["k_rows"], "v_rows": s["v_rows"]}
    if op == "rope":
        plan.run_async(c["n"], s["q"], s["k"], s["q_out"], s["k_rows"], pos0=c["pos0"],
                       d_pos=s["pos"] if c["scattered"] else None, q_gamma=s.get("q_gamma"),
                       k_gamma=s.get("k_gamma"))
        return {"q": s["q_out"], "k": s["k_rows"]}
    plan.append_async(0, 0, c["pos0"], c["n"], s["q"], s["k"], s["v"], q_out=s["q_out"], k_rows=s["k_rows"],
                      v_rows=s["v_rows"])
    return {"q": s["q_out"], "k_rows": s["k_rows"], "v_rows": s["v_rows"]}


# ---------------------------------------------------------------------------------------- work
def _seen_keys(at, keys, c):
    """Keys below `keys` that a query at position `at` sees."""
    below = min(at + 1, keys)
    if below <= 0:
        return 0
    if not c["window"]:
        return below
    first = max(0, at - c["window"] + 1)
    return max(0, below - first) + min(c["sinks"], first, below)


def work(case):
    c = case
    nq, nk = _sizes(c)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e = size[c["type"]]
    if c["op"] == "window":
        read = pairs = 0
        for p0, keys in zip(*_spans(c)):
            seen = [_seen_keys(p0 + i, keys, c) for i in range(c["n"])]
            pairs += sum(seen)
            first = max(0, p0 - c["window"] + 1) if c["window"] else 0
            last = min(p0 + c["n"], keys)
            read += max(0, last - first) + min(c["sinks"], first, max(last, 0)) if last > 0 else 0
        return {"bytes": c["batch"] * c["n"] * nq * 2 * e + read * 2 * nk * e, "flops": 4.0 * nq * pairs}
    f = size[c["out"]]
    if c["op"] == "rope":
        return {"bytes": c["n"] * (nq + nk) * (e + f) + (4 * c["n"] if c["scattered"] else 0),
                "flops": c["n"] * (nq + nk) * (6.0 if c["norm"] else 3.0)}
    packed = 18 / 32  # bytes of a cached value
    if c["op"] == "append":
        return {"bytes": c["n"] * ((nq + 2 * nk) * (e + f) + 2 * nk * packed),
                "flops": c["n"] * ((nq + nk) * (6.0 if c["norm"] else 3.0) + 8.0 * nk)}
    at = [p for p in _positions(c) if p >= 0]
    past = sum(_seen_keys(p, p, c) for p in at)
    return {"bytes": past * 2 * nk * packed + c["rows"] * (2 * nq * e + 2 * nk * (e + f)) + len(at) * 2 * nk * packed,
            "flops": 4.0 * nq * (past + len(at))}


# ---------------------------------------------------------------------------------------- in 64 bits
def _exact_blocks(blocks):
    """4-bit blocks in 64 bits, element by element of the block."""
    scale = blocks[..., :2].contiguous().view(torch.float16).double()
    out = torch.empty(*blocks.shape[:-1], 32, dtype=torch.float64, device=blocks.device)
    out[..., :16] = (blocks[..., 2:] % 16).double()
    out[..., 16:] = torch.div(blocks[..., 2:], 16, rounding_mode="floor").double()
    return ((out - 8) * scale).reshape(*blocks.shape[:-2], -1)


def _exact_round(x):
    """What a 4-bit cache holds of x, in 64 bits."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    big, small = y.max(-1).values, y.min(-1).values
    scale = (torch.where(big >= -small, big, small) / -8).half().double()[..., None]
    code = torch.where(scale == 0, 0.0, torch.round(y / torch.where(scale == 0, 1.0, scale)))
    return (code.clamp(-8, 7) * scale).reshape(x.shape)


def _exact_head(x, gamma, places, c):
    """x [n, width] normed by heads and rotated at `places`, as complex numbers: [n, heads, dim]."""
    x = x.double().reshape(x.shape[0], -1, c["dim"])
    if gamma is not None:
        x = gamma.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + 1e-6)
    rd = c["rope_dim"]
    turned, rest = x[..., :rd], x[..., rd:]
    z = (torch.complex(turned[..., 0::2].contiguous(), turned[..., 1::2].contiguous()) if c["layout"] == "adjacent" else
         torch.complex(*(h.contiguous() for h in turned.chunk(2, -1))))
    angle = places.double()[:, None, None] * _frequencies(c).to(x.device)
    z = z * torch.polar(torch.ones_like(angle), angle)
    turned = torch.view_as_real(z).flatten(-2) if c["layout"] == "adjacent" else torch.cat([z.real, z.imag], -1)
    return torch.cat([turned, rest], -1)


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    if c["op"] == "window":
        return _exact_window(s, c)
    if c["op"] == "decode":
        places = torch.tensor(_positions(c), device=DEV)
    else:
        places = s["pos"] if c.get("scattered") else c["pos0"] + torch.arange(c["n"], device=DEV)
    q = _exact_head(s["q"], s.get("q_gamma"), places.clamp(min=0), c)
    k = _exact_head(s["k"], s.get("k_gamma"), places.clamp(min=0), c)
    if c["op"] == "rope":
        return {"q": q.reshape(c["n"], -1), "k": k.reshape(c["n"], -1)}
    v = s["v"].double().reshape(k.shape)
    k_rows, v_rows = (_exact_round(x).reshape(x.shape[0], -1) for x in (k, v))
    if c["op"] == "append":
        return {"q": q.reshape(c["n"], -1), "k_rows": k_rows, "v_rows": v_rows}
    out = torch.zeros(c["rows"], *q.shape[1:], dtype=torch.float64, device=DEV)
    group = c["heads"] // c["kv_heads"]
    for r, p in enumerate(_positions(c)):
        if p < 0:
            k_rows[r], v_rows[r] = 0, 0
            continue
        keys = [j for j in range(p) if not c["window"] or j > p - c["window"] or j < c["sinks"]]
        keys = torch.tensor(keys, dtype=torch.long, device=DEV)
        kk = torch.cat([_exact_blocks(s["k_blocks"][r].index_select(0, keys)), k[r:r + 1]])
        vv = torch.cat([_exact_blocks(s["v_blocks"][r].index_select(0, keys)), v[r:r + 1]])
        for h in range(c["heads"]):
            w = torch.softmax(kk[:, h // group] @ q[r, h] * c["dim"] ** -0.5, 0)
            out[r, h] = w @ vv[:, h // group]
    return {"out": out.reshape(c["rows"], -1), "k_rows": k_rows, "v_rows": v_rows}


def _exact_window(s, c):
    d, group = c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], c["n"], c["heads"] * d, dtype=torch.float64, device=DEV)
    for b, (p0, keys) in enumerate(zip(*_spans(c))):
        if not keys:
            continue
        i = torch.arange(p0, p0 + c["n"], device=DEV)[:, None]
        j = torch.arange(keys, device=DEV)[None]
        hidden = j > i
        if c["window"]:
            hidden |= (j <= i - c["window"]) & (j >= c["sinks"])
        for h in range(c["heads"]):
            g = h // group
            a = s["q"][b, :, h * d:(h + 1) * d].double() @ s["k"][b, :keys, g * d:(g + 1) * d].double().T * d ** -0.5
            w = torch.softmax(a.masked_fill(hidden, -torch.inf), -1).masked_fill(hidden.all(-1, keepdim=True), 0.0)
            out[b, :, h * d:(h + 1) * d] = w @ s["v"][b, :keys, g * d:(g + 1) * d].double()
    return out
