"""A long conversation through the long-context operators, as a serving loop runs them.

A synthetic decoder layer stack (random projections in place of weights; heads, rotation and norms of the
32/8-head, head_dim 128 layout) takes a prompt in chunks, then a checked draft, then single tokens:

  prompt   Kv4Cache.append_async   norms, rotates and quantizes a chunk into the 4-bit cache, and hands out its
                                   queries and the rows as the cache holds them
           WindowAttention         the chunk's queries over those rows: sliding window and visible first tokens
  draft    QkRope                  norms and rotates a few proposed tokens
           WindowAttention         all of them at once over the rows so far
  tokens   Kv4Cache.decode_async   one launch a layer and token

    python examples/long_context.py [--prompt 3000] [--chunk 700] [--tokens 8]

Every result of the last layer is checked against plain torch in 64 bits on what the cache holds.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def attend(q, k, v, pos, window, sinks):
    """q [n, H, D] at positions pos [n] over rows k, v [m, Hk, D], in 64 bits."""
    import torch
    n, H, D = q.shape
    k, v = (x.double().repeat_interleave(H // k.shape[1], 1) for x in (k, v))
    j = torch.arange(k.shape[0], device=q.device)
    seen = (j <= pos[:, None]) & ((j > pos[:, None] - window) | (j < sinks))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / D ** 0.5
    return torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -torch.inf), -1), v)


def run(prompt=3000, chunk=700, tokens=8, draft=4, layers=2, heads=32, kv_heads=8, dim=128, window=1024, sinks=4, seed=0):
    """Returns the largest error of each stage, relative to the largest value of its result."""
    import torch
    from ligguf_b200 import (KV_BF16, KV_F32, Kv4Cache, Kv4Config, QkRope, QkRopeConfig, RopeConfig, WindowAttention,
                             WindowConfig)

    g = torch.Generator(device="cuda").manual_seed(seed)
    total = prompt + max(tokens, draft)
    nq, nk, row = heads * dim, kv_heads * dim, (heads + 2 * kv_heads) * dim
    # A context four times the trained one: frequencies blended by wavelength, logits a little larger for it.  (A model
    # whose ramp runs over the pairs' indices passes its own table: freq=.)
    rope = RopeConfig(dim, dim, "halves", base=1e6, scaling="blend", factor=4.0, orig_context=8192, low=1.0, high=32.0,
                      magnitude=1.1386)
    layout = dict(n_heads=heads, n_kv_heads=kv_heads)
    cache = Kv4Cache(Kv4Config(rope=rope, **layout, n_layers=layers, n_seqs=1, n_context=total, qk_norm=True,
                               window=window, sinks=sinks, in_type=KV_F32, rows_type=KV_BF16, q_stride=row,
                               k_stride=row, v_stride=row))
    turn = QkRope(QkRopeConfig(rope=rope, **layout, qk_norm=True, in_type=KV_F32, out_type=KV_BF16, q_stride=row,
                               k_stride=row))
    attn = WindowAttention(WindowConfig(**layout, head_dim=dim, window=window, sinks=sinks, in_type=KV_BF16,
                                        out_type=KV_F32))
    gammas = [1.0 + 0.02 * torch.randn(2, dim, generator=g, device="cuda") for _ in range(layers)]
    for layer, w in enumerate(gammas):
        cache.set_qk_norm(layer, w[0].cpu().numpy(), w[1].cpu().numpy())
    # Per layer, the rows of keys and values in 16 bits that a prompt's queries attend over.
    keys, values = (torch.zeros(layers, total, nk, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def projections(n):  # q, k and v of n tokens side by side, as one fused projection writes them
        return torch.randn(n, row, generator=g, device="cuda")

    def error(got, want):
        return float((got.double().reshape(want.shape) - want).abs().max() / want.abs().max())

    errors = {}
    for pos0 in range(0, prompt, chunk):
        n = min(chunk, prompt - pos0)
        for layer in range(layers):
            x = projections(n)
            q = torch.empty(n, nq, dtype=torch.bfloat16, device="cuda")
            out = torch.empty(n, nq, device="cuda")
            cache.append_async(layer, 0, pos0, n, x, x[:, nq:], x[:, nq + nk:], q_out=q,
                               k_rows=keys[layer, pos0:], v_rows=values[layer, pos0:])
            attn.attn_async(1, n, pos0 + n, q, keys[layer], values[layer], out)
        want = attend(q.view(n, heads, dim), keys[-1, :pos0 + n].view(-1, kv_heads, dim),
                      values[-1, :pos0 + n].view(-1, kv_heads, dim), torch.arange(pos0, pos0 + n, device="cuda"), window, sinks)
        errors["prompt"] = max(errors.get("prompt", 0.0), error(out, want))

    # A draft: its rows go behind the prompt's without entering the cache.
    x = projections(draft)
    q = torch.empty(draft, nq, dtype=torch.bfloat16, device="cuda")
    k, v = keys[-1].clone(), values[-1].clone()
    turn.run_async(draft, x, x[:, nq:], q, k[prompt:], pos0=prompt, q_gamma=gammas[-1][0], k_gamma=gammas[-1][1])
    v[prompt:prompt + draft] = x[:, nq + nk:].bfloat16()
    out = torch.empty(draft, nq, device="cuda")
    attn.attn_async(1, draft, prompt + draft, q, k, v, out)
    errors["draft"] = error(out, attend(q.view(draft, heads, dim), k[:prompt + draft].view(-1, kv_heads, dim),
                                        v[:prompt + draft].view(-1, kv_heads, dim),
                                        torch.arange(prompt, prompt + draft, device="cuda"), window, sinks))

    # Single tokens; the position lies on the device, so a captured step can be replayed.
    pos = torch.full((1,), prompt, dtype=torch.int32, device="cuda")
    out = torch.empty(1, nq, device="cuda")
    exact = Kv4Cache(Kv4Config(rope=rope, **layout, n_layers=1, n_seqs=1, n_context=total, rows_type=KV_F32))
    rows = [torch.empty(total, nk, device="cuda") for _ in range(2)]
    blocks = [torch.empty(1, total, nk // 32, 18, dtype=torch.uint8, device="cuda") for _ in range(2)]
    full = QkRope(QkRopeConfig(rope=rope, **layout, qk_norm=True, q_stride=row, k_stride=row))
    fq, fk = torch.empty(1, nq, device="cuda"), torch.empty(1, nk, device="cuda")
    for step in range(tokens):
        p = prompt + step
        for layer in range(layers):
            x = projections(1)
            cache.decode_async(layer, 1, x, x[:, nq:], x[:, nq + nk:], out, d_pos=pos)
        # What the cache holds below p, and the token's own key and value, unquantized.
        cache.store_async(layers - 1, 0, 1, 0, total, *blocks)
        exact.load_async(0, 0, 1, 0, total, *blocks)
        exact.read_async(0, 0, 0, total, *rows)
        full.run_async(1, x, x[:, nq:], fq, fk, pos0=p, q_gamma=gammas[-1][0], k_gamma=gammas[-1][1])
        kk, vv = (r[:p + 1].clone() for r in rows)
        kk[p], vv[p] = fk[0], x[0, nq + nk:]
        want = attend(fq.view(1, heads, dim), kk.view(-1, kv_heads, dim), vv.view(-1, kv_heads, dim), pos.long(), window, sinks)
        errors["tokens"] = max(errors.get("tokens", 0.0), error(out, want))
        pos += 1
    cache.status()
    attn.status()
    return errors


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=3000)
    ap.add_argument("--chunk", type=int, default=700)
    ap.add_argument("--tokens", type=int, default=8)
    a = ap.parse_args(argv)
    errors = run(a.prompt, a.chunk, a.tokens)
    for stage, e in errors.items():
        print(f"{stage:8s} largest error {e:.2e} of the largest value")


if __name__ == "__main__":
    main()
