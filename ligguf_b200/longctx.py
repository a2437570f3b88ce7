"""Long contexts: rotary positions and head norms in one pass, a 4-bit key/value cache with the decode
that attends over it, and windowed attention over 16-bit rows (thin wrappers over the C ABI).

A layer of a decoder runs them one after another: a prompt's projections go through ``QkRope`` (or
``Kv4Cache.append_async``, which also quantizes keys and values into the cache) and
``WindowAttention.attn_async``; each later token is one ``Kv4Cache.decode_async``.

Tensors are device memory: anything with ``data_ptr()`` (torch) or raw ints.  Calls are enqueued on
``stream`` (default: torch's current stream) and allocate nothing.  Errors raise ``LigGufAttnError``.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import Kv4Cfg, QkRopeCfg, RopeCfg, WindowCfg, check

__all__ = ["RopeConfig", "QkRopeConfig", "QkRope", "Kv4Config", "Kv4Cache", "WindowConfig", "WindowAttention"]

LAYOUTS = {"adjacent": _lib.ROPE_ADJACENT, "halves": _lib.ROPE_HALVES}
SCALINGS = {"none": _lib.ROPE_SCALE_NONE, "linear": _lib.ROPE_SCALE_LINEAR, "blend": _lib.ROPE_SCALE_BLEND}


def _p(x):
    return x if x is None or isinstance(x, int) else x.data_ptr()


_raw_stream = None


def _stream(stream, device):
    """The stream's handle; by default torch's current stream of the handle's device, asked for without making a
    Stream object (3 us, more than a small call's whole kernel)."""
    if stream is not None:
        return stream if isinstance(stream, int) else stream.cuda_stream
    global _raw_stream
    if _raw_stream is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda device: torch.cuda.current_stream(device).cuda_stream)
    return _raw_stream(device)


@dataclass
class RopeConfig:
    """Rotation of the leading ``rope_dim`` elements of a head (``ligguf_rope_cfg``)."""

    head_dim: int
    rope_dim: int
    layout: str = "adjacent"  # pairs (2i, 2i+1), or "halves": (i, i + rope_dim/2)
    base: float = 10000.0
    scaling: str = "none"     # "linear", or "blend": a ramp linear in the turns within orig_context
    factor: float = 1.0
    orig_context: int = 0
    low: float = 1.0
    high: float = 4.0
    magnitude: float = 0.0    # of the rotated elements; 0 = 1
    freq: np.ndarray | None = None  # rope_dim/2 inverse frequencies in place of base and scaling (other ramps: YaRN by pairs)

    def to_c(self):
        if self.layout not in LAYOUTS or self.scaling not in SCALINGS:
            raise ValueError(f"layout {self.layout!r} or scaling {self.scaling!r}")
        c = RopeCfg(head_dim=self.head_dim, rope_dim=self.rope_dim, layout=LAYOUTS[self.layout],
                    scaling=SCALINGS[self.scaling], base=self.base, factor=self.factor,
                    orig_context=self.orig_context, low=self.low, high=self.high, magnitude=self.magnitude)
        if self.freq is not None:
            f = np.ascontiguousarray(self.freq, dtype=np.float32)
            if f.size != self.rope_dim // 2:
                raise ValueError(f"freq has {f.size} values for rope_dim {self.rope_dim}")
            c.freq = f.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
            c._keep = f  # the table outlives the struct that points to it
        return c


class _Handle:
    """Owns one handle of the library."""

    _kind = ""

    def __init__(self, c):
        self.lib = _lib.load()
        self._h = ctypes.c_void_p()
        name = f"ligguf_cuda_{self._kind}_init"
        check(getattr(self.lib, name)(ctypes.byref(c), ctypes.byref(self._h)), name)

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            getattr(self.lib, f"ligguf_cuda_{self._kind}_free")(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass


@dataclass
class QkRopeConfig:
    rope: RopeConfig
    n_heads: int
    n_kv_heads: int
    qk_norm: bool = False
    rms_epsilon: float = 1e-6
    in_type: int = _lib.KV_F32
    out_type: int = _lib.KV_F32
    q_stride: int = 0
    k_stride: int = 0
    q_out_stride: int = 0
    k_out_stride: int = 0
    device: int = 0

    def to_c(self):
        rope = self.rope.to_c()
        c = QkRopeCfg(rope=rope, n_heads=self.n_heads, n_kv_heads=self.n_kv_heads, qk_norm=int(self.qk_norm),
                      rms_epsilon=self.rms_epsilon, in_type=self.in_type, out_type=self.out_type,
                      q_stride=self.q_stride, k_stride=self.k_stride, q_out_stride=self.q_out_stride,
                      k_out_stride=self.k_out_stride, device=self.device)
        c._keep = rope
        return c


class QkRope(_Handle):
    """Norm and rotation of query and key rows in one pass (ligguf_cuda_qk_rope_async)."""

    _kind = "qk_rope"

    def __init__(self, cfg: QkRopeConfig):
        self.cfg = cfg
        super().__init__(cfg.to_c())

    def run_async(self, n: int, q, k, q_out, k_out, pos0: int = 0, d_pos=None, q_gamma=None, k_gamma=None,
                  stream=None):
        """n tokens at pos0 + i, or at d_pos[i] (device int32)."""
        rc = self.lib.ligguf_cuda_qk_rope_async(self._h, n, pos0, _p(d_pos), _p(q), _p(k), _p(q_gamma), _p(k_gamma),
                                                _p(q_out), _p(k_out), _stream(stream, self.cfg.device))
        if rc:
            check(rc, "ligguf_cuda_qk_rope_async")


@dataclass
class Kv4Config:
    rope: RopeConfig
    n_layers: int
    n_seqs: int
    n_context: int
    n_heads: int
    n_kv_heads: int
    qk_norm: bool = False
    rms_epsilon: float = 1e-6
    window: int = 0
    sinks: int = 0
    scale: float = 0.0
    in_type: int = _lib.KV_F32
    rows_type: int = _lib.KV_F16
    q_stride: int = 0
    k_stride: int = 0
    v_stride: int = 0
    device: int = 0

    def to_c(self):
        rope = self.rope.to_c()
        c = Kv4Cfg(rope=rope, n_layers=self.n_layers, n_seqs=self.n_seqs, n_context=self.n_context,
                   n_heads=self.n_heads, n_kv_heads=self.n_kv_heads, qk_norm=int(self.qk_norm),
                   rms_epsilon=self.rms_epsilon, window=self.window, sinks=self.sinks, scale=self.scale,
                   in_type=self.in_type, rows_type=self.rows_type, q_stride=self.q_stride, k_stride=self.k_stride,
                   v_stride=self.v_stride, device=self.device)
        c._keep = rope
        return c


class Kv4Cache(_Handle):
    """A cache of 4-bit keys and values of n_seqs sequences, and the decode that attends over it."""

    _kind = "kv4"

    def __init__(self, cfg: Kv4Config):
        self.cfg = cfg
        super().__init__(cfg.to_c())

    def set_qk_norm(self, layer: int, q_gamma, k_gamma):
        """One layer's norm weights (host arrays of head_dim)."""
        qg = np.ascontiguousarray(q_gamma, dtype=np.float32)
        kg = np.ascontiguousarray(k_gamma, dtype=np.float32)
        if qg.size != self.cfg.rope.head_dim or kg.size != self.cfg.rope.head_dim:
            raise ValueError("norm weights do not match head_dim")
        check(self.lib.ligguf_cuda_kv4_set_qk_norm(self._h, layer, qg.ctypes.data, kg.ctypes.data),
              "ligguf_cuda_kv4_set_qk_norm")

    def append_async(self, layer: int, seq: int, pos0: int, n: int, q, k, v, q_out=None, k_rows=None, v_rows=None,
                     stream=None):
        """A prompt's n tokens into sequence ``seq``; the rotated queries and the rows as the cache holds them
        where an output is given."""
        rc = self.lib.ligguf_cuda_kv4_append_async(self._h, layer, seq, pos0, n, _p(q), _p(k), _p(v), _p(q_out),
                                                   _p(k_rows), _p(v_rows), _stream(stream, self.cfg.device))
        if rc:
            check(rc, "ligguf_cuda_kv4_append_async")

    def decode_async(self, layer: int, n_rows: int, q, k, v, out, pos: int = 0, d_pos=None, k_rows=None, v_rows=None,
                     stream=None):
        """One token of each of the first n_rows sequences, at ``pos`` or d_pos[r] (device int32, negative: idle)."""
        rc = self.lib.ligguf_cuda_kv4_decode_async(self._h, layer, n_rows, pos, _p(d_pos), _p(q), _p(k), _p(v),
                                                   _p(out), _p(k_rows), _p(v_rows), _stream(stream, self.cfg.device))
        if rc:
            check(rc, "ligguf_cuda_kv4_decode_async")

    def read_async(self, layer: int, seq: int, pos0: int, n: int, k_rows, v_rows, stream=None):
        """Cached positions as rows of ``rows_type``."""
        check(self.lib.ligguf_cuda_kv4_read_async(self._h, layer, seq, pos0, n, _p(k_rows), _p(v_rows),
                                                  _stream(stream, self.cfg.device)), "ligguf_cuda_kv4_read_async")

    def load_async(self, layer: int, seq0: int, n_seqs: int, pos0: int, n: int, k_blocks, v_blocks, stream=None):
        """Q4_0 blocks [n_seqs][n][n_kv_heads*head_dim/32][18 bytes] into the cache, bit for bit."""
        check(self.lib.ligguf_cuda_kv4_load_async(self._h, layer, seq0, n_seqs, pos0, n, _p(k_blocks), _p(v_blocks),
                                                  _stream(stream, self.cfg.device)), "ligguf_cuda_kv4_load_async")

    def store_async(self, layer: int, seq0: int, n_seqs: int, pos0: int, n: int, k_blocks, v_blocks, stream=None):
        """The same out of the cache."""
        check(self.lib.ligguf_cuda_kv4_store_async(self._h, layer, seq0, n_seqs, pos0, n, _p(k_blocks), _p(v_blocks),
                                                   _stream(stream, self.cfg.device)), "ligguf_cuda_kv4_store_async")

    def status(self, stream=None):
        """Waits for the stream; raises if a decode met a position beyond the context or gave up waiting."""
        check(self.lib.ligguf_cuda_kv4_status(self._h, _stream(stream, self.cfg.device)), "ligguf_cuda_kv4_status")


@dataclass
class WindowConfig:
    n_heads: int
    n_kv_heads: int
    head_dim: int
    window: int = 0  # 0 = plain causal
    sinks: int = 0
    scale: float = 0.0
    in_type: int = _lib.KV_BF16
    out_type: int = _lib.KV_BF16
    q_stride: int = 0
    k_stride: int = 0
    v_stride: int = 0
    q_batch_stride: int = 0
    k_batch_stride: int = 0
    v_batch_stride: int = 0
    device: int = 0
    round_weights: bool = False  # prompts: softmax weights rounded once to in_type, faster

    def to_c(self):
        return WindowCfg(**{f: getattr(self, f) for f, _ in WindowCfg._fields_})


class WindowAttention(_Handle):
    """Causal attention with a sliding window and visible first tokens (ligguf_cuda_window_attn_async)."""

    _kind = "window"

    def __init__(self, cfg: WindowConfig):
        self.cfg = cfg
        super().__init__(cfg.to_c())

    def attn_async(self, batch: int, n: int, m: int, q, k, v, out, d_pos0=None, d_lens=None, stream=None):
        """n queries a sequence over m rows of keys and values; query i at d_pos0[b] + i (default: the last of the
        sequence's d_lens[b], or m, keys)."""
        rc = self.lib.ligguf_cuda_window_attn_async(self._h, batch, n, m, _p(q), _p(k), _p(v), _p(d_pos0), _p(d_lens),
                                                    _p(out), _stream(stream, self.cfg.device))
        if rc:
            check(rc, "ligguf_cuda_window_attn_async")

    def status(self, stream=None):
        check(self.lib.ligguf_cuda_window_status(self._h, _stream(stream, self.cfg.device)), "ligguf_cuda_window_status")
