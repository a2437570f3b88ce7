"""The long-context operators' argument checks and layouts (CPU only: every call here returns before it
touches a device)."""
import ctypes
import re

import numpy as np
import pytest

import longctx_ref as ref
from ligguf_b200 import RopeConfig, _lib
from ligguf_b200.longctx import Kv4Config, QkRopeConfig, WindowConfig
from test_abi import HEADER


@pytest.fixture(scope="module")
def lib():
    from ligguf_b200 import build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("name,struct", [("rope", _lib.RopeCfg), ("qk_rope", _lib.QkRopeCfg), ("kv4", _lib.Kv4Cfg),
                                         ("window", _lib.WindowCfg)])
def test_cfg_structs_match_header(name, struct):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct ligguf_%s_cfg \{(.*?)\} ligguf_%s_cfg;" % (name, name), text, re.S).group(1)
    fields = [f for d in body.split(";") for f in re.findall(r"(\w+)\s*(?:,|$)", d.strip())]
    assert fields == [f for f, _ in struct._fields_]


ROPE = dict(head_dim=128, rope_dim=128)


def refused(lib, kind, cfg, status, word):
    out = ctypes.c_void_p(1)
    c = cfg.to_c()
    assert getattr(lib, f"ligguf_cuda_{kind}_init")(ctypes.byref(c), ctypes.byref(out)) == status
    assert word in lib.ligguf_cuda_attn_last_error().decode()
    assert not out.value


@pytest.mark.parametrize("change,status,word", [
    (dict(head_dim=96), _lib.EUNSUPPORTED, "head_dim"), (dict(rope_dim=130), _lib.EINVAL, "rope_dim"),
    (dict(rope_dim=7), _lib.EINVAL, "rope_dim"), (dict(rope_dim=-2), _lib.EINVAL, "rope_dim"),
    (dict(base=0.0), _lib.EINVAL, "base"), (dict(base=float("nan")), _lib.EINVAL, "base"),
    (dict(scaling="linear", factor=0.5), _lib.EINVAL, "factor"),
    (dict(scaling="blend", factor=2.0), _lib.EINVAL, "blend"),
    (dict(scaling="blend", factor=2.0, orig_context=10, low=4.0, high=4.0), _lib.EINVAL, "blend"),
    (dict(magnitude=-1.0), _lib.EINVAL, "magnitude")])
def test_rope_refusals(lib, change, status, word):
    rope = RopeConfig(**(ROPE | change))
    refused(lib, "qk_rope", QkRopeConfig(rope=rope, n_heads=4, n_kv_heads=2), status, word)
    refused(lib, "kv4", Kv4Config(rope=rope, n_layers=1, n_seqs=1, n_context=8, n_heads=4, n_kv_heads=2), status, word)


def test_rope_python_refusals():
    with pytest.raises(ValueError):
        RopeConfig(64, 64, layout="rows").to_c()
    with pytest.raises(ValueError):
        RopeConfig(64, 64, scaling="more").to_c()
    with pytest.raises(ValueError):
        RopeConfig(64, 64, freq=np.ones(31)).to_c()


@pytest.mark.parametrize("change,word", [
    (dict(n_heads=0), "heads"), (dict(n_kv_heads=-1), "heads"), (dict(in_type=3), "types"), (dict(out_type=-1), "types"),
    (dict(q_stride=500), "q_stride"), (dict(k_stride=257), "k_stride"), (dict(q_out_stride=514), "q_out_stride"),
    (dict(k_out_stride=8), "k_out_stride"), (dict(qk_norm=True, rms_epsilon=-1.0), "rms_epsilon")])
def test_qk_rope_refusals(lib, change, word):
    cfg = QkRopeConfig(**(dict(rope=RopeConfig(**ROPE), n_heads=4, n_kv_heads=2) | change))
    refused(lib, "qk_rope", cfg, _lib.EINVAL, word)


@pytest.mark.parametrize("change,status,word", [
    (dict(n_heads=5), _lib.EINVAL, "multiple"), (dict(n_heads=6), _lib.EUNSUPPORTED, "supported: 1, 2, 4, 8"),
    (dict(n_layers=0), _lib.EINVAL, "positive"), (dict(n_seqs=0), _lib.EINVAL, "positive"),
    (dict(n_seqs=70000), _lib.EINVAL, "n_seqs"), (dict(n_context=0), _lib.EINVAL, "positive"),
    (dict(n_context=(1 << 30) + 1), _lib.EINVAL, "n_context"), (dict(window=-1), _lib.EINVAL, "window"),
    (dict(sinks=4), _lib.EINVAL, "sinks"), (dict(window=4, sinks=-1), _lib.EINVAL, "sinks"),
    (dict(scale=-1.0), _lib.EINVAL, "scale"), (dict(in_type=7), _lib.EINVAL, "types"),
    (dict(rows_type=7), _lib.EINVAL, "types"), (dict(v_stride=100), _lib.EINVAL, "v_stride")])
def test_kv4_refusals(lib, change, status, word):
    cfg = Kv4Config(**(dict(rope=RopeConfig(**ROPE), n_layers=1, n_seqs=1, n_context=64, n_heads=4, n_kv_heads=2) | change))
    refused(lib, "kv4", cfg, status, word)


@pytest.mark.parametrize("change,status,word", [
    (dict(n_heads=5), _lib.EINVAL, "multiple"), (dict(n_kv_heads=0), _lib.EINVAL, "positive"),
    (dict(head_dim=80), _lib.EUNSUPPORTED, "head_dim"), (dict(window=-1), _lib.EINVAL, "window"),
    (dict(sinks=1), _lib.EINVAL, "sinks"), (dict(scale=float("inf")), _lib.EINVAL, "scale"),
    (dict(in_type=_lib.KV_F32, out_type=_lib.KV_F32), _lib.EUNSUPPORTED, "in_type"),
    (dict(out_type=_lib.KV_F16), _lib.EUNSUPPORTED, "out_type"), (dict(q_stride=12), _lib.EINVAL, "q_stride"),
    (dict(k_stride=260), _lib.EINVAL, "k_stride"), (dict(v_batch_stride=4), _lib.EINVAL, "batch stride"),
    (dict(q_batch_stride=-8), _lib.EINVAL, "batch stride")])
def test_window_refusals(lib, change, status, word):
    refused(lib, "window", WindowConfig(**(dict(n_heads=4, n_kv_heads=2, head_dim=128) | change)), status, word)


def test_null_handles_and_arguments(lib):
    for kind in ("qk_rope", "kv4", "window"):
        assert getattr(lib, f"ligguf_cuda_{kind}_init")(None, None) == _lib.EINVAL
        assert getattr(lib, f"ligguf_cuda_{kind}_free")(None) == _lib.OK
    z = None
    assert lib.ligguf_cuda_qk_rope_async(z, 1, 0, z, z, z, z, z, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_set_qk_norm(z, 0, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_append_async(z, 0, 0, 0, 1, z, z, z, z, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_decode_async(z, 0, 1, 0, z, z, z, z, z, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_read_async(z, 0, 0, 0, 1, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_load_async(z, 0, 0, 1, 0, 1, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_store_async(z, 0, 0, 1, 0, 1, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_kv4_status(z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_window_attn_async(z, 1, 1, 1, z, z, z, z, z, z, z) == _lib.EINVAL
    assert lib.ligguf_cuda_window_status(z, z) == _lib.EINVAL


def test_tile_layout_gives_every_position_whole_bytes():
    """Restates the byte maps of ligguf_b200/csrc/kv4.cuh: a bijection from (position, element pair) onto the
    tile's code bytes, and the nibbles of a lane's word where an m16n8k16 A fragment wants them."""
    def key_byte(p, e):
        j, t, b = e >> 3, e >> 1 & 3, e & 1
        return (j >> 2) * 512 + ((p & 7) * 4 + t) * 16 + (j & 3) * 4 + 2 * b + (p >> 3)

    def value_byte(p, e):
        i, g = e >> 3, e & 7
        return (i >> 2) * 512 + (g * 4 + ((p & 7) >> 1)) * 16 + (i & 3) * 4 + 2 * (p & 1) + (p >> 3)

    for dim in (64, 128):
        for f in (key_byte, value_byte):
            assert sorted(f(p, e) for p in range(16) for e in range(dim // 2)) == list(range(8 * dim))
        for lane in range(32):
            g, t = lane >> 2, lane & 3
            for w in range(dim // 16):
                base = (w >> 2) * 512 + lane * 16 + (w & 3) * 4
                for reg in range(4):       # a0 (g, 2t..), a1 (g + 8, 2t..), a2 (g, 2t + 8..), a3 (g + 8, 2t + 8..)
                    for b in range(2):
                        row, col = g + 8 * (reg & 1), 2 * t + b + 8 * (reg >> 1)
                        # keys: nibble reg >> 1 of byte (reg & 1); columns are elements 16w + 4t + 2b + c
                        el = 16 * w + 4 * t + 2 * b + (reg >> 1)
                        assert key_byte(row, el >> 1) == base + 2 * b + (reg & 1) and el & 1 == reg >> 1
                        # values: nibble reg & 1 of byte (reg >> 1); rows are elements 16w + 2g, 16w + 2g + 1
                        el = 16 * w + 2 * g + (reg & 1)
                        assert value_byte(col, el >> 1) == base + 2 * b + (reg >> 1)


def test_reference_blocks():
    x = np.linspace(-3, 5, 64).astype(np.float32)
    b = ref.q40(x)
    assert b.shape == (2, 18)
    step = np.abs(b[:, :2].copy().view(np.float16).astype(float))
    err = np.abs(ref.q40_values(b).reshape(2, 32) - x.reshape(2, 32))
    assert (err <= step * 1.01).all()
