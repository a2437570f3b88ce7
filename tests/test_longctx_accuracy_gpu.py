"""How exact the long-context operators are, against plain numpy in 64 bits."""
import numpy as np
import pytest

from test_longctx_gpu import BF16, F16, F32, close, dev, run_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kin", [BF16, F16])
@pytest.mark.parametrize("n", [2, 200])
def test_window_many_small_weights_add_up(gpu, kin, n):
    """One key of weight 1 and value 0 before 4000 of weight e^-18 (2^-26, below fp16's range as it is) and value 1.
    A half of 2^-26 * 2^7 has five bits: within 2^-5.  (So many heads that no head's keys are split.)"""
    from ligguf_b200 import WindowConfig
    m, H, dim = 4001 + n, 300, 64
    q, k, v = np.zeros((1, n, H, dim)), np.zeros((1, m, H, dim)), np.ones((1, m, H, dim))
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 16.0, 1.125, 0.0
    cfg = WindowConfig(H, H, dim, scale=1.0, in_type=kin, out_type=F32)
    out = run_window(cfg, *(dev(x.astype(np.float32), kin) for x in (q, k, v)), None, None, 1, n, m)
    small = np.exp(-18.0) * (m - n + np.arange(n))
    want = np.broadcast_to((small / (1 + small))[None, :, None, None], out.shape)
    close(out, want, 0, 2.0 ** -5)
