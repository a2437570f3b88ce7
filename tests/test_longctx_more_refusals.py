"""More of the long-context operators' argument checks (CPU only: every call here returns before it touches a
device)."""
import pytest

from ligguf_b200 import _lib
from ligguf_b200.longctx import WindowConfig
from test_longctx_refusals import lib, refused  # noqa: F401 (lib is a fixture)


@pytest.mark.parametrize("value", [-1, 2])
def test_window_round_weights_is_a_truth_value(lib, value):  # noqa: F811
    refused(lib, "window", WindowConfig(4, 2, 128, round_weights=value), _lib.EINVAL, "round_weights")
