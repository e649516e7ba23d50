"""Sizes that the attention entries take, before they touch a GPU."""
import pytest

from gdnx_amd import _lib


@pytest.mark.parametrize("dtype", [_lib.DTYPE_BF16, _lib.DTYPE_F32])
@pytest.mark.parametrize("sizes", [
    (64, 32768, 32768, 32, 32, 128, 1024, 0), (64, 32769, 32769, 32, 32, 64, 64, 0),
    (512, 8192, 8192, 16, 16, 128, 0, 0), (64, 32768, 32768, 32, 32, 128, 1024, 16)], ids=str)
def test_a_forward_that_is_taken_has_a_backward(sizes, dtype):
    lib = _lib.load()
    assert lib.gdnx_win_attn_fwd_workspace_bytes(*sizes, dtype) >= 0
    B, Tq, _, Hq = sizes[:4]
    assert lib.gdnx_win_attn_bwd_workspace_bytes(*sizes, dtype) >= 4 * B * Tq * Hq


def test_grids_beyond_the_limit_are_refused():
    lib = _lib.load()
    too_many = (512, 1 << 20, 1 << 20, 32, 32, 128, 0, 0, _lib.DTYPE_BF16)        # 2^28 tiles of 64 tokens
    assert lib.gdnx_win_attn_fwd_workspace_bytes(*too_many) == -1
    assert lib.gdnx_win_attn_bwd_workspace_bytes(*too_many) == -1
