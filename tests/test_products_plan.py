"""How a dense product is cut, as the workspace query shows it: shares of K meet in it, 4 bytes an output and share."""
import ctypes as C

import pytest

from project_aeon_amd import capi, dense


def shares(tokens, in_dim, out_dim, gated=False):
    p = dense.Projection(1, in_dim, out_dim, 4 if gated else 0, 1 << 22, (1 << 23) if gated else None, in_dim, None, None, 7.0)
    need = capi.lib().aeon_linear_workspace_bytes(C.byref(p), tokens)
    per = 4 * tokens * out_dim * (2 if gated else 1)
    assert need % per == 0
    return need // per if need else 1


@pytest.mark.parametrize("in_dim,out_dim", [(7168, 28672), (7168, 65536), (4096, 14336), (2048, 8192)])
def test_a_full_window_of_128_tokens_is_cut_as_one_of_127(in_dim, out_dim):
    """The same tiles and weights: one more token in a window that has room for it changes neither."""
    assert shares(128, in_dim, out_dim) == shares(127, in_dim, out_dim)
    assert shares(128, in_dim, out_dim // 2, gated=True) == shares(127, in_dim, out_dim // 2, gated=True)
