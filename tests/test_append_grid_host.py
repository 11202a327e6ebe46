"""ssq_append checks a search grid before it writes anything (host code; no GPU call is made): the same grid is refused
for few tokens and for many, and by the workspace query."""

import ctypes

import pytest

from sunshape_amd import _native as N
from test_step_host import ALIGNED, _append_args


def _args(seq_len, need=0, **enc):
    a = _append_args(block_dim=2, n_blocks=32, seq_len=seq_len)
    a.enc.grid, a.enc.grid_bytes = ALIGNED, N.lib().ssq_encode_grid_bytes(ctypes.byref(a.enc)) + need
    for k, v in enc.items():
        setattr(a.enc, k, v)
    return a


@pytest.mark.parametrize("seq_len", [1, 16384])
@pytest.mark.parametrize("bad, word", [(dict(need=-1), "grid"), (dict(grid_bytes=0), "grid"), (dict(grid=ALIGNED + 8), "16-byte aligned")])
def test_grids_that_do_not_fit(seq_len, bad, word):
    a = _args(seq_len, **bad)
    assert N.lib().ssq_append_workspace_size(ctypes.byref(a)) == 0
    assert N.lib().ssq_append(ctypes.byref(a), ALIGNED, 1 << 40, None) == N.SSQ_ERR_INVALID
    assert word.encode() in N.lib().ssq_last_error()


def test_grids_that_are_not_used():
    """Another block dim, a block metric, the direct distance, the exact scan: the grid is not looked at, as in ssq_encode."""
    lib = N.lib()
    size = lib.ssq_append_workspace_size(ctypes.byref(_args(16384)))
    assert size == 2 * 16384 * 8
    for kw in (dict(block_dim=4, n_blocks=16), dict(metric=ALIGNED), dict(direct_dist=1), dict(kernel=1)):
        a = _args(1 << 21, need=-1, **kw)
        assert lib.ssq_append_workspace_size(ctypes.byref(a)) == 2 * (1 << 21) * 8, kw
