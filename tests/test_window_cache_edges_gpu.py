"""Windowed attention and the 8-bit paged cache on the GPU, at the edges of their numerics and of
captured calls."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*shape, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).bfloat16()


# ------------------------------------------------------------------ windowed attention
@pytest.mark.parametrize("splits", [1, 2, 3, 8])
def test_rows_that_meet_nan_are_nan_however_the_keys_are_split(splits):
    """A NaN in a query, or in a key that it sees, makes the row and its lse NaN; the other
    rows are as without it."""
    from drivedit_b200.ops._ext import ext
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = _randn(1, 150, 2, 64), _randn(1, 2100, 2, 64), _randn(1, 2100, 2, 64)
    args = ("token", 1, 1500, 130, 1950)
    prev = ext().attn_fwd_set_kv_splits(splits)
    try:
        want, wl = window_attention(q, k, v, *args, return_lse=True)
        q2, k2 = q.clone(), k.clone()
        q2[0, 37, 1, 5] = math.nan
        k2[0, 2000, 0, 3] = math.nan     # seen by the queries from 2000 on
        k2[0, 470, 1, 9] = math.nan      # seen by the queries before 1970
        o, lse = window_attention(q2, k2, v, *args, return_lse=True)
    finally:
        ext().attn_fwd_set_kv_splits(prev)
    pos = torch.arange(1950, 2100, device="cuda")
    bad = torch.stack([pos >= 2000, (pos < 1970) | (pos == 1987)], 1)  # [T, H]
    assert bad.any(0).all() and not bad.all(0).any()
    assert o[0][bad].isnan().all() and lse[0].T[bad].isnan().all()
    assert torch.equal(o[0][~bad], want[0][~bad]) and torch.equal(lse[0].T[~bad], wl[0].T[~bad])


def test_status_clean():
    from drivedit_b200.ops._ext import check_device_status
    torch.cuda.synchronize()
    check_device_status()
