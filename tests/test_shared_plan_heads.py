"""A shared plan holds rows and head groups: the launch takes it for its own row and
head counts alone. Every refusal comes before a device is reached."""
import ctypes

import numpy as np
import pytest

from kunserve_amd import _lib

from test_shared_plan import plan_of, rows


def decode(info, heads, kv_heads, seqs):
    buf = np.zeros(64, np.uint8)
    at = -(-buf.ctypes.data // 16) * 16
    three = _lib.Tensor3(at, 128 * heads, 128)
    pool = _lib.KVPool(k=at, v=at, num_pages=1, page_stride=1 << 40, layer_stride=1 << 39,
                       head_stride=1 << 38, token_stride=128, num_layers=1, num_kv_heads=kv_heads,
                       page_size=16, head_dim=128, dtype=0)
    table = _lib.PageTable(at, at, at, seqs)
    # a workspace that is too small: what passes the checks before it is refused there
    _lib.call("kunserve_shared_decode", ctypes.byref(pool), 0, ctypes.byref(table), None,
              ctypes.byref(three), ctypes.byref(three), heads, 1.0, at, ctypes.byref(info), None, 0,
              None)


# the same group size of 4 (2, 1) each
@pytest.mark.parametrize("made,used", [((16, 4), (8, 2)), ((8, 2), (16, 4)), ((8, 4), (4, 2)),
                                       ((4, 4), (2, 2)), ((32, 2), (16, 1))])
@pytest.mark.parametrize("min_bytes", [0, 1 << 40])
def test_other_head_counts_are_refused(made, used, min_bytes):
    info, _ = plan_of(rows(4, [1] * 3), [70, 70, 70], *made, 16, 128, min_bytes=min_bytes)
    assert info.num_segments == (min_bytes == 0)
    with pytest.raises(_lib.KunserveError, match=f"made for {made[0]} query heads on {made[1]}"):
        decode(info, *used, 3)


@pytest.mark.parametrize("seqs", [0, 2, 4])
def test_other_row_counts_are_refused(seqs):
    info, _ = plan_of(rows(4, [1] * 3), [70, 70, 70], 8, 2, 16, 128)
    with pytest.raises(_lib.KunserveError, match="made for 3 rows"):
        decode(info, 8, 2, seqs)


def test_its_own_counts_pass_on():
    info, _ = plan_of(rows(4, [1] * 3), [70, 70, 70], 8, 2, 16, 128)
    with pytest.raises(_lib.KunserveError, match="workspace holds") as e:
        decode(info, 8, 2, 3)
    assert e.value.code == _lib.ENOSPC
