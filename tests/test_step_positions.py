"""Positions of their own are a kunserve_rotary's: a layer with them and a step's plain
frequencies is refused by the C entry, before anything is launched."""
import ctypes

import numpy as np
import pytest

from kunserve_amd import _lib


def layer(positions, inv_freq, rotary):
    buf = np.zeros(64, np.uint8)
    at = -(-buf.ctypes.data // 16) * 16
    step, extras = _lib.Step(), _lib.StepExtras()
    extras.positions_dev = at if positions else None
    io = _lib.STEP_IO.pack(*([at, 64, 64] * 4), at if inv_freq else 0, 0)
    rot = ctypes.byref(_lib.Rotary(at, 16, 0, 1.0)) if rotary else None
    _lib.call("kunserve_attention_step_with", ctypes.byref(step), ctypes.byref(extras), 0, io, rot,
              None)


def test_positions_with_plain_frequencies():
    with pytest.raises(_lib.KunserveError, match="positions need a rotary"):
        layer(True, True, False)


@pytest.mark.parametrize("case", [(True, True, True), (True, False, True), (True, False, False),
                                  (False, True, False)])
def test_what_passes_on(case):
    """To the check of a pool, which is a null one here."""
    with pytest.raises(_lib.KunserveError) as e:
        layer(*case)
    assert "positions" not in str(e.value)
