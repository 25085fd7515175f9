"""Where shared attention's workgroups make the plan themselves, asked of the rule (csrc/dispatch.h through tests/hw/shared.hip, on
the host): where that measured faster than a launch for it."""
import ctypes

import pytest

from routes import CUS, library


@pytest.mark.parametrize("dim,slots,itself", [(64, 976, True), (64, 1025, False), (96, 690, True), (96, 874, True), (128, 774, True), (128, 960, True),
                                              (128, 1025, False), (256, 96, True), (256, 576, True), (256, 636, True), (256, 752, False),
                                              (256, 864, False), (256, 960, False), (256, 976, False)])
def test_as_measured(dim, slots, itself):
    assert library().ckh_shared_plans_itself(ctypes.c_int64(5), ctypes.c_int64(slots), dim, CUS) == itself


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_no_more_spans_than_a_wave_plans(dim):
    assert library().ckh_shared_plans_itself(ctypes.c_int64(64), ctypes.c_int64(100), dim, CUS)
    assert not library().ckh_shared_plans_itself(ctypes.c_int64(65), ctypes.c_int64(100), dim, CUS)
