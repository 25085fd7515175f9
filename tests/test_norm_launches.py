"""The launches of the norm's rows, asked of their rule (csrc/dispatch.h through tests/hw/norms.hip, on the host)."""
import ctypes

import pytest

from routes import CUS, library


def launch(pieces, rows, codes):
    threads = ctypes.c_int()
    held = library().ckh_norm_launch(pieces, ctypes.c_int64(rows), int(codes), CUS, ctypes.byref(threads))
    return held, threads.value


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("rows", [1, CUS - 1, CUS, 6000, 32 * CUS - 1, 32 * CUS, 1 << 24])
def test_every_row_is_held_by_a_kernel_that_there_is(rows, codes):
    """A thread holds 1, 2, 4 or 8 pieces, which hold the row, and of several over half are the row's."""
    for pieces in range(1, 8193):
        held, threads = launch(pieces, rows, codes)
        assert held in (1, 2, 4, 8), pieces
        assert threads % 64 == 0 and 64 <= threads <= 1024 and held * threads >= pieces, pieces
        assert held == 1 or 2 * pieces > held * threads, pieces
