"""Arguments at the ends of their ranges, as far as they are checked before any
device work."""
import ctypes

import pytest

from tributary_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_temperatures_whose_square_fp32_cannot_hold(lib):
    """T^2 is a factor of the divergence: below 2^-126 it would be zero, and a
    difference of logits over T infinite."""
    some = ctypes.c_void_p(1 << 21)

    def calls(t):
        args = (some, 0, 0, 10, some, some, some, 3, t, 1.0, 0.0, 1.0)  # no rows: nothing is launched
        return (lib.rt_distill_loss(*args, some, some, None), lib.rt_distill_loss_bwd(*args, some, some, some, None))

    for t in (1e-38, 1e-30, 1e-20, 2.0 ** -63.5, 2.0 ** 64):
        assert calls(t) == (_lib.RT_ERR_INVALID_ARGUMENT,) * 2, t
    for t in (2.0 ** -63, 1e-10, 1.0, 2.0 ** 63):
        assert calls(t) == (0, 0), t


def test_teacher_with_more_entries_than_categories_is_refused():
    from encoder_ref import make_cells
    assert make_cells(5, teacher_entries=16)["teacher_ids"].shape[-1] == 16
    with pytest.raises(ValueError, match="teacher_entries"):
        make_cells(5, teacher_entries=17)
