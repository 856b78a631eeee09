"""Rows of a pass of the 8-bit head that keeps no logits, without a GPU."""

import pytest

from bitnet_tt.lm_head import _pass_rows


@pytest.mark.parametrize("m", [1, 64, 65, 500, 1024, 1025, 65535])
@pytest.mark.parametrize("v", [1, 1000, 128256, 131072, 200000, 2097152, 1 << 24])
def test_a_pass_is_bounded_in_bytes(m, v):
    """The buffer of a pass is no more than 512 MiB, unless it is of 64 rows or fewer, which need none."""
    rows = _pass_rows(m, v)
    assert 1 <= rows <= min(m, 1024)
    assert rows <= 64 or rows * v * 4 <= 1 << 29
    assert rows == min(m, 1024) or v > 131072  # no shorter where 1024 rows fit
