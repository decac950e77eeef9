"""The number of active sequences as the C interface takes it (no GPU needed)."""
from __future__ import annotations

import pytest

from asterq import _lib
from test_rows_ops_capi import BAD, ROWS, _call


@pytest.mark.parametrize("n,status", [(-1, BAD), (-(2**31), BAD)])
def test_a_negative_number_is_refused(n, status):
    assert _call("asterq_rows_attention", _lib.RowsAttentionParams, ROWS | dict(n_active=n)) == status
    assert b"rows_attention" in _lib.load().asterq_last_error()
