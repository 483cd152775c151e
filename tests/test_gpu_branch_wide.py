"""Rows of states wider than one launch of copy_rows numbers, through the C++ host API."""
import pytest

from test_host_api import _run

pytestmark = pytest.mark.gpu


def test_states_of_many_rows(gpu):
    out = _run("branch_wide_gpu_test")
    assert "ok   slices_of_a_wide_state" in out and "ok   rows_of_a_wide_state" in out
