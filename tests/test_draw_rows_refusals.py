"""Rows of draw states and numbers of continuations that the C++ host API refuses (no GPU)."""
from test_host_api import _run


def test_draw_rows_that_are_refused():
    out = _run("draw_rows_cpu_test")
    assert "ok   draw_rows_that_are_refused" in out and "ok   numbers_of_continuations_that_are_refused" in out
