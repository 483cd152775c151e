"""How texts are split into calls when they are scored (tests/cpp/score_cpu_test.cpp; no GPU)."""
from test_host_api import _run


def test_texts_are_scored_in_groups():
    out = _run("score_cpu_test")
    assert "ok   many_texts_go_in_groups" in out
