"""Workspaces of the log-probability entry points (no GPU)."""
from test_host_api import _run


def test_workspaces_for_any_count_of_cus():
    out = _run("logprobs_cpu_test")
    assert "ok   a_blocks_workspace_serves_every_shorter_block" in out
