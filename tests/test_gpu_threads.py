"""Several threads on one backend: decode graphs, copies, allocations and continuations at the same time, through the C++ host API."""
import pytest

from test_host_api import _run

pytestmark = pytest.mark.gpu


def test_threads_of_one_process(gpu):
    out = _run("threads_gpu_test")
    for name in ("decode_graphs_beside_calls_of_other_threads", "decode_graphs_of_several_threads", "branches_of_several_threads_at_once"):
        assert "ok   " + name in out
