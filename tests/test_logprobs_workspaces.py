"""Workspaces of the log-probability entry points (no GPU)."""
import re

import pytest

from test_host_api import _run


def test_workspaces_for_any_count_of_cus():
    out = _run("logprobs_cpu_test")
    assert "ok   a_blocks_workspace_serves_every_shorter_block" in out


@pytest.fixture(scope="module")
def hip():
    from rwkv_lightning_cuda_amd import hip
    hip.load()
    return hip


@pytest.mark.parametrize("V", [1, 9000, 50277, 65536, 1048576])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_logprobs_of_fewer_rows_fit_the_workspace_of_more(hip, V, top):
    """A server that makes one workspace for its largest batch runs smaller ones in it."""
    sizes = [hip.token_logprobs_workspace(rows, V, top) for rows in range(1, 500)]
    assert sizes == sorted(sizes)
    assert hip.token_logprobs_workspace(1 << 20, V, top) >= sizes[-1]


ADDRESS = 4096  # aligned and never followed: the call is refused first


class NoWorkspace:
    nbytes = 0

    def __int__(self):
        return ADDRESS


def head_needs(hip, fmt, M, N, K, top, x_int8):
    """What the call itself asks for, out of its refusal."""
    with pytest.raises(hip.RwkvHipError, match="workspace of") as e:
        hip.linear_logprobs(fmt, M, N, K, ADDRESS, ADDRESS, ADDRESS, ADDRESS, NoWorkspace(), x_scale=ADDRESS if x_int8 else None, logprob=ADDRESS,
                            top_n=top, top_ids=ADDRESS if top else None, top_logprobs=ADDRESS if top else None)
    return int(re.search(r"workspace of (\d+) bytes", str(e.value)).group(1))


@pytest.mark.parametrize("fmt,x_int8", [(0, False), (1, False), (1, True)])
@pytest.mark.parametrize("N", [32, 2080, 65536, 200032, 1048576])
@pytest.mark.parametrize("top", [0, 1, 5, 64])
def test_heads_of_fewer_rows_fit_the_workspace_of_more(hip, fmt, x_int8, N, top):
    rows = (1, 2, 4, 5, 16, 17, 32, 33, 64, 128, 129, 192, 193, 256, 257, 333, 512, 700, 768, 1500, 1700, 2048, 2049, 8192, 8193, 100000)
    for K in (256, 1024, 4096, 16384):
        sizes = [hip.linear_logprobs_workspace(fmt, M, N, K, top, x_int8=x_int8) for M in rows]
        needs = [head_needs(hip, fmt, M, N, K, top, x_int8) for M in rows]
        assert sizes == sorted(sizes), K
        assert all(need <= size for need, size in zip(needs, sizes)), K


@pytest.mark.parametrize("fmt,x_int8", [(0, False), (1, True)])
@pytest.mark.parametrize("N", [32, 2048, 65536, 200032, 262144, 524288, 1048576])
def test_head_workspaces_keep_within_what_is_documented(hip, fmt, x_int8, N):
    size = lambda M, K, top: hip.linear_logprobs_workspace(fmt, M, N, K, top, x_int8=x_int8)  # noqa: E731
    for K in (256, 4096, 16384):
        for M in (1, 32, 33, 600, 8192, 8193, 1 << 20):
            assert size(M, K, 0) <= 45e6
            few = min(M, 32) * N * 4 + 3e6      # (their logits, and the sums of at most 256 parts)
            assert size(M, K, 1) <= max(45e6, few)
            for top in (2, 64):
                assert size(M, K, top) <= (0.7e9 if N <= 524288 else 1.11e9)
