"""Arguments that the log-probability entry points refuse: the checks run on the host, before anything touches a device."""
import ctypes

import pytest

P = 4096  # an address that is aligned and never followed


@pytest.fixture(scope="module")
def hip():
    from rwkv_lightning_cuda_amd import hip
    hip.load()
    return hip


class Workspace:
    """What hip asks of a workspace."""

    def __init__(self, nbytes, ptr=P):
        self.nbytes, self.ptr = nbytes, ptr

    def __int__(self):
        return self.ptr


def norm(hip, **kw):
    a = dict(rows=2, C=64, x=P, res=P, w=P, b=P, q=P, scale=P)
    a.update(kw)
    hip.add_norm_q8(**a)


@pytest.mark.parametrize("change,message", [
    (dict(norm=2), "unknown norm"), (dict(rows=0), "rows"), (dict(rows=-1), "rows"), (dict(C=0), "multiple of 8"),
    (dict(C=12), "multiple of 8"), (dict(C=8200), "up to 8192"), (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(q=None), "NULL"),
    (dict(scale=None), "NULL"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=P + 2), "16 bytes"),
    (dict(res=P + 8), "16 bytes"), (dict(x_out=P + 4), "16 bytes"), (dict(q=P + 4), "8 bytes"), (dict(scale=P + 2), "4")])
def test_norm_refuses(hip, change, message):
    with pytest.raises(hip.RwkvHipError, match=message):
        norm(hip, **change)


def logprobs(hip, **kw):
    a = dict(rows=2, V=100, logits=P, tokens=P, workspace=Workspace(0), logprob=P, entropy=P, rank=P)
    a.update(kw)
    hip.token_logprobs(**a)


@pytest.mark.parametrize("change,message", [
    (dict(rows=0), "rows"), (dict(V=0), "V must"), (dict(V=1048577), "V must"), (dict(io=2), "element type"), (dict(logits=None), "NULL"),
    (dict(ld=99), "apart"), (dict(logits=P + 2), "misaligned"), (dict(logits=P + 1, io=0), "misaligned"), (dict(top_n=-1), "top_n"),
    (dict(top_n=65, top_ids=P, top_logprobs=P), "top_n"), (dict(top_n=1, top_ids=P), "two outputs"), (dict(tokens=None), "need tokens"),
    (dict(tokens=None, logprob=None), "need tokens"), (dict(logprob=None, entropy=None, rank=None), "no output"),
    (dict(tokens=P + 2), "4 bytes")])
def test_token_logprobs_refuses(hip, change, message):
    with pytest.raises(hip.RwkvHipError, match=message):
        logprobs(hip, **change)


def head(hip, **kw):
    a = dict(fmt=hip.FMT_W8, M=2, N=64, K=256, x=P, packed=P, scale=P, tokens=P, workspace=Workspace(1 << 30), logprob=P, entropy=P)
    a.update(kw)
    hip.linear_logprobs(**a)


@pytest.mark.parametrize("change,message", [
    (dict(fmt=2), "fp16 or int8"), (dict(fmt=7), "fp16 or int8"), (dict(fmt=0, x_scale=P), "int8 weights"), (dict(M=0), "M must"),
    (dict(N=48), "unsupported shape"), (dict(K=128), "unsupported shape"), (dict(K=16640), "K up to"), (dict(N=1048608), "N up to"),
    (dict(x=None), "NULL"), (dict(packed=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=P + 8), "16"), (dict(packed=P + 8), "16"),
    (dict(scale=P + 2), "8"), (dict(x_scale=P + 1), "4"), (dict(top_n=65, top_ids=P, top_logprobs=P), "top_n"),
    (dict(top_n=2), "two outputs"), (dict(tokens=None), "need tokens"), (dict(logprob=None, entropy=None), "no output"),
    (dict(workspace=None), "workspace"), (dict(workspace=Workspace(16)), "workspace"), (dict(workspace=Workspace(1 << 30, P + 8)), "workspace")])
def test_linear_logprobs_refuses(hip, change, message):
    with pytest.raises(hip.RwkvHipError, match=message):
        head(hip, **change)


def test_workspace_queries_refuse(hip):
    for args in ((0, 10, 0), (1, 0, 0), (1, 1048577, 0), (1, 10, 65), (1, 10, -1)):
        with pytest.raises(hip.RwkvHipError):
            hip.token_logprobs_workspace(*args)
    for args in ((2, 1, 64, 256, 0), (0, 0, 64, 256, 0), (0, 1, 63, 256, 0), (0, 1, 64, 255, 0), (0, 1, 64, 256, 65)):
        with pytest.raises(hip.RwkvHipError):
            hip.linear_logprobs_workspace(*args)
    with pytest.raises(hip.RwkvHipError):
        hip.linear_logprobs_workspace(hip.FMT_F16, 1, 64, 256, x_int8=True)
    assert hip.load().rwkv_hip_token_logprobs_workspace(ctypes.c_int(1), ctypes.c_int(10), ctypes.c_int(0), None) == -1
    # what is asked for is there for every size, the largest among them
    for rows, V, top in ((1, 1, 0), (1, 65536, 64), (4096, 1048576, 64)):
        assert hip.token_logprobs_workspace(rows, V, top) >= 0
    for M, N, K, top in ((1, 32, 256, 0), (1 << 20, 65536, 4096, 64), (1, 1048576, 16384, 64)):
        assert 0 < hip.linear_logprobs_workspace(hip.FMT_W8, M, N, K, top, x_int8=True) < 1 << 33
