"""Session.score: a forward pass with the log probability of given tokens at every position, and the host API above it."""
import numpy as np
import pytest

from test_gpu_logprobs import STEP, check_logprobs, ref_logprobs, ref_norm
from test_host_api import _run

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -11  # half a step of fp16


def dims_of(V=2048):
    from rwkv_lightning_cuda_amd.model import ModelDims
    return ModelDims(L=2, C=256, H=4, F=1024, V=V, Rw=32, Ra=32, Rg=64, Rv=16)


_MODELS = {}


def model_of(hip, fmt, V=2048):
    from rwkv_lightning_cuda_amd.model import HipModel, synth_weights
    if (fmt, V) not in _MODELS:
        weights = synth_weights(dims_of(V), 21)
        _MODELS[fmt, V] = (weights, HipModel.from_host_weights(dims_of(V), weights, fmt))
    return _MODELS[fmt, V]


def head_of(hip, model, dims):
    """The head's weights in 64 bits, as the model holds them."""
    mat = model.mats[-1, hip.M_HEAD]
    if mat.fmt == hip.FMT_F16:
        return mat.data.numpy().astype(np.float64)
    w = hip.DeviceArray((dims.V, dims.C), np.float16)
    if mat.fmt == hip.FMT_W8:
        return mat.data.numpy().astype(np.float64) * mat.scale.numpy().astype(np.float64)[:, None]
    q, zp = mat.data.numpy(), mat.zp.numpy().astype(np.float64)
    codes = np.empty((dims.V, dims.C))
    codes[:, 0::2], codes[:, 1::2] = q & 15, q >> 4
    return (codes - np.repeat(zp, 128, axis=1)) * np.repeat(mat.scale.numpy().astype(np.float64), 128, axis=1)


def run_score(hip, session, state, tokens, targets, top, logits=None, act_int8=False):
    B, T = tokens.shape
    out = dict(logprob=hip.DeviceArray.zeros((B * T,), np.float32), entropy=hip.DeviceArray.zeros((B * T,), np.float32))
    ids, tops = hip.DeviceArray.zeros((B * T, top), np.int32), hip.DeviceArray.zeros((B * T, top), np.float32)
    session.score(tokens, targets, state, out["logprob"], out["entropy"], top, ids if top else None, tops if top else None, logits, act_int8)
    got = {n: v.numpy() for n, v in out.items()}
    if top:
        got.update(ids=ids.numpy(), tops=tops.numpy())
    return got


@pytest.mark.parametrize("fmt,V,act_int8", [(0, 2048, False), (1, 2048, False), (1, 2048, True), (2, 2048, False), (0, 2052, False), (1, 2052, False)])
@pytest.mark.parametrize("B,T,top,wkv_fp16", [(1, 1, 3, False), (2, 1, 0, True), (1, 7, 5, False), (3, 33, 0, False), (2, 100, 4, True), (5, 64, 1, False)])
def test_score_is_the_norm_and_the_head_of_every_position(gpu, fmt, V, act_int8, B, T, top, wkv_fp16):
    """x1 + cm, what the layers leave, is read back; the norm and the head over it in 64 bits."""
    from rwkv_lightning_cuda_amd.model import Session, State
    hip = gpu
    dims = dims_of(V)
    weights, model = model_of(hip, fmt, V)
    rng = np.random.default_rng(B * 100 + T)
    tokens, targets = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T))
    targets[B - 1, T // 2] = -1
    session, state, plain = Session(model), State(dims, B, wkv_fp16), State(dims, B, wkv_fp16)
    logits = hip.DeviceArray.zeros((B, V), np.float32)
    got = run_score(hip, session, state, tokens, targets, top, logits, act_int8)
    x1, cm = session.debug_buffer("x1", (B * T, dims.C)), session.debug_buffer("cm", (B * T, dims.C))
    y = ref_norm(x1, cm, weights["ln_out_w"], weights["ln_out_b"], False)[1]
    w = head_of(hip, model, dims)
    z = y @ w.T
    if act_int8:    # half a code, and the code's own error (a few steps of fp32)
        slack = (np.abs(y).max(axis=1) / 254 * 1.001)[:, None] * np.abs(w).sum(axis=1)[None, :]
    else:           # half a step of fp16 per value, sums eight at a time
        slack = (HALF * 1.01 + (dims.C / 8 + 8) * STEP) * (np.abs(y) @ np.abs(w).T)
        if fmt == hip.FMT_W4 or V % 32:
            slack = slack + HALF * np.abs(z) * 1.01
    slack = slack.max()
    ref = ref_logprobs(z, targets.ravel(), top)
    if top:
        ids = got.pop("ids")
        for r in range(B * T):
            assert np.all(np.abs(z[r][ids[r]] - np.sort(z[r])[::-1][:top]) <= 2 * slack)
    check_logprobs(got, ref, V, slack=slack)
    # the pass itself is forward()'s: logits and state bit for bit
    want = hip.DeviceArray.zeros((B, V), np.float32)
    other = Session(model)
    other.set_graph(False)
    other.forward(tokens, plain, want)
    for a, b in ((logits, want), (state.shift, plain.shift), (state.wkv, plain.wkv), (state.elapsed, plain.elapsed)):
        a, b = a.numpy(), b.numpy()
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    session.close()
    other.close()


def test_a_text_in_several_calls_between_other_work(gpu):
    """Chunks of a text with the state between them, a larger call and decode steps of the same session in between; again, bit for bit."""
    from rwkv_lightning_cuda_amd.model import Session, State
    hip = gpu
    dims = dims_of()
    _, model = model_of(hip, hip.FMT_W8)
    rng = np.random.default_rng(4)
    text = rng.integers(0, dims.V, (1, 61))
    tokens, targets = text[:, :-1], text[:, 1:]
    session = Session(model)
    logits = hip.DeviceArray.zeros((1, dims.V), np.float32)
    runs = []
    for _ in range(2):
        state, parts = State(dims, 1), []
        for i in range(0, 60, 20):
            parts.append(run_score(hip, session, state, tokens[:, i:i + 20], targets[:, i:i + 20], 3))
            big = State(dims, 4)
            run_score(hip, session, big, rng.integers(0, dims.V, (4, 50)), rng.integers(0, dims.V, (4, 50)), 0)
            mark = State(dims, 1)
            session.decode_greedy(np.array([5]), 4, mark, logits)
        runs.append({n: np.concatenate([p[n] for p in parts]) for n in parts[0]})
    for name in runs[0]:
        assert np.array_equal(runs[0][name].view(np.uint32), runs[1][name].view(np.uint32))
    whole = run_score(hip, session, State(dims, 1), tokens, targets, 3)
    # other launches, fp16 activations: hundredths
    assert np.abs(whole["logprob"] - runs[0]["logprob"]).max() <= 0.05
    session.close()


def test_score_refuses(gpu):
    from rwkv_lightning_cuda_amd.model import Session, State
    hip = gpu
    dims = dims_of()
    session = Session(model_of(hip, hip.FMT_F16)[1])
    state = State(dims, 1)
    out = hip.DeviceArray((4,), np.float32)
    ones = np.ones((1, 2), np.int64)
    for tokens, targets, kw, message in ((ones * dims.V, ones, {}, "token id"), (ones, ones * dims.V, {}, "target id"), (ones, -2 * ones, {}, "target id"),
                                         (ones, None, {}, "need tokens"), (ones, ones, dict(act_int8=True), "int8 head"),
                                         (ones, ones, dict(top_n=65), "top_n"), (ones, ones, dict(top_n=1), "two outputs")):
        with pytest.raises(hip.RwkvHipError, match=message):
            session.score(tokens, targets, state, out, **kw)
    with pytest.raises(hip.RwkvHipError, match="no output"):
        session.score(ones, ones, state)
    with pytest.raises(ValueError):
        session.score(ones, np.ones((1, 3), np.int64), state, out)
    session.set_profile(1)
    with pytest.raises(hip.RwkvHipError, match="profiling"):
        session.score(ones, ones, state, out)
    session.set_profile(0)
    session.score(ones, None, state, entropy=out)   # entropy alone needs no targets
    assert np.all(out.numpy()[:2] > 0)
    session.close()


def test_host_api_scores(gpu):
    _run("score_gpu_test")
