"""Session.score with a head whose logits go through memory in blocks of rows, at vocabularies where a row is read in several parts."""
import numpy as np
import pytest

from test_gpu_logprobs import STEP, check_logprobs, ref_logprobs, ref_norm
from test_gpu_score import HALF, head_of, run_score

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,top", [(3, 100, 5), (1, 257, 64), (2, 150, 0), (1, 40, 20)])
def test_int4_head_of_a_long_vocabulary(gpu, B, T, top):
    """Blocks of 256 rows and a shorter one behind them, whose rows go in more parts than the full block's."""
    from rwkv_lightning_cuda_amd.model import HipModel, ModelDims, Session, State, synth_weights
    hip = gpu
    dims = ModelDims(L=1, C=256, H=4, F=512, V=65536, Rw=32, Ra=32, Rg=64, Rv=16)
    weights = synth_weights(dims, 5)
    model = HipModel.from_host_weights(dims, weights, hip.FMT_W4)
    rng = np.random.default_rng(B * 1000 + T)
    tokens, targets = rng.integers(0, dims.V, (B, T)), rng.integers(0, dims.V, (B, T))
    session, state = Session(model), State(dims, B)
    got = run_score(hip, session, state, tokens, targets, top)
    rows = np.unique(np.clip(np.r_[0, 1, 43, 255, 256, 257, B * T - 2, B * T - 1], 0, B * T - 1))
    x1, cm = session.debug_buffer("x1", (B * T, dims.C))[rows], session.debug_buffer("cm", (B * T, dims.C))[rows]
    y = ref_norm(x1, cm, weights["ln_out_w"], weights["ln_out_b"], False)[1]
    w = head_of(hip, model, dims)
    z = y @ w.T
    # half a step of fp16 per value, sums eight at a time, and the logits' own rounding to fp16
    slack = ((HALF * 1.01 + (dims.C / 8 + 8) * STEP) * (np.abs(y) @ np.abs(w).T) + HALF * np.abs(z) * 1.01).max()
    got = {n: v[rows] for n, v in got.items()}
    ref = ref_logprobs(z, targets.ravel()[rows], top)
    if top:
        ids = got.pop("ids")
        for r in range(len(rows)):
            assert len(set(ids[r])) == top
            assert np.all(np.abs(z[r][ids[r]] - np.sort(z[r])[::-1][:top]) <= 2 * slack)
    check_logprobs(got, ref, dims.V, slack=slack)
    session.close()
    model.close()
