"""Sequences that branch, from Python: a prompt's state forked, tokens drawn for all of them, the ended ones' rows given away - and the same
through the C++ host API."""
import numpy as np
import pytest

from test_host_api import _run

pytestmark = pytest.mark.gpu


def test_host_api_branches(gpu):
    out = _run("branch_gpu_test")
    assert "ok   branches_go_on_from_their_own_states" in out


@pytest.mark.parametrize("wkv_fp16", [False, True])
def test_a_batch_that_branches(gpu, wkv_fp16):
    """Prefill, fork, draw, decode, compact - against the same sequences run without any of it."""
    from rwkv_lightning_cuda_amd.model import HipModel, ModelDims, Session, State
    hip = gpu
    dims = ModelDims(L=3, C=256, H=4, F=1024, V=2048, Rw=32, Ra=32, Rg=64, Rv=16)
    model = HipModel.random_on_device(dims, hip.FMT_W8, seed=4)
    session = Session(model)
    V, n = dims.V, 6
    dev = hip.DeviceArray
    prompt = np.arange(7)[None] * 13 % V
    one, logits1 = State(dims, 1, wkv_fp16), dev((1, V), np.float32)
    session.forward(prompt, one, logits1)
    pool, logits = State(dims, n, wkv_fp16), dev((n, V), np.float32)
    hip.device_sync()
    pool.copy_rows(range(n), [0] * n, source=one, stream=session.stream)
    hip.device_sync()
    rng = np.random.default_rng(3)
    token, ws = dev((n,), np.int32), dev((hip.draw_tokens_workspace(n, V),), np.uint8)
    source = dev.zeros((n,), np.int32)
    top_k, temperature = dev.from_numpy(np.array([0, 1, 3, 0, 50, 0], np.int32)), dev.from_numpy(np.array([1, 1, 1, 0, 2, 5], np.float32))
    hip.draw_tokens(n, V, logits1, dev.from_numpy(rng.random(n).astype(np.float32)), token, ws, top_k=top_k, temperature=temperature, source=source,
                    logit_rows=1)
    hip.device_sync()
    first = token.numpy()
    assert first[1] == logits1.numpy()[0].argmax()
    said = [[int(t)] for t in first]
    where = list(range(n))          # row of the pool -> sequence
    for step in range(5):
        session.forward(np.array([[said[i][-1]] for i in where]), pool, logits)
        hip.draw_tokens(n, V, logits, dev.from_numpy(rng.random(n).astype(np.float32)), token, ws, top_k=top_k, temperature=temperature)
        hip.device_sync()
        got = token.numpy()
        for row, i in enumerate(where):
            said[i].append(int(got[row]))
        # sequences change rows; in the last step but one, one ends and another goes on twice
        order = rng.permutation(n)
        pool.copy_rows(range(n), order, stream=session.stream)
        where = [where[r] for r in order]
        if step == 3:
            pool.copy_rows([2], [5], stream=session.stream)
            said[where[2]] = list(said[where[5]])
    session.forward(np.array([[said[i][-1]] for i in where]), pool, logits)
    got = logits.numpy()
    # each sequence alone in a batch of as many copies: the same kernels, row by row the same bits
    for row, i in enumerate(where):
        state, z = State(dims, n, wkv_fp16), dev((n, V), np.float32)
        session.forward(prompt, one_again := State(dims, 1, wkv_fp16), logits1)
        hip.device_sync()
        state.copy_rows(range(n), [0] * n, source=one_again, stream=session.stream)
        for t in said[i]:
            session.forward(np.full((n, 1), t), state, z)
        assert np.array_equal(z.numpy()[row], got[row]), (row, i)
    with pytest.raises(ValueError):
        pool.copy_rows([0], [0], source=State(dims, 1, not wkv_fp16))
    session.close()
    model.close()
