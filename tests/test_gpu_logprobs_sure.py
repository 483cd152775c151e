"""linear_logprobs of rows that are nearly sure of one entry."""
import numpy as np
import pytest

from test_gpu_logprobs import STEP, run_head

pytestmark = pytest.mark.gpu


def sure_head(hip, types, M, N, K, best, second):
    """Logits of whole halves, exact in every type: 50 at `best`, 32 at `second`, -20 elsewhere."""
    codes = np.full(N, -40)
    codes[second], codes[best] = 64, 100
    unit = 2.0 ** -9 * (256 / K)                       # a code times K ones times this: half the code
    fmt = hip.FMT_F16 if types == "f16" else hip.FMT_W8
    rows = np.repeat(codes[:, None], K, axis=1)
    data = (rows * unit).astype(np.float16) if types == "f16" else rows.astype(np.int8)
    packed = hip.DeviceArray((data.nbytes,), np.uint8)
    src = hip.DeviceArray.from_numpy(data)
    hip.pack_weights(fmt, N, K, src, packed)
    hip.device_sync()
    z = np.broadcast_to(codes / 2.0, (M, N))
    return dict(fmt=fmt, x=hip.DeviceArray.from_numpy(np.ones((M, K), np.int8 if types == "i8" else np.float16)), packed=packed,
                scale=None if types == "f16" else hip.DeviceArray.from_numpy(np.full(N, unit, np.float16)),
                x_scale=hip.DeviceArray.from_numpy(np.ones(M, np.float32)) if types == "i8" else None, z=z, off=0.0)


@pytest.mark.parametrize("types", ["f16", "w8", "i8"])
@pytest.mark.parametrize("M,top", [(8, 0), (64, 0), (300, 0), (300, 1), (300, 3)])
@pytest.mark.parametrize("best,second", [(520, 521), (521, 520), (576, 576 + 27), (640, 644), (1000, 3)])
def test_what_is_left_beside_a_sure_entry_is_kept(gpu, types, M, top, best, second):
    """However few rows, wherever the runner-up lies (one lane's 32 columns, the strip's other half, another tile): log probability and entropy
    are right relative to themselves, the largest entry's 1 being kept apart from the other terms."""
    N, K = 2048, 512
    c = sure_head(gpu, types, M, N, K, best, second)
    got = run_head(gpu, c, np.full(M, best), top)
    d = c["z"][0] - 50.0
    rest = np.exp(np.delete(d, best)).sum()
    # the exponent's d = -18 comes out exact, times log2 e in three roundings; exp2 to a step; sums in chains of N / 256 + 64
    tol = (3 * 19 + 4 + N / 256 + 64) * STEP
    assert np.all(np.abs(got["logprob"] + np.log1p(rest)) <= tol * rest)
    entropy = np.log1p(rest) - (d * np.exp(d)).sum() / (1 + rest)
    assert np.all(np.abs(got["entropy"] - entropy) <= 2 * tol * entropy)
    if top:
        assert np.all(got["ids"][:, 0] == best) and np.all(np.abs(got["tops"][:, 0] + np.log1p(rest)) <= tol * rest)


@pytest.mark.parametrize("types", ["f16", "w8", "i8"])
@pytest.mark.parametrize("M", [8, 64, 300])
def test_equal_best_entries_each_count(gpu, types, M):
    """Two best entries in one lane's columns: ln 2 and what is left beside them."""
    N, K = 2048, 512
    c = sure_head(gpu, types, M, N, K, [520, 521], 522)
    got = run_head(gpu, c, np.full(M, 521), 0)
    d = c["z"][0] - 50.0
    total = np.exp(d).sum()
    # 2 + 1.5e-8 rounds to 2 (half a step of 1 in the logarithm), which is good to a step, and one difference
    assert np.all(np.abs(got["logprob"] + np.log(total)) <= 4 * STEP)
    assert np.all(np.abs(got["entropy"] - (np.log(total) - (d * np.exp(d)).sum() / total)) <= 4 * STEP)


@pytest.mark.parametrize("M,top", [(8, 2), (64, 0), (300, 1), (300, 3)])
def test_logits_of_minus_infinity(gpu, M, top):
    """Columns whose logits are -infinity (one in each lane's columns, a whole strip, a whole tile) count for nothing."""
    N, K, best, second = 2048, 512, 520, 524
    c = sure_head(gpu, "f16", M, N, K, best, second)
    gone = np.unique(np.r_[np.arange(4, N, 8), np.arange(64, 128), np.arange(1024, 1280)])
    gone = gone[(gone != best) & (gone != second)]
    codes = np.full(N, -40)
    codes[second], codes[best] = 99, 100               # half a nat below
    w = np.repeat((codes * 2.0 ** -10).astype(np.float16)[:, None], K, axis=1)
    w[gone] = -np.inf
    src = gpu.DeviceArray.from_numpy(w)
    gpu.pack_weights(gpu.FMT_F16, N, K, src, c["packed"])
    got = run_head(gpu, c, np.full(M, best), top)
    d = codes / 2.0 - 50.0
    d = np.delete(d, gone)
    total = np.exp(d).sum()
    # ln 1.6 and 0.66, each of a sum that is good to a few half steps of 1
    assert np.all(np.abs(got["logprob"] + np.log(total)) <= 8 * STEP)
    assert np.all(np.abs(got["entropy"] - (np.log(total) - (d * np.exp(d)).sum() / total)) <= 8 * STEP)
    if top:
        want = np.array([best, second, 0])[:top]       # then the first of the equal ones
        assert np.all(got["ids"] == want)
