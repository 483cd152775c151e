"""linear_logprobs of more rows than one set of sums has room for, at a wide vocabulary."""
import numpy as np
import pytest

from test_gpu_logprobs import STEP, check_logprobs, crafted_head, poisoned_workspace, ref_logprobs, run_head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,top", [(513, 0), (1100, 1)])
def test_rows_in_several_blocks_without_lists(gpu, M, top):
    hip = gpu
    N, K = 1048576, 256
    rng = np.random.default_rng(M)
    codes = rng.integers(-3, 4, N)
    codes[rng.integers(0, N, 40)] = 5
    c = crafted_head(hip, M, N, K, codes, top)
    tokens = rng.integers(0, N, M)
    tokens[::7] = np.flatnonzero(codes == 5)[0]
    got = run_head(hip, c, tokens, top, workspace=poisoned_workspace(hip, c, M, N, K, top))
    z = codes.astype(np.float64) * K
    ref = ref_logprobs(z[None], tokens[:1], top)
    total = z[tokens[0]] - ref["logprob"][0]
    for r in range(M):       # every row is the same but for its token
        ref["logprob"][0] = z[tokens[r]] - total
        check_logprobs({n: v[r:r + 1] for n, v in got.items()}, ref, N, slack=3 * STEP * np.abs(z).max())
