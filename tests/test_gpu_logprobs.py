"""add_norm_q8, token_logprobs and linear_logprobs against plain formulas in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24  # half a step of fp32


# ---- formulas -------------------------------------------------------------------------------------------------------
def ref_norm(x, res, w, b, rms, eps=1e-5):
    s = x.astype(np.float64) + (0.0 if res is None else res.astype(np.float64))
    c = s if rms else s - s.mean(axis=1, keepdims=True)
    return s, c / np.sqrt((c * c).mean(axis=1, keepdims=True) + eps) * w.astype(np.float64) + (0.0 if b is None else b.astype(np.float64))


def ref_logprobs(z, tokens, top):
    """logprob, entropy, rank, ids, top logprobs, and the averages of |d| and d^2 (d = z - max) that the tolerances need."""
    z = z.astype(np.float64)
    rows, V = z.shape
    out = dict(logprob=np.zeros(rows), entropy=np.zeros(rows), rank=np.full(rows, -1, np.int32), ids=np.full((rows, top), -1, np.int32),
               tops=np.full((rows, top), -np.inf), d1=np.zeros(rows), d2=np.zeros(rows))
    for r in range(rows):
        row, t = z[r], int(tokens[r])
        bad = bool(np.isnan(row).any() or np.isposinf(row).any())
        nothing = bool(np.all(np.isneginf(row)))
        if bad:
            logp = np.full(V, np.nan)
            out["entropy"][r] = np.nan
        elif nothing:
            logp = np.full(V, -np.inf)
        else:
            d = row - row.max()
            p = np.exp(d)
            lse = np.log(p.sum())
            logp = d - lse
            p /= p.sum()
            live = p > 0
            out["entropy"][r] = -(p[live] * logp[live]).sum()
            out["d1"][r], out["d2"][r] = (p[live] * -d[live]).sum(), (p[live] * d[live] ** 2).sum()
        out["logprob"][r] = 0.0 if t < 0 else np.nan if t >= V else logp[t]
        if 0 <= t < V and not np.isnan(row[t]):
            out["rank"][r] = int((row > row[t]).sum() + (row[:t] == row[t]).sum())
        order = np.lexsort((np.arange(V), -np.where(np.isnan(row), -np.inf, row)))
        order = order[np.where(np.isnan(row[order]), -np.inf, row[order]) > -np.inf][:top]
        out["ids"][r, :len(order)] = order
        out["tops"][r, :len(order)] = logp[order]
    return out


def check_logprobs(got, ref, V, slack=0.0):
    """got: arrays by the same names.  z - max and its product with log2 e are rounded (|d| half steps each), exp2 is good to a step, a sum
    of V positive terms in chains of at most V / 256 + 64 is good to as many half steps; `slack`: how far the logits themselves may be off."""
    chain = (V / 256 + 64) * STEP
    lse = (3 * ref["d1"] + 4) * STEP + chain + 2 * slack
    for name, value in (("logprob", "logprob"), ("tops", "tops")):
        if name not in got:
            continue
        want = ref[value]
        tol = (lse if want.ndim == 1 else lse[:, None]) + 4 * STEP * np.abs(np.where(np.isfinite(want), want, 0.0))
        same = (got[name] == want) | (np.isnan(got[name]) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            near = np.abs(got[name] - want) <= tol
        assert np.all(same | near), (name, np.nanmax(np.where(same, 0, np.abs(got[name] - want))), tol.max())
    if "entropy" in got:
        want = ref["entropy"]
        tol = (3 * ref["d2"] + 8 * ref["d1"] + 8 * (1 + np.abs(np.nan_to_num(want)))) * STEP + 2 * chain * (1 + ref["d1"]) + 2 * slack * (1 + ref["d1"])
        ok = (np.abs(got["entropy"] - want) <= tol) | (np.isnan(got["entropy"]) & np.isnan(want))
        assert np.all(ok), (np.abs(got["entropy"] - want).max(), tol.max())
    for name in ("rank", "ids"):
        if name in got:
            assert np.array_equal(got[name], ref[name]), name


# ---- norm -----------------------------------------------------------------------------------------------------------
def run_norm(hip, x, res, w, b, rms, in_place=False):
    rows, C = x.shape
    dev = hip.DeviceArray.from_numpy
    dx, dw = dev(x), dev(w)
    dr = None if res is None else dev(res)
    db = None if b is None else dev(b)
    q, scale = hip.DeviceArray((rows, C), np.int8), hip.DeviceArray((rows,), np.float32)
    xo = dx if in_place else hip.DeviceArray((rows, C), np.float16)
    hip.add_norm_q8(rows, C, dx, dr, dw, db, q, scale, x_out=xo, norm=hip.NORM_RMS if rms else hip.NORM_LAYER)
    hip.device_sync()
    return xo.numpy(), q.numpy(), scale.numpy()


@pytest.mark.parametrize("rows,C", [(1, 8), (3, 64), (2, 520), (5, 768), (7, 2048), (4, 2056), (4, 4096), (3, 8192), (1, 8184), (300, 768),
                                    (1031, 512), (2048, 64)])
@pytest.mark.parametrize("rms,with_res,with_b", [(False, True, True), (True, True, False), (False, False, False), (True, False, True)])
def test_norm_matches_the_formula(gpu, rows, C, rms, with_res, with_b):
    rng = np.random.default_rng(rows * 131 + C)
    x = (rng.standard_normal((rows, C)) * 2 + 0.3).astype(np.float16)
    res = rng.standard_normal((rows, C)).astype(np.float16) if with_res else None
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float16)
    b = (0.2 * rng.standard_normal(C)).astype(np.float16) if with_b else None
    xo, q, scale = run_norm(gpu, x, res, w, b, rms)
    s, y = ref_norm(x, res, w, b, rms)
    want_out = (x.astype(np.float32) + (0 if res is None else res.astype(np.float32))).astype(np.float16)
    assert np.array_equal(xo.view(np.uint16), want_out.view(np.uint16))
    amax = np.abs(y).max(axis=1)
    # sums of C terms in chains of 8 and a tree (30 half steps), subtraction, reciprocal root, product, fma, quotient; the spread of
    # the values is of the size of the values, so that nothing cancels by more than a factor of eight
    tol = 8 * 48 * STEP
    assert np.all(np.abs(scale - amax / 127) <= tol * amax / 127 + 1e-30)
    codes = y / scale.astype(np.float64)[:, None]
    assert np.abs(codes - q).max() <= 0.5 + 2 * 127 * tol
    assert np.array_equal(np.abs(q.astype(np.int32)).max(axis=1), np.full(rows, 127))


def test_norm_of_special_rows(gpu):
    C = 768
    rng = np.random.default_rng(5)
    x = rng.standard_normal((7, C)).astype(np.float16)
    x[1] = 0.0
    x[2, 5] = np.nan
    x[3, 700] = np.inf
    x[4] = 3.0                 # no variance
    x[5] = 65504.0             # the sum leaves fp16
    x[5, ::2] = -65504.0
    res = np.zeros_like(x)
    res[5] = x[5]
    w = np.ones(C, np.float16)
    for rms in (False, True):
        xo, q, scale = run_norm(gpu, x, res, w, None, rms, in_place=True)
        assert np.isnan(scale[2]) and np.isnan(scale[3]) and not q[2].any() and not q[3].any()
        assert scale[1] == 0 and not q[1].any()
        assert np.isinf(xo[5]).all() and abs(scale[5] * 127 - 1) <= 1e-5 and np.array_equal(np.abs(q[5]), np.full(C, 127))
        assert np.isfinite(scale[[0, 4, 6]]).all() and np.abs(q[[0, 6]]).max() == 127
        if not rms:
            assert scale[4] == 0 and not q[4].any()
        y = ref_norm(x[:1], None, w, None, rms)[1]
        assert np.abs(y / scale[0] - q[0]).max() <= 0.51


# ---- log probabilities of logits ------------------------------------------------------------------------------------
def run_logprobs(hip, z, tokens, top, io=None, ld=None, lead=0, stream=None, workspace=None):
    rows, V = z.shape
    dtype = np.float16 if z.dtype == np.float16 else np.float32
    ld = V if ld is None else ld
    flat = np.full(lead + rows * ld, 1e4, dtype)      # whatever lies between the rows would show
    for r in range(rows):
        flat[lead + r * ld:lead + r * ld + V] = z[r]
    d = hip.DeviceArray.from_numpy(flat)
    dt = hip.DeviceArray.from_numpy(np.asarray(tokens, np.int32))
    out = {n: hip.DeviceArray.zeros((rows,), t) for n, t in (("logprob", np.float32), ("entropy", np.float32), ("rank", np.int32))}
    ids, tops = hip.DeviceArray.zeros((rows, top), np.int32), hip.DeviceArray.zeros((rows, top), np.float32)
    need = hip.token_logprobs_workspace(rows, V, top)
    ws = workspace if workspace is not None else hip.DeviceArray((max(need, 16),), np.uint8)
    hip.token_logprobs(rows, V, d.view(lead, (rows * ld,)), dt, ws, out["logprob"], out["entropy"], out["rank"], top, ids if top else None,
                       tops if top else None, io=hip.IO_F16 if dtype == np.float16 else hip.IO_F32, ld=ld, stream=stream)
    hip.device_sync()
    got = {n: v.numpy() for n, v in out.items()}
    if top:
        got.update(ids=ids.numpy(), tops=tops.numpy())
    return got


def logits_of(kind, rng, rows, V, dtype):
    z = rng.standard_normal((rows, V)) * 2.5 - 3
    if kind == "ties":
        z = np.round(z)
    elif kind == "equal":
        z[:] = 1.25
    elif kind == "rising":
        z = np.sort(z, axis=1)
    elif kind == "falling":
        z = -np.sort(z, axis=1)
    elif kind == "sure":
        z[np.arange(rows), rng.integers(0, V, rows)] = 60.0
    elif kind == "masked":
        z[rng.random((rows, V)) < 0.98] = -np.inf
        z[0] = -np.inf                                # nothing left
        z[-1, 1:] = -np.inf                           # one left, or that and nothing
    elif kind == "lowest":
        z[rng.random((rows, V)) < 0.9] = np.finfo(dtype).min
        z[0] = np.finfo(dtype).min
    elif kind == "far":
        z *= 3000.0 if dtype == np.float16 else 1e37
    return z.astype(dtype)


@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 3), (5, 31), (4, 64), (3, 255), (2, 1000), (3, 4097), (2, 8192), (2, 50277), (1, 65536),
                                    (9, 65536), (1, 131073), (300, 100), (700, 517)])
@pytest.mark.parametrize("dtype,top", [(np.float32, 5), (np.float16, 20), (np.float32, 64), (np.float32, 0)])
def test_logprobs_match_the_formula(gpu, rows, V, dtype, top):
    rng = np.random.default_rng(V * 7 + rows)
    z = logits_of("plain", rng, rows, V, dtype)
    tokens = rng.integers(0, V, rows)
    check_logprobs(run_logprobs(gpu, z, tokens, top), ref_logprobs(z, tokens, top), V)


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "rising", "falling", "masked"])
@pytest.mark.parametrize("dtype,top", [(np.float32, 20), (np.float16, 3), (np.float32, 64)])
def test_logprobs_of_many_long_rows(gpu, kind, dtype, top):
    """Rows that a block reads alone, over many batches; a few of them are checked."""
    rows, V = 1100, 20003
    rng = np.random.default_rng(29)
    z = np.tile(logits_of(kind, rng, 11, V, dtype), (100, 1))
    tokens = rng.integers(0, V, rows)
    got = run_logprobs(gpu, z, tokens, top)
    some = np.r_[0:11, 545:550, 1098:1100]
    check_logprobs({n: v[some] for n, v in got.items()}, ref_logprobs(z[some], tokens[some], top), V)


@pytest.mark.parametrize("kind", ["ties", "equal", "rising", "falling", "sure", "masked", "lowest", "far"])
@pytest.mark.parametrize("rows,V,dtype,top", [(2, 70, np.float32, 64), (3, 1000, np.float16, 20), (2, 5001, np.float32, 20), (3, 65536, np.float32, 5),
                                              (2, 65536, np.float16, 64), (260, 4096, np.float32, 3)])
def test_logprobs_of_awkward_rows(gpu, kind, rows, V, dtype, top):
    rng = np.random.default_rng(11)
    z = logits_of(kind, rng, rows, V, dtype)
    tokens = rng.integers(0, V, rows)
    tokens[0] = V - 1
    check_logprobs(run_logprobs(gpu, z, tokens, top), ref_logprobs(z, tokens, top), V)


@pytest.mark.parametrize("V,rows", [(517, 6), (9001, 6), (65536, 6), (517, 600)])
def test_logprobs_of_rows_that_are_not_finite_and_of_tokens_that_are_none(gpu, V, rows):
    rng = np.random.default_rng(3)
    z = logits_of("plain", rng, rows, V, np.float32)
    z[1, V // 2] = np.nan
    z[2, 3] = np.inf
    z[3, 5], z[3, V - 1] = np.nan, -np.inf
    z[4] = np.nan
    tokens = rng.integers(0, V, rows)
    tokens[0], tokens[1], tokens[2], tokens[3] = -1, V // 2, 3, 5
    tokens[5] = V
    ref = ref_logprobs(z, tokens, 4)
    check_logprobs(run_logprobs(gpu, z, tokens, 4), ref, V)
    tokens[5] = -7
    check_logprobs(run_logprobs(gpu, z, tokens, 4), ref_logprobs(z, tokens, 4), V)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("lead,extra,V,rows", [(0, 1, 1000, 3), (1, 0, 1000, 3), (3, 5, 4099, 4), (5, 2, 65536, 2), (1, 1, 70, 300)])
def test_logprobs_of_rows_anywhere(gpu, dtype, lead, extra, V, rows):
    rng = np.random.default_rng(17)
    z = logits_of("plain", rng, rows, V, dtype)
    tokens = rng.integers(0, V, rows)
    check_logprobs(run_logprobs(gpu, z, tokens, 7, ld=V + extra, lead=lead), ref_logprobs(z, tokens, 7), V)


@pytest.mark.parametrize("rows,V,dtype", [(3, 100, np.float32), (2, 65536, np.float32), (400, 5000, np.float32), (2, 50277, np.float16)])
def test_rows_that_are_nearly_sure_keep_what_is_left(gpu, rows, V, dtype):
    """Log probability and entropy near 0 are right relative to themselves: what remains beside the largest entry's 1 is not lost in it."""
    rng = np.random.default_rng(37)
    z = rng.standard_normal((rows, V)).astype(dtype)
    at = rng.integers(0, V, rows)
    z[np.arange(rows), at] = 30.0
    got, ref = run_logprobs(gpu, z, at, 0), ref_logprobs(z, at, 0)
    exact = z.astype(np.float64) - 30.0
    exact[np.arange(rows), at] = -np.inf
    rest = np.exp(exact).sum(axis=1)                  # beside the 1: some 1e-13 V
    # 35 in the exponent, rounded three times, and the sum's chain; the entropy's terms carry d as a factor
    tol = (3 * 36 + 4 + V / 256 + 64) * STEP
    assert np.all(np.abs(got["logprob"] + np.log1p(rest)) <= tol * rest)
    exact[np.arange(rows), at] = 0.0
    entropy = np.log1p(rest) - (exact * np.exp(exact)).sum(axis=1) / (1 + rest)
    assert np.all(np.abs(got["entropy"] - entropy) <= 2 * tol * entropy)
    assert np.all(got["rank"] == ref["rank"])


def test_a_row_does_not_depend_on_the_other_rows_and_calls_repeat(gpu):
    rng = np.random.default_rng(23)
    z = logits_of("plain", rng, 12, 65536, np.float32)
    tokens = rng.integers(0, 65536, 12)
    first = run_logprobs(gpu, z, tokens, 20)
    again = run_logprobs(gpu, z, tokens, 20)
    turned = run_logprobs(gpu, z[::-1].copy(), tokens[::-1].copy(), 20)
    for name in first:
        assert np.array_equal(first[name].view(np.uint32), again[name].view(np.uint32))
        assert np.array_equal(first[name].view(np.uint32), turned[name][::-1].copy().view(np.uint32))


def test_a_long_tensor_passes_32_bits(gpu):
    """Rows whose offsets pass 2^31 and 2^32 bytes and 2^31 entries: a row stride of 2^30 entries over a tensor that is not filled."""
    hip = gpu
    V, ld, rows = 1000, 1 << 30, 3
    rng = np.random.default_rng(2)
    z = logits_of("plain", rng, rows, V, np.float16)
    big = hip.DeviceArray((2 * ld + V,), np.float16)
    for r in range(rows):
        big.view(r * ld, (V,)).upload(z[r])
    tokens = rng.integers(0, V, rows)
    out = [hip.DeviceArray((rows,), t) for t in (np.float32, np.float32, np.int32)]
    ids, tops = hip.DeviceArray((rows, 3), np.int32), hip.DeviceArray((rows, 3), np.float32)
    ws = hip.DeviceArray((max(16, hip.token_logprobs_workspace(rows, V, 3)),), np.uint8)
    hip.token_logprobs(rows, V, big, hip.DeviceArray.from_numpy(tokens.astype(np.int32)), ws, *out, 3, ids, tops, io=hip.IO_F16, ld=ld)
    hip.device_sync()
    got = dict(zip(("logprob", "entropy", "rank"), (o.numpy() for o in out)), ids=ids.numpy(), tops=tops.numpy())
    check_logprobs(got, ref_logprobs(z, tokens, 3), V)


# ---- the head -------------------------------------------------------------------------------------------------------
def head_case(hip, orc, types, M, N, K, seed, logits=True):
    """x, weights and logits in 64 bits with the bound of their error."""
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((N, K)) * 0.05).astype(np.float16)
    x = rng.standard_normal((M, K)).astype(np.float32)
    dev = hip.DeviceArray.from_numpy
    fmt = hip.FMT_F16 if types == "f16" else hip.FMT_W8
    scale, x_scale, sc = None, None, None
    if fmt == hip.FMT_W8:
        codes, sc = orc.quantize_w8(w)
        wd, data = codes.astype(np.float64) * sc.astype(np.float64)[:, None], codes
        scale = dev(sc)
    else:
        wd, data = w.astype(np.float64), w
    packed = hip.DeviceArray((data.nbytes,), np.uint8)
    src = dev(data)
    hip.pack_weights(fmt, N, K, src, packed)
    hip.device_sync()
    if types == "i8":
        xs = (np.abs(x).max(axis=1) / 127).astype(np.float32)
        xq = np.clip(np.rint(x / xs[:, None]), -127, 127).astype(np.int8)
        xd, dx, x_scale = xq.astype(np.float64) * xs.astype(np.float64)[:, None], dev(xq), dev(xs)
    else:
        x16 = x.astype(np.float16)
        xd, dx = x16.astype(np.float64), dev(x16)
    z = xd @ wd.T if logits else np.broadcast_to(0.0, (M, N))
    if types == "i8":
        off = 3 * STEP * (np.abs(xd).max(axis=0) @ np.abs(wd).T).max()  # the whole number's conversion and two products
    else:                                             # exact products, summed eight at a time
        off = (K / 8 + 8) * STEP * (np.abs(xd).max(axis=0) @ np.abs(wd).T).max()
    return dict(xd=xd, wd=wd, fmt=fmt, x=dx, packed=packed, scale=scale, x_scale=x_scale, z=z, off=off)


def run_head(hip, c, tokens, top, stream=None, workspace=None):
    M, N = c["z"].shape
    K = c["x"].shape[1]
    out = [hip.DeviceArray.zeros((M,), np.float32) for _ in range(2)]
    ids, tops = hip.DeviceArray.zeros((M, top), np.int32), hip.DeviceArray.zeros((M, top), np.float32)
    need = hip.linear_logprobs_workspace(c["fmt"], M, N, K, top, x_int8=c["x_scale"] is not None)
    ws = workspace if workspace is not None else hip.DeviceArray((need,), np.uint8)
    hip.linear_logprobs(c["fmt"], M, N, K, c["x"], c["packed"], c["scale"], hip.DeviceArray.from_numpy(np.asarray(tokens, np.int32)), ws,
                        x_scale=c["x_scale"], logprob=out[0], entropy=out[1], top_n=top, top_ids=ids if top else None,
                        top_logprobs=tops if top else None, stream=stream)
    hip.device_sync()
    got = dict(logprob=out[0].numpy(), entropy=out[1].numpy())
    if top:
        got.update(ids=ids.numpy(), tops=tops.numpy())
    return got


def check_head(got, c, tokens, top):
    z = c["z"]
    ref = ref_logprobs(z, tokens, top)
    if top:
        # neighbours nearer than the logits' error may change places: what is named must be worth what the place is worth
        ids = got.pop("ids")
        for r in range(len(z)):
            n = min(top, z.shape[1])
            assert len(set(ids[r, :n])) == n and np.all(ids[r, n:] == -1)
            best = np.sort(z[r])[::-1][:n]
            assert np.all(np.abs(z[r][ids[r, :n]] - best) <= 2 * c["off"])
    check_logprobs(got, ref, z.shape[1], slack=c["off"])


@pytest.mark.parametrize("types", ["f16", "w8", "i8"])
@pytest.mark.parametrize("M,N,K,top", [(1, 32, 256, 0), (1, 32, 256, 40), (1, 4096, 768, 5), (2, 1056, 512, 0), (5, 2080, 1280, 3), (16, 4096, 256, 1),
                                       (17, 640, 256, 20), (32, 1024, 1024, 0), (33, 1024, 768, 2), (64, 2048, 2048, 0), (129, 992, 512, 64),
                                       (300, 2592, 256, 0), (257, 8192, 512, 5), (600, 1024, 768, 1)])
def test_head_matches_the_formula(gpu, orc, types, M, N, K, top):
    c = head_case(gpu, orc, types, M, N, K, seed=M + N + K)
    tokens = np.random.default_rng(M).integers(0, N, M)
    tokens[0] = N - 1
    check_head(run_head(gpu, c, tokens, top), c, tokens, top)


@pytest.mark.parametrize("types,M", [("f16", 3), ("i8", 3), ("w8", 200), ("i8", 200), ("f16", 200)])
def test_head_tokens_that_are_none_and_rows_that_are_not_finite(gpu, orc, types, M):
    N, K = 1024, 512
    c = head_case(gpu, orc, types, M, N, K, seed=9)
    tokens = np.full(M, 7)
    tokens[0], tokens[1] = -1, N
    if types == "i8":
        xs = c["x_scale"].numpy()
        xs[2] = np.nan
        xs[M - 1] = 0.0 if M > 3 else np.nan
        c["x_scale"].upload(xs)
        if M > 3:
            c["z"][M - 1] = 0.0
    else:
        x = c["x"].numpy()
        x[2, 100] = np.nan
        c["x"].upload(x)
    c["z"][2] = np.nan
    got = run_head(gpu, c, tokens, 2)
    assert got["logprob"][0] == 0 and np.isnan(got["logprob"][1]) and np.isnan(got["logprob"][2]) and np.isnan(got["entropy"][2])
    assert np.all(got["ids"][2] == -1) and np.all(np.isneginf(got["tops"][2]))
    keep = [r for r in range(M) if r != 2]
    c["z"] = c["z"][keep]
    check_head({k: v[keep] for k, v in got.items()}, c, tokens[keep], 2)


def crafted_head(hip, M, N, K, codes_of_column, top):
    """int8 x and weights whose logits are whole numbers: every code of column c is codes_of_column[c], x is 1."""
    src = hip.DeviceArray.from_numpy(np.repeat(codes_of_column.astype(np.int8)[:, None], K, axis=1))
    packed = hip.DeviceArray((N * K,), np.uint8)
    hip.pack_weights(hip.FMT_W8, N, K, src, packed)
    hip.device_sync()
    z = np.broadcast_to(codes_of_column.astype(np.float64) * K, (M, N))
    return dict(fmt=hip.FMT_W8, x=hip.DeviceArray.from_numpy(np.ones((M, K), np.int8)), packed=packed,
                scale=hip.DeviceArray.from_numpy(np.ones(N, np.float16)), x_scale=hip.DeviceArray.from_numpy(np.ones(M, np.float32)), z=z, off=0.0)


def poisoned_workspace(hip, c, M, N, K, top):
    """What a call has not written itself looks like the best logits."""
    need = hip.linear_logprobs_workspace(c["fmt"], M, N, K, top, x_int8=True)
    ws = hip.DeviceArray((need,), np.uint8)
    piece = np.full(1 << 22, 1e30, np.float32)
    for at in range(0, need, piece.nbytes):
        n = min(piece.nbytes, need - at)
        ws.view(at, (n,)).upload(piece.view(np.uint8)[:n])
    return ws


@pytest.mark.parametrize("top", [1, 5, 30, 64])
@pytest.mark.parametrize("kind", ["one group", "first only", "last only", "equal"])
def test_head_of_many_rows_finds_alternatives_wherever_they_lie(gpu, top, kind):
    """Calls of many tiles write the logits of the strips that reach a bound only.  The best entries in strips that one group of threads looks
    after, all among the columns that give the bound, none among them, or no entry better than another."""
    hip = gpu
    M, N, K = 2048, 65536, 256
    rng = np.random.default_rng(3)
    codes = rng.integers(-3, 4, N)
    if kind == "one group":
        for i, block in enumerate((0, 64, 128, 192)):
            codes[block * 256:block * 256 + 256:64] = 40 + 4 * i + np.arange(4)
    elif kind == "first only":
        codes[(np.arange(N) // 256) % 8 == 0] += 20
    elif kind == "last only":
        codes[(np.arange(N) // 256) % 8 != 0] += 20
    else:
        codes[:] = 2
    c = crafted_head(hip, M, N, K, codes, top)
    got = run_head(hip, c, np.full(M, 777), top, workspace=poisoned_workspace(hip, c, M, N, K, top))
    want = np.lexsort((np.arange(N), -codes))[:top]
    assert np.array_equal(got["ids"], np.tile(want.astype(np.int32), (M, 1)))
    ref = ref_logprobs(c["z"][:1], [777], top)
    for name, value in (("logprob", "logprob"), ("entropy", "entropy"), ("tops", "tops")):
        assert np.all(got[name] == got[name][0])
    check_logprobs({n: got[n][:1] for n in ("logprob", "entropy", "tops")}, ref, N, slack=3 * STEP * np.abs(c["z"][0]).max())


@pytest.mark.parametrize("M,top", [(40, 5), (40, 64), (700, 20)])
@pytest.mark.parametrize("kind", ["rising", "last only", "equal"])
def test_head_of_a_wide_vocabulary_finds_alternatives_wherever_they_lie(gpu, M, top, kind):
    """More strips of columns than the last launch looks at in one turn: each turn's better than the one before, all in the last strips, or
    no entry better than another."""
    hip = gpu
    N, K = 200032, 256
    codes = np.random.default_rng(4).integers(-3, 4, N)
    if kind == "rising":
        codes = codes + np.arange(N) // 2048
    elif kind == "last only":
        codes[-96:] += 50
    else:
        codes[:] = 2
    c = crafted_head(hip, M, N, K, codes, top)
    got = run_head(hip, c, np.full(M, N - 1), top, workspace=poisoned_workspace(hip, c, M, N, K, top))
    want = np.lexsort((np.arange(N), -codes))[:top]
    assert np.array_equal(got["ids"], np.tile(want.astype(np.int32), (M, 1)))
    for name in ("logprob", "entropy", "tops"):
        assert np.all(got[name] == got[name][0])
    ref = ref_logprobs(c["z"][:1], [N - 1], top)
    check_logprobs({n: got[n][:1] for n in ("logprob", "entropy", "tops")}, ref, N, slack=3 * STEP * np.abs(c["z"][0]).max())


@pytest.mark.parametrize("types,M,top", [("i8", 2049, 5), ("f16", 1700, 2), ("w8", 2048, 20)])
def test_head_of_many_rows_matches_the_formula(gpu, orc, types, M, top):
    """Two launches of tiles with a bound between them (and a second block of rows), some rows checked."""
    hip = gpu
    N, K = 65536, 256
    c = head_case(hip, orc, types, M, N, K, seed=12, logits=False)
    tokens = np.random.default_rng(M).integers(0, N, M)
    got = run_head(hip, c, tokens, top)
    rows = np.unique(np.r_[0, 1, 127, 128, 255, 256, 1023, M - 2, M - 1])
    c["z"] = c["xd"][rows] @ c["wd"].T
    check_head({k: v[rows] for k, v in got.items()}, c, tokens[rows], top)


def test_head_equal_logits_go_by_index(gpu, orc):
    """Columns of one value: whole-number products tie exactly, wherever the columns lie."""
    hip = gpu
    M, N, K = 40, 2048, 256
    c = head_case(hip, orc, "i8", M, N, K, seed=1)
    codes = np.ones((N, K), np.int8)
    codes[100::7] = 2
    src = hip.DeviceArray.from_numpy(codes)
    hip.pack_weights(hip.FMT_W8, N, K, src, c["packed"])
    c["scale"].upload(np.ones(N, np.float16))
    x = np.ones((M, K), np.int8)
    c["x"].upload(x)
    got = run_head(hip, c, np.zeros(M), 30)
    assert np.array_equal(got["ids"], np.tile(np.arange(100, N, 7)[:30], (M, 1)).astype(np.int32))


@pytest.mark.parametrize("types,M,N,K,top", [("i8", 3, 4096, 768, 5), ("i8", 300, 4096, 256, 5), ("f16", 300, 4096, 256, 0)])
def test_head_repeats_and_shares_a_workspace(gpu, orc, types, M, N, K, top):
    hip = gpu
    c = head_case(hip, orc, types, M, N, K, seed=4)
    other = head_case(hip, orc, types, 1, 64, 256, seed=5)
    tokens = np.random.default_rng(1).integers(0, N, M)
    ws = hip.DeviceArray((hip.linear_logprobs_workspace(c["fmt"], M, N, K, top, x_int8=types == "i8"),), np.uint8)
    ws.upload(np.full(ws.shape, 0xff, np.uint8))
    first = run_head(hip, c, tokens, top, workspace=ws)
    run_head(hip, other, [1], min(top, 1), workspace=ws)
    again = run_head(hip, c, tokens, top, workspace=ws)
    for name in first:
        assert np.array_equal(first[name].view(np.uint32), again[name].view(np.uint32))


def test_norm_codes_feed_the_head(gpu, orc):
    """The operators as a scoring pass runs them: residual, norm, codes, product, log probabilities."""
    hip = gpu
    M, N, K, top = 70, 4096, 768, 4
    rng = np.random.default_rng(8)
    c = head_case(hip, orc, "i8", M, N, K, seed=6)
    w = (rng.standard_normal((N, K)) * 0.05).astype(np.float16)
    codes, sc = orc.quantize_w8(w)
    src = hip.DeviceArray.from_numpy(codes)
    hip.pack_weights(hip.FMT_W8, N, K, src, c["packed"])
    c["scale"].upload(sc)
    x = rng.standard_normal((M, K)).astype(np.float16)
    res = rng.standard_normal((M, K)).astype(np.float16)
    g, b = np.ones(K, np.float16), np.zeros(K, np.float16)
    dx, dr, dg, db = (hip.DeviceArray.from_numpy(v) for v in (x, res, g, b))
    hip.add_norm_q8(M, K, dx, dr, dg, db, c["x"], c["x_scale"])
    tokens = rng.integers(0, N, M)
    q, xs = c["x"].numpy().astype(np.float64), c["x_scale"].numpy().astype(np.float64)
    c["z"] = (q @ (codes.astype(np.float64) * sc.astype(np.float64)[:, None]).T) * xs[:, None]
    c["off"] = 3 * STEP * np.abs(c["z"]).max()
    check_head(run_head(hip, c, tokens, top), c, tokens, top)
    # and against the fp16 text: half a code step per value, weights' size times the root of the count, five of them
    y = ref_norm(x, res, g, b, False)[1]
    z = y @ (codes.astype(np.float64) * sc.astype(np.float64)[:, None]).T
    spread = np.sqrt(((codes.astype(np.float64) * sc.astype(np.float64)[:, None]) ** 2).sum(axis=1)).max() * xs.max() / np.sqrt(12)
    assert np.abs(c["z"] - z).max() <= 6 * spread


# ---- streams and graphs ---------------------------------------------------------------------------------------------
class Stream:
    def __init__(self, hip):
        import ctypes
        self.hip, self.lib = hip, hip.load()
        p = ctypes.c_void_p(0)
        hip.check(self.lib.rwkv_hip_stream_create(ctypes.byref(p)))
        self.ptr = p.value

    def sync(self):
        import ctypes
        self.hip.check(self.lib.rwkv_hip_stream_sync(ctypes.c_void_p(self.ptr)))

    def close(self):
        import ctypes
        self.hip.check(self.lib.rwkv_hip_stream_destroy(ctypes.c_void_p(self.ptr)))


def scoring_chain(hip, orc, types, M, N, K, top, seed):
    """Buffers of a norm, a head over its codes (or fp16 rows) and the log probabilities of some logits; launch(stream) enqueues all three."""
    rng = np.random.default_rng(seed)
    c = head_case(hip, orc, types, M, N, K, seed=seed)
    new = lambda shape, t: hip.DeviceArray.zeros(shape, t)  # noqa: E731
    x = hip.DeviceArray.from_numpy(rng.standard_normal((M, K)).astype(np.float16))
    res = hip.DeviceArray.from_numpy(rng.standard_normal((M, K)).astype(np.float16))
    w = hip.DeviceArray.from_numpy((1 + 0.1 * rng.standard_normal(K)).astype(np.float16))
    z = hip.DeviceArray.from_numpy(rng.standard_normal((M, N)).astype(np.float32))
    tokens = hip.DeviceArray.from_numpy(rng.integers(0, N, M).astype(np.int32))
    out = dict(x_out=new((M, K), np.float16), q=new((M, K), np.int8), qs=new((M,), np.float32), hl=new((M,), np.float32), he=new((M,), np.float32),
               hi=new((M, top), np.int32), ht=new((M, top), np.float32), ll=new((M,), np.float32), le=new((M,), np.float32),
               lr=new((M,), np.int32), li=new((M, top), np.int32), lt=new((M, top), np.float32))
    int8 = types == "i8"
    ws = hip.DeviceArray((hip.linear_logprobs_workspace(c["fmt"], M, N, K, top, x_int8=int8),), np.uint8)
    ws2 = hip.DeviceArray((max(16, hip.token_logprobs_workspace(M, N, top)),), np.uint8)

    def launch(stream):
        hip.add_norm_q8(M, K, x, res, w, None, out["q"], out["qs"], x_out=out["x_out"], norm=hip.NORM_RMS, stream=stream)
        hip.linear_logprobs(c["fmt"], M, N, K, out["q"] if int8 else out["x_out"], c["packed"], c["scale"], tokens, ws,
                            x_scale=out["qs"] if int8 else None, logprob=out["hl"], entropy=out["he"], top_n=top, top_ids=out["hi"] if top else None,
                            top_logprobs=out["ht"] if top else None, stream=stream)
        hip.token_logprobs(M, N, z, tokens, ws2, out["ll"], out["le"], out["lr"], top, out["li"] if top else None, out["lt"] if top else None,
                           stream=stream)

    return launch, out, (x, res, z, tokens, c)


def bits(out):
    return {n: v.numpy().view(np.uint8).copy() for n, v in out.items()}


@pytest.mark.parametrize("types,M,N,K,top", [("i8", 3, 4096, 768, 5), ("f16", 200, 2048, 512, 3), ("i8", 300, 4096, 256, 0), ("i8", 1600, 65536, 256, 2)])
def test_a_captured_call_replays(gpu, orc, types, M, N, K, top):
    import ctypes
    hip = gpu
    launch, out, (x, res, z, tokens, keep) = scoring_chain(hip, orc, types, M, N, K, top, seed=31)
    s = Stream(hip)
    lib = s.lib                              # (the runtime that the library loads)
    graph, run = ctypes.c_void_p(0), ctypes.c_void_p(0)
    assert lib.hipStreamBeginCapture(ctypes.c_void_p(s.ptr), ctypes.c_int(1)) == 0
    launch(s.ptr)
    assert lib.hipStreamEndCapture(ctypes.c_void_p(s.ptr), ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    rng = np.random.default_rng(1)
    for _ in range(3):
        x.upload(rng.standard_normal((M, K)).astype(np.float16))
        z.upload(rng.standard_normal((M, N)).astype(np.float32))
        tokens.upload(rng.integers(0, N, M).astype(np.int32))
        launch(None)
        hip.device_sync()
        want = bits(out)
        for v in out.values():
            v.fill0()
        hip.device_sync()
        assert lib.hipGraphLaunch(run, ctypes.c_void_p(s.ptr)) == 0
        s.sync()
        got = bits(out)
        for name in want:
            assert np.array_equal(got[name], want[name]), name
    assert lib.hipGraphExecDestroy(run) == 0 and lib.hipGraphDestroy(graph) == 0
    s.close()


def test_calls_on_two_streams_at_once(gpu, orc):
    hip = gpu
    a, out_a, keep_a = scoring_chain(hip, orc, "i8", 40, 8192, 512, 4, seed=51)
    b, out_b, keep_b = scoring_chain(hip, orc, "f16", 9, 16384, 256, 6, seed=52)
    a(None)
    b(None)
    hip.device_sync()
    want_a, want_b = bits(out_a), bits(out_b)
    for v in list(out_a.values()) + list(out_b.values()):
        v.fill0()
    hip.device_sync()
    s, t = Stream(hip), Stream(hip)
    for _ in range(20):
        a(s.ptr)
        b(t.ptr)
    s.sync()
    t.sync()
    for out, want in ((out_a, want_a), (out_b, want_b)):
        got = bits(out)
        for name in want:
            assert np.array_equal(got[name], want[name]), name
    s.close()
    t.close()


def test_calls_of_two_threads(gpu, orc):
    import threading
    hip = gpu
    chains = [scoring_chain(hip, orc, "i8", 5, 4096, 512, 3, seed=61 + i) for i in range(3)]
    want = []
    for launch, out, _keep in chains:
        launch(None)
        hip.device_sync()
        want.append(bits(out))
    streams = [Stream(hip) for _ in chains]
    errors = []

    def work(i):
        try:
            for _ in range(50):
                chains[i][0](streams[i].ptr)
                streams[i].sync()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (launch, out, _keep), w in zip(chains, want):
        got = bits(out)
        for name in w:
            assert np.array_equal(got[name], w[name]), name
    for s in streams:
        s.close()


def test_outputs_that_are_not_asked_for(gpu):
    """Every output alone gives what all together give."""
    hip = gpu
    rng = np.random.default_rng(5)
    for rows, V in ((2, 65536), (500, 700)):
        z = logits_of("plain", rng, rows, V, np.float32)
        tokens = rng.integers(0, V, rows)
        whole = run_logprobs(hip, z, tokens, 6)
        d, dt = hip.DeviceArray.from_numpy(z), hip.DeviceArray.from_numpy(tokens.astype(np.int32))
        ws = hip.DeviceArray((max(16, hip.token_logprobs_workspace(rows, V, 6)),), np.uint8)
        for name, kind in (("logprob", np.float32), ("entropy", np.float32), ("rank", np.int32)):
            one = hip.DeviceArray.zeros((rows,), kind)
            hip.token_logprobs(rows, V, d, None if name == "entropy" else dt, ws, **{name: one})
            hip.device_sync()
            assert np.array_equal(one.numpy().view(np.uint32), whole[name].view(np.uint32)), name
        ids, tops = hip.DeviceArray.zeros((rows, 6), np.int32), hip.DeviceArray.zeros((rows, 6), np.float32)
        hip.token_logprobs(rows, V, d, None, ws, top_n=6, top_ids=ids, top_logprobs=tops)
        hip.device_sync()
        assert np.array_equal(ids.numpy(), whole["ids"]) and np.array_equal(tops.numpy(), whole["tops"])


@pytest.mark.parametrize("types,M,top", [("i8", 3, 1), ("i8", 150, 1), ("f16", 150, 4), ("w8", 40, 1)])
def test_head_outputs_that_are_not_asked_for(gpu, orc, types, M, top):
    hip = gpu
    N, K = 2080, 512
    c = head_case(hip, orc, types, M, N, K, seed=71)
    tokens = np.random.default_rng(2).integers(0, N, M)
    whole = run_head(hip, c, tokens, top)
    int8 = types == "i8"
    dt = hip.DeviceArray.from_numpy(tokens.astype(np.int32))
    ws = hip.DeviceArray((hip.linear_logprobs_workspace(c["fmt"], M, N, K, top, x_int8=int8),), np.uint8)
    call = lambda t, **kw: hip.linear_logprobs(c["fmt"], M, N, K, c["x"], c["packed"], c["scale"], t, ws, x_scale=c["x_scale"], **kw)  # noqa: E731
    one = hip.DeviceArray.zeros((M,), np.float32)
    # (without alternatives a call may share its columns out otherwise: the last bits of the sums)
    for name, t in (("logprob", dt), ("entropy", None)):
        call(t, **{name: one})
        hip.device_sync()
        assert np.abs(one.numpy() - whole[name]).max() <= (N / 256 + 64) * 4 * STEP * 12
    ids, tops = hip.DeviceArray.zeros((M, top), np.int32), hip.DeviceArray.zeros((M, top), np.float32)
    call(None, top_n=top, top_ids=ids, top_logprobs=tops)
    hip.device_sync()
    assert np.array_equal(ids.numpy(), whole["ids"]) and np.array_equal(tops.numpy().view(np.uint32), whole["tops"].view(np.uint32))


def test_norm_writes_the_sum_over_the_residual(gpu):
    hip = gpu
    rng = np.random.default_rng(3)
    x, res = (rng.standard_normal((5, 768)).astype(np.float16) for _ in range(2))
    w = np.ones(768, np.float16)
    dx, dr, dw = (hip.DeviceArray.from_numpy(v) for v in (x, res, w))
    q, scale = hip.DeviceArray((5, 768), np.int8), hip.DeviceArray((5,), np.float32)
    hip.add_norm_q8(5, 768, dx, dr, dw, None, q, scale, x_out=dr)
    hip.device_sync()
    want = run_norm(hip, x, res, w, None, False)
    assert np.array_equal(dr.numpy(), want[0]) and np.array_equal(q.numpy(), want[1]) and np.array_equal(scale.numpy(), want[2])
    assert np.array_equal(dx.numpy(), x)
