"""draw_tokens against its definition in 64 bits."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24  # half a step of fp32
# A log probability is -ln(1 + x) of a ratio x of sums that are good to a few 1e-13 (powers of up to 1000 octaves): as |ln(1 + x)| is at
# least x / (1 + x), the error stays below that share of the value, and then it is rounded once.
RTOL = STEP + 1e-11


class Stream:
    def __init__(self, hip):
        self.hip, self.lib = hip, hip.load()
        p = ctypes.c_void_p(0)
        hip.check(self.lib.rwkv_hip_stream_create(ctypes.byref(p)))
        self.ptr = p.value

    def sync(self):
        self.hip.check(self.lib.rwkv_hip_stream_sync(ctypes.c_void_p(self.ptr)))

    def close(self):
        self.hip.check(self.lib.rwkv_hip_stream_destroy(ctypes.c_void_p(self.ptr)))


# ---- the definition -------------------------------------------------------------------------------------------------
def ref_row(z, t, k, p, mp, u):
    """(token, log probability) of one row of fp32 numbers"""
    if not (t >= 0) or np.isnan(p) or np.isnan(mp) or not (0 <= u <= 1) or np.isnan(z).any() or np.isposinf(z).any() or np.isneginf(z).all():
        return -1, 0.0
    V = len(z)
    z = z.astype(np.float64)
    order = np.lexsort((np.arange(V), -z))
    if t == 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        y = (z - z.max()) / float(t) / np.log(2.0)
    y[np.isneginf(z)] = -np.inf
    e = np.where(y < -1000.0, 0.0, np.exp2(np.maximum(y, -1010.0)))
    n = V
    if 0 < k < V:
        n = min(n, k)
    if p < 1:
        n = min(n, int((np.cumsum(e[order]) < float(p) * e.sum()).sum()) + 1)
    if mp > 0:
        n = min(n, int((e >= min(float(mp), 1.0)).sum()))
    kept = np.zeros(V)
    kept[order[:max(n, 1)]] = e[order[:max(n, 1)]]
    upto = np.cumsum(kept)
    hit = np.nonzero((upto > float(u) * upto[-1]) & (kept > 0))[0]
    token = int(hit[0]) if len(hit) else int(np.nonzero(kept > 0)[0][-1])
    others = kept.sum() - kept[token] if kept[token] < 0.5 * kept.sum() else np.delete(kept, token).sum()
    return token, -np.log1p(others / e[token])


def ref(z, t, k, p, mp, u):
    t, p, mp, u = (np.asarray(v, np.float32) for v in (t, p, mp, u))  # (as the call gets them)
    rows = [ref_row(*args) for args in zip(z, t, k, p, mp, u)]
    return np.array([r[0] for r in rows], np.int32), np.array([r[1] for r in rows])


def check(got, want):
    assert np.array_equal(got[0], want[0]), [(i, g, w) for i, (g, w) in enumerate(zip(got[0], want[0])) if g != w][:5]
    # (below fp32's smallest normal number a rounding is off by half a step of 2^-149)
    assert np.all(np.abs(got[1] - want[1]) <= RTOL * np.abs(want[1]) + 2.0 ** -150), (got[1], want[1])


def run(hip, z, t=None, k=None, p=None, mp=None, u=None, source=None, rows=None, ld=None, offset=0, penalties=None, out=False, stream=None, **more):
    """z [logit_rows,V] -> tokens, log probabilities (and the penalties after).  ld: entries between rows; offset: entries in front"""
    of, V = z.shape
    rows = of if rows is None else rows
    ld = V if ld is None else ld
    flat = np.full(offset + of * ld + 16, np.nan, z.dtype)
    for i in range(of):
        flat[offset + i * ld:offset + i * ld + V] = z[i]
    dev = lambda v, kind: None if v is None else hip.DeviceArray.from_numpy(np.asarray(v, kind))  # noqa: E731
    d = dev(flat, z.dtype)
    args = dict(temperature=dev(t, np.float32), top_k=dev(k, np.int32), top_p=dev(p, np.float32), min_p=dev(mp, np.float32), source=dev(source, np.int32),
                penalties=dev(penalties, np.float32), **{n: dev(v, np.float32) for n, v in more.items()})
    if out:
        args["penalties_out"] = hip.DeviceArray((rows, V), np.float32) if out == "apart" else args["penalties"]
    du = dev(np.full(rows, 0.5) if u is None else u, np.float32)
    token, logprob = hip.DeviceArray.from_numpy(np.full(rows + 1, -9, np.int32)), hip.DeviceArray.from_numpy(np.full(rows + 1, 7.0, np.float32))
    ws = hip.DeviceArray((hip.draw_tokens_workspace(rows, V),), np.uint8)
    hip.check(hip.load().rwkv_hip_memset(hip._p(ws), 0xff, ctypes.c_size_t(ws.nbytes)))  # (need not be cleared)
    hip.draw_tokens(rows, V, d.ptr + offset * z.itemsize, du, token, ws, logprob=logprob, logit_rows=of, io=hip.IO_F16 if z.dtype == np.float16 else hip.IO_F32,
                    ld=ld, stream=stream, **args)
    hip.device_sync()
    tokens, logprobs = token.numpy(), logprob.numpy()
    assert tokens[-1] == -9 and logprobs[-1] == 7.0
    got = (tokens[:-1], logprobs[:-1].astype(np.float64))
    return got + (args["penalties_out"].numpy(),) if out else got


STYLES = dict(free=(1.0, 0, 1.0, 0.0), engine=(1.0, 20, 0.3, 0.0), chat=(0.8, 50, 0.9, 0.0), nucleus=(1.0, 0, 0.95, 0.0), min_p=(1.2, 0, 1.0, 0.05),
              greedy=(0.0, 0, 1.0, 0.0), wide=(1.5, 1000, 0.99, 0.001), two=(0.7, 2, 1.0, 0.0), flat=(5.0, 0, 0.9, 0.0), many=(2.0, 5000, 1.0, 0.0),
              sharp=(0.05, 0, 0.5, 0.3), rest=(1.0, 0, 0.999999, 1e-6))


def styles(rows):
    names = list(STYLES)
    table = [STYLES[names[i % len(names)]] for i in range(rows)]
    return [np.array(c) for c in zip(*table)]


def logits_of(rng, rows, V, kind, dtype=np.float32):
    if kind == "peaked":
        z = rng.standard_normal((rows, V)) * 2.5 - 3.0
        for r in range(rows):
            at = rng.integers(0, V, 8)
            z[r, at] += rng.random(8) * 10.0 + rng.random() * 12.0
        z[:, rng.integers(0, V, V // 50)] = -np.inf
        z[:, V - 1] = 0.5
    elif kind == "flat":
        z = rng.standard_normal((rows, V)) * 0.3
    elif kind == "few values":
        z = np.round(rng.standard_normal((rows, V)) * 2.0) * 0.5
    elif kind == "equal":
        z = np.full((rows, V), 1.25)
    elif kind == "powers":  # every scale of fp32: a histogram of equal widths splits these slowly
        z = -np.exp2(rng.random((rows, V)) * 60.0 - 50.0)
    elif kind == "rising":
        z = np.tile(np.arange(V) * (20.0 / V), (rows, 1))
    return z.astype(dtype)


@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 1000, 1023, 4097, 9001, 65536])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_rows_of_any_length(gpu, V, dtype):
    rng = np.random.default_rng(V)
    rows = 24 if V < 60000 else 13
    z = logits_of(rng, rows, V, "peaked", dtype)
    args = styles(rows)
    u = rng.random(rows).astype(np.float32)
    check(run(gpu, z, *args, u), ref(z.astype(np.float32), *args, u))


@pytest.mark.parametrize("kind", ["flat", "few values", "equal", "powers", "rising"])
@pytest.mark.parametrize("V,dtype", [(700, np.float32), (20000, np.float32), (50277, np.float16), (131071, np.float32)])
def test_rows_of_any_shape(gpu, kind, V, dtype):
    """Rows with many candidates, ties at the end of the kept entries and values that lie unevenly: what the list does not hold"""
    rng = np.random.default_rng(3)
    z = logits_of(rng, 12, V, kind, dtype)
    args = styles(12)
    u = rng.random(12).astype(np.float32)
    check(run(gpu, z, *args, u), ref(z.astype(np.float32), *args, u))


@pytest.mark.parametrize("V", [20000, 65536, 400000])
@pytest.mark.parametrize("kind", ["peaked", "flat", "few values"])
def test_every_top_k(gpu, kind, V):
    """Where the lists end and the histograms begin, and candidates in more slots than either holds"""
    rng = np.random.default_rng(21)
    k = np.array([63, 64, 65, 192, 255, 256, 257, 258, 600, 2000, 7000, 384, 500, 511, 512, 513, V // 128 - 1, V // 128, V // 128 + 1])
    rows = len(k)
    z = logits_of(rng, rows, V, kind)
    args = np.ones(rows), k, np.where(np.arange(rows) % 2, 0.98, 1.0), np.zeros(rows)
    u = rng.random(rows).astype(np.float32)
    check(run(gpu, z, *args, u), ref(z, *args, u))


def test_the_largest_vocabulary(gpu):
    rng = np.random.default_rng(8)
    z = logits_of(rng, 6, 1048576, "flat")
    t, k, p, mp = np.ones(6), np.array([0, 0, 50, 900000, 0, 0]), np.array([1.0, 0.9, 1, 1, 0.0, 1.0]), np.array([0, 0, 0, 0, 0, 0.9])
    u = rng.random(6).astype(np.float32)
    check(run(gpu, z, t, k, p, mp, u), ref(z, t, k, p, mp, u))
    with pytest.raises(gpu.RwkvHipError, match="V must lie in"):
        gpu.draw_tokens(1, 1048577, 4096, 4096, 4096, None)


@pytest.mark.parametrize("ld,offset", [(1001, 0), (1000, 1), (1003, 3), (1024, 2), (1024, 4), (4096, 8)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_rows_apart_and_anywhere(gpu, ld, offset, dtype):
    rng = np.random.default_rng(5)
    z = logits_of(rng, 12, 1000, "peaked", dtype)
    args, u = styles(12), rng.random(12).astype(np.float32)
    got = run(gpu, z, *args, u, ld=ld, offset=offset)
    check(got, ref(z.astype(np.float32), *args, u))
    same = run(gpu, z, *args, u)
    assert np.array_equal(got[0], same[0]) and np.array_equal(got[1], same[1])


def test_equal_entries_are_counted_exactly(gpu):
    """Every entry alike: token j belongs to u in [j, j + 1) / V, and filters keep the first ones by index."""
    for V in (64, 1024, 8192, 65536):
        z = np.full((16, V), -2.5, np.float32)
        u = (np.arange(16) * (V // 16) / V).astype(np.float32)
        assert np.array_equal(run(gpu, z, u=u)[0], np.arange(16) * (V // 16))
        assert np.array_equal(run(gpu, z, k=np.full(16, V // 2), u=u)[0], np.arange(16) * (V // 32))
        assert np.array_equal(run(gpu, z, p=np.full(16, 0.5), u=u)[0], np.arange(16) * (V // 32))
        got = run(gpu, z, p=np.full(16, 0.25), k=np.full(16, 10 ** 9), mp=np.ones(16), u=np.full(16, 1.0))
        assert np.array_equal(got[0], np.full(16, V // 4 - 1)) and np.array_equal(got[1], np.full(16, np.float32(-np.log(V // 4)), np.float64))


def test_the_ends_of_every_parameter(gpu):
    rng = np.random.default_rng(2)
    V = 3000
    cases = [(t, k, p, mp, u) for t in (0.0, 1e-45, 1e-3, 1.0, 1e30, np.inf) for k in (-5, 0, 1, 2, V - 1, V, V + 1, 2 ** 31 - 1)
             for p, mp, u in ((1.0, 0.0, 0.0), (1.0, 0.0, 1.0), (0.0, 0.0, 0.7), (-1.0, 2.0, 0.3), (2.0, -1.0, 0.999), (1e-38, 1e-38, 0.5), (0.7, 1.0, 0.5),
                              (np.inf, 1e-45, 0.25), (-np.inf, np.inf, 0.5))]
    args = [np.array(c) for c in zip(*cases)]
    z = logits_of(rng, len(cases), V, "peaked")
    z[:, 7] = z[:, 1234] = 20.0  # two largest ones
    with np.errstate(over="ignore"):
        check(run(gpu, z, *args[:4]), ref(z, *args[:4], np.full(len(cases), 0.5)))
        check(run(gpu, z, *args[:4], args[4]), ref(z, *args))


@pytest.mark.parametrize("V", [130, 70000])
def test_rows_without_a_distribution(gpu, V):
    rng = np.random.default_rng(4)
    z = logits_of(rng, 14, V, "flat")
    z[0] = -np.inf                       # nothing left
    z[1, V - 1] = np.nan
    z[2, 0] = np.inf
    z[3, :] = -np.inf
    z[3, 77] = -3.0                      # one left
    z[4, :] = np.finfo(np.float32).min   # masked with the type's lowest value, all
    z[5, :] = np.finfo(np.float32).min   # and all but two
    z[5, 5], z[5, 99] = 1.0, 1.5
    z[6] = -np.inf
    z[6, 3] = np.nan                     # nothing but masked places and a NaN
    z[7, 1::2] = -np.inf
    z[8] = np.finfo(np.float32).max      # the largest finite ones are entries like any other
    t, k, p, mp, u = (np.ones(14), np.zeros(14), np.ones(14), np.zeros(14), np.full(14, 0.4, np.float32))
    t[9], p[10], mp[11], u[12], u[13] = np.nan, np.nan, np.nan, np.nan, 1.25
    for kk, pp in ((0, 1.0), (50, 0.9), (0, 0.9), (20000, 1.0)):
        args = (t, np.full(14, kk), np.where(np.isnan(p), p, pp), mp, u)
        got = run(gpu, z, *args)
        check(got, ref(z, *args))
        assert list(got[0][[0, 1, 2, 6, 9, 10, 11, 12, 13]]) == [-1] * 9 and got[0][3] == 77
    t[0] = -1.0
    assert run(gpu, z, t, k, p, mp, u)[0][0] == -1


def test_half_precision_masks(gpu):
    z = np.full((3, 500), np.finfo(np.float16).min, np.float16)
    z[0, 100:103] = 1.0
    z[2] = -np.inf
    u = np.array([0.5, 0.5, 0.5], np.float32)
    got = run(gpu, z, u=u)
    check(got, ref(z.astype(np.float32), np.ones(3), np.zeros(3), np.ones(3), np.zeros(3), u))
    assert list(got[0]) == [101, 250, -1]


@pytest.mark.parametrize("V", [60, 1000, 4600, 20000])
def test_the_last_entry_of_all(gpu, V):
    """A number of 1 takes the last kept entry, however the sums in front of it are rounded"""
    rng = np.random.default_rng(V)
    rows = 600 if V < 5000 else 48
    for kind in ("peaked", "flat"):
        z = logits_of(rng, rows, V, kind)
        z[:, -3:] = z.max() - 60.0  # (beside which they vanish)
        args = styles(rows)
        u = np.ones(rows, np.float32)
        check(run(gpu, z, *args, u), ref(z, *args, u))


@pytest.mark.parametrize("mask", [-65504.0, -3.4e38, -800.0, -600.0])
@pytest.mark.parametrize("V,dtype", [(5000, np.float32), (65536, np.float32), (50277, np.float16)])
def test_masks_of_a_finite_value(gpu, mask, V, dtype):
    """Fewer entries that are not masked than the filters ask for; masks with a probability of nothing, and of a little"""
    rng = np.random.default_rng(31)
    rows = 12
    z = np.full((rows, V), max(mask, float(np.finfo(dtype).min)), dtype)
    for r in range(rows):
        z[r, rng.integers(0, V, 1 + 5 * r)] = rng.standard_normal(1 + 5 * r) * 3.0
    args = styles(rows)
    for top_k in (args[1], np.full(rows, 50), np.full(rows, 700)):
        args[1] = top_k
        for u in (rng.random(rows), np.zeros(rows), np.ones(rows)):
            u = u.astype(np.float32)
            check(run(gpu, z, *args, u), ref(z.astype(np.float32), *args, u))


@pytest.mark.parametrize("u", [0.0, 1.0])
def test_entries_below_every_power(gpu, u):
    """Entries some 1000 octaves below the largest have no probability, whatever they are beside the largest of their own part"""
    rows, V = 8, 9000
    z = np.full((rows, V), -np.inf, np.float32)
    octave = np.float32(np.log(2.0))
    z[:, 5000] = 0.0
    z[:, 100:200] = -1040.0 * octave - np.arange(100, dtype=np.float32) * 0.25   # (the first part's and the last one's own largest)
    z[:, 8500:8600] = -1040.0 * octave
    z[:, 4500] = z[:, 5500] = -990.0 * octave
    z[::2, 3000] = z[::2, 8700] = -990.0 * octave
    args = [np.ones(rows), np.array([0, 0, 2, 50, 600, 0, 0, 0]), np.array([1, 1, 1, 1, 1, 0.999, 1, 1]), np.array([0, 1e-30, 0, 0, 0, 0, 0, 0])]
    u = np.full(rows, u, np.float32)
    check(run(gpu, z, *args, u), ref(z, *args, u))


def test_rows_that_are_nearly_sure(gpu):
    """The log probability of a token that has nearly all of the row: what is left is not lost beside the 1"""
    rng = np.random.default_rng(6)
    z = np.full((30, 65536), -np.inf, np.float32)
    z[:, 40000] = 0.0
    for i in range(30):
        z[i, rng.integers(0, 40000, 5)] = -2.0 * i
    for args in ((0, 1.0), (100, 1.0), (0, 0.9999999)):
        a = (np.ones(30), np.full(30, args[0]), np.full(30, args[1]), np.zeros(30), np.full(30, 0.999999, np.float32))
        check(run(gpu, z, *a), ref(z, *a))


def test_several_rows_draw_from_one(gpu):
    rng = np.random.default_rng(9)
    z = logits_of(rng, 3, 9000, "peaked")
    source = np.array([2, 2, 0, 1, 2, 0, 2, 3, -1, 2, 1, 0])
    args, u = styles(12), rng.random(12).astype(np.float32)
    got = run(gpu, z, *args, u, source=source, rows=12)
    want = ref(z[np.clip(source, 0, 2)], *args, u)
    for i in (7, 8):  # outside the rows
        want[0][i], want[1][i] = -1, 0.0
    check(got, want)


def test_a_row_does_not_depend_on_its_batch(gpu):
    rng = np.random.default_rng(10)
    for V in (3001, 65536):
        z = logits_of(rng, 40, V, "peaked")
        args, u = styles(40), rng.random(40).astype(np.float32)
        whole = run(gpu, z, *args, u)
        order = rng.permutation(40)
        moved = run(gpu, z[order], *[a[order] for a in args], u[order])
        assert np.array_equal(moved[0], whole[0][order]) and np.array_equal(moved[1], whole[1][order])
        for i in range(0, 40, 7):
            one = run(gpu, z[i:i + 1], *[a[i:i + 1] for a in args], u[i:i + 1])
            assert one[0][0] == whole[0][i] and one[1][0] == whole[1][i]


@pytest.mark.parametrize("rows", [300, 1100])
def test_many_rows(gpu, rows):
    """Launches of every width"""
    rng = np.random.default_rng(rows)
    V = 4500
    z = logits_of(rng, rows, V, "peaked")
    args, u = styles(rows), rng.random(rows).astype(np.float32)
    check(run(gpu, z, *args, u), ref(z, *args, u))


@pytest.mark.parametrize("out", ["apart", "in place"])
@pytest.mark.parametrize("V", [1000, 4099])
def test_penalties(gpu, out, V):
    rng = np.random.default_rng(11)
    rows = 14
    z = logits_of(rng, rows, V, "peaked")
    pen = np.where(rng.random((rows, V)) < 0.2, rng.random((rows, V)) * 3.0, 0.0).astype(np.float32)
    pen[:, int(np.argmax(z[0]))] = 0.0
    args, u = styles(rows), rng.random(rows).astype(np.float32)
    presence, frequency, decay = (rng.random(rows).astype(np.float32) + s for s in (1.0, 0.1, 0.0))
    z[3] = -np.inf  # no token: decayed all the same
    token, logprob, after = run(gpu, z, *args, u, penalties=pen, out=out, presence=presence, frequency=frequency, decay=decay)
    want = ref(z - pen, *args, u)
    check((token, logprob), want)
    for i in range(rows):
        p = pen[i].astype(np.float64) * np.float64(decay[i])
        if token[i] >= 0:
            p[token[i]] += np.float64(presence[i] if pen[i, token[i]] == 0 else frequency[i])
        assert np.array_equal(after[i], p.astype(np.float32))  # (one rounding on both sides)
    # only subtracted, and only decayed
    check(run(gpu, z, *args, u, penalties=pen), want)
    token, _, after = run(gpu, z, *args, u, penalties=pen, out=out)
    assert np.array_equal(after, pen)


def test_penalties_that_are_not_finite_leave_no_distribution(gpu):
    z = np.zeros((3, 100), np.float32)
    pen = np.zeros((3, 100), np.float32)
    pen[0, 5], pen[1, 5], pen[2, 5] = np.nan, -np.inf, np.inf
    assert list(run(gpu, z, u=np.full(3, 0.5), penalties=pen)[0]) == [-1, -1, 50]


def test_rows_beyond_32_bits(gpu):
    """Rows 1.2e9 entries apart: the last one lies behind 2^31 entries and 4 GiB."""
    hip = gpu
    rng = np.random.default_rng(12)
    V, ld, rows = 5000, 1200000000, 3
    z = logits_of(rng, rows, V, "peaked", np.float16)
    big = hip.DeviceArray(((rows - 1) * ld + V,), np.float16)
    for i in range(rows):
        big.view(i * ld, (V,)).upload(z[i])
    u = np.array([0.2, 0.5, 0.8], np.float32)
    token, logprob, ws = hip.DeviceArray((rows,), np.int32), hip.DeviceArray((rows,), np.float32), hip.DeviceArray((hip.draw_tokens_workspace(rows, V),), np.uint8)
    hip.draw_tokens(rows, V, big, hip.DeviceArray.from_numpy(u), token, ws, logprob=logprob, io=hip.IO_F16, ld=ld)
    hip.device_sync()
    check((token.numpy(), logprob.numpy().astype(np.float64)), ref(z.astype(np.float32), np.ones(3), np.zeros(3), np.ones(3), np.zeros(3), u))
    big.free()


def call_of(hip, rows, V, seed):
    rng = np.random.default_rng(seed)
    dev = hip.DeviceArray.from_numpy
    t, k, p, mp = styles(rows)
    keep = dict(z=dev(logits_of(rng, rows, V, "peaked")), u=dev(rng.random(rows).astype(np.float32)), t=dev(t.astype(np.float32)), k=dev(k.astype(np.int32)),
                p=dev(p.astype(np.float32)), mp=dev(mp.astype(np.float32)), pen=dev(rng.random((rows, V)).astype(np.float32)),
                decay=dev(np.full(rows, 0.5, np.float32)), ws=hip.DeviceArray((hip.draw_tokens_workspace(rows, V),), np.uint8))
    out = dict(token=hip.DeviceArray.zeros((rows,), np.int32), logprob=hip.DeviceArray.zeros((rows,), np.float32), pen=hip.DeviceArray.zeros((rows, V), np.float32))

    def launch(stream):
        hip.draw_tokens(rows, V, keep["z"], keep["u"], out["token"], keep["ws"], logprob=out["logprob"], temperature=keep["t"], top_k=keep["k"],
                        top_p=keep["p"], min_p=keep["mp"], penalties=keep["pen"], decay=keep["decay"], penalties_out=out["pen"], stream=stream)

    return launch, out, keep


def bits(out):
    return {n: v.numpy().view(np.uint8).copy() for n, v in out.items()}


def test_a_captured_call_replays(gpu):
    hip = gpu
    launch, out, keep = call_of(hip, 13, 20000, 21)
    s = Stream(hip)
    lib = s.lib
    graph, exe = ctypes.c_void_p(0), ctypes.c_void_p(0)
    assert lib.hipStreamBeginCapture(ctypes.c_void_p(s.ptr), ctypes.c_int(1)) == 0
    launch(s.ptr)
    assert lib.hipStreamEndCapture(ctypes.c_void_p(s.ptr), ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    rng = np.random.default_rng(1)
    for _ in range(4):
        keep["z"].upload(logits_of(rng, 13, 20000, "peaked"))
        keep["u"].upload(rng.random(13).astype(np.float32))
        launch(None)
        hip.device_sync()
        want = bits(out)
        for v in out.values():
            v.fill0()
        hip.device_sync()
        assert lib.hipGraphLaunch(exe, ctypes.c_void_p(s.ptr)) == 0
        s.sync()
        got = bits(out)
        assert all(np.array_equal(got[n], want[n]) for n in want)
    assert lib.hipGraphExecDestroy(exe) == 0 and lib.hipGraphDestroy(graph) == 0
    s.close()


def test_calls_of_several_threads_and_streams(gpu):
    import threading
    hip = gpu
    calls = [call_of(hip, rows, V, seed) for rows, V, seed in ((5, 9000, 31), (40, 4100, 32), (2, 65536, 33))]
    want = []
    for launch, out, _ in calls:
        launch(None)
        hip.device_sync()
        want.append(bits(out))
        for v in out.values():
            v.fill0()
    hip.device_sync()
    streams, errors = [Stream(hip) for _ in calls], []

    def work(i):
        try:
            for _ in range(50):
                calls[i][0](streams[i].ptr)
                streams[i].sync()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (_, out, _), w in zip(calls, want):
        got = bits(out)
        assert all(np.array_equal(got[n], w[n]) for n in w)
    for s in streams:
        s.close()


def test_draws_follow_the_probabilities(gpu):
    """4096 evenly spaced numbers draw every token as often as its probability says, to one draw at either end"""
    rng = np.random.default_rng(13)
    z = logits_of(rng, 1, 300, "flat")
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    token, _ = run(gpu, z, t=np.full(n, 0.5), u=u, source=np.zeros(n), rows=n)
    p = np.exp((z[0].astype(np.float64) - z.max()) / 0.5)
    count = np.bincount(token, minlength=300)
    assert np.all(np.abs(count - n * p / p.sum()) <= 1.0 + 1e-9) and np.all(np.diff(token) >= 0)
