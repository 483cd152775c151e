"""draw_tokens where the cut lies among entries that are tens of octaves below the largest: how many of them are kept is a comparison of sums
that agree in their first eight digits or more.  Rows of few values, so that the definition can be taken with fifty digits."""
import math
from decimal import Decimal, getcontext

import numpy as np
import pytest

from test_gpu_draw_tokens import check, run

pytestmark = pytest.mark.gpu

getcontext().prec = 50
BELOW_ONE = 1.0 - 2.0 ** -24  # the largest top_p that is on


def ref_levels(z, t, k, p, u):
    """(token, log probability) of a row of few values.  Powers and sums with fifty digits.  What decides is asserted to lie further from a border
    than 64-bit sums can be off: sums of at most 2 with some 32 roundings of 2^-53, and powers beside the largest good to 4e-14."""
    t, p, u = (Decimal(float(np.float32(v))) for v in (t, p, u))
    values, which = np.unique(z, return_inverse=True)
    m = Decimal(float(values[-1]))
    e = [Decimal(0) if v == -np.inf else ((Decimal(float(v)) - m) / t).exp() for v in values]
    have = np.bincount(which, minlength=len(values))
    total = sum(int(n) * w for n, w in zip(have, e))
    tail = total - int(have[-1])
    slack = (1 + tail) * 32 * Decimal(2) ** -53 + tail * Decimal("1e-13")
    # kept entries of every level, the largest first
    keep = np.zeros(len(values), np.int64)
    above, number = Decimal(0), 0
    left = k if 0 < k < len(z) else len(z)
    for level in range(len(values) - 1, -1, -1):
        n = int(have[level])
        if e[level] == 0:
            break
        want = n
        if p < 1:
            need = p * total - above
            assert abs(need - n * e[level]) > slack, "the end of a level"
            if need <= n * e[level]:
                want = max(1, int((need / e[level]).to_integral_value("ROUND_CEILING")))
                if need > 0:
                    assert min(want * e[level] - need, need - (want - 1) * e[level]) > slack, "an entry's end"
        keep[level] = min(want, left - number)
        above += int(keep[level]) * e[level]
        number += int(keep[level])
        if want < n or number == left:
            break
        if p < 1 and above >= p * total:
            break
    # running sums by index: entries of each level so far that are kept
    so_far = [np.minimum(np.cumsum(which == level), keep[level]) if e[level] > 0 else None for level in range(len(values))]
    upto = lambda i: sum((int(c[i]) * w for c, w in zip(so_far, e) if c is not None), Decimal(0)) if i >= 0 else Decimal(0)  # noqa: E731
    kept = upto(len(z) - 1)
    if u == 1:
        token = max(int(np.nonzero(np.diff(c, prepend=0))[0][-1]) for c, n in zip(so_far, keep) if n > 0)
    else:
        lo, hi = 0, len(z) - 1  # the first with a sum above u times the whole
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if upto(mid) > u * kept else (mid + 1, hi)
        token = lo
        assert upto(token) - u * kept > slack and (token == 0 or u * kept - upto(token - 1) > slack or upto(token - 1) == 0), "a token's end"
    weight = e[which[token]]
    return token, float(-((kept - weight) / weight + 1).ln())


def check_levels(hip, rows, chunk=4):
    """rows: (z, t, k, p, u), all of one length"""
    for at in range(0, len(rows), chunk):
        some = rows[at:at + chunk]
        z = np.stack([r[0] for r in some])
        t, k, p, u = (np.array([r[i] for r in some]) for i in range(1, 5))
        want = [ref_levels(*r) for r in some]
        got = run(hip, z, t, k, p, np.zeros(len(some)), u.astype(np.float32))
        check(got, (np.array([w[0] for w in want], np.int32), np.array([w[1] for w in want])))


def two_levels(V, seed, first, second, share):
    """The largest entry alone in its part; behind it entries of two values in any order"""
    rng = np.random.default_rng(seed)
    z = np.full(V, -np.inf, np.float32)
    z[0] = 0.0
    rest = np.full(V - 4096, second, np.float32)
    rest[rng.permutation(V - 4096)[:share]] = first
    z[4096:] = rest
    return z


def level_end(z, first):
    """The largest top_p with which the entries from `first` up are just enough"""
    values, have = np.unique(z[z > -np.inf], return_counts=True)
    w = [int(n) * Decimal(float(v)).exp() for v, n in zip(values, have)]
    share = sum(x for x, v in zip(w, values) if v >= first) / sum(w)
    p = np.float32(share)
    return p if Decimal(float(p)) <= share else np.nextafter(p, np.float32(0))


@pytest.mark.parametrize("V", [65536, 1048576])
def test_what_lies_below_the_window_is_not_kept(gpu, V):
    """The cut is the last entry of a level of many, in front of another: sums that are rounded otherwise than the histograms' miss it"""
    if V == 65536:
        z = two_levels(V, 1, -14.296875, -15.296875, 32768)
        rows = [(z, 1.0, 0, 0.9936519861221313, u) for u in (0.99, 0.995, 1.0)]
    else:
        rows = []
        for i, step in enumerate((1802, 1811, 1823, 1832, 1840, 1857)):
            first = -step / 128
            z = two_levels(V, 2 + i, first, first - 1.0, V // 2)
            rows += [(z, 1.0, 0, level_end(z, first), u) for u in (0.8, 1.0)]
    check_levels(gpu, rows)


def down(octaves):
    """A value so many octaves below 0 or a little more, exact in 32 bits beside numbers of a few tens"""
    return -math.ceil(octaves * math.log(2.0) * 64) / 64


def floor_row(V, seed, levels, n=None, alone=True, top=0.0):
    """One large entry and `n` (default: all) others of the values `levels` in turn, in any order; alone: the first part has only the large one"""
    rng = np.random.default_rng(seed)
    z = np.full(V, -np.inf, np.float32)
    free = np.arange(4096 if alone else 0, V)
    at = free if n is None else rng.permutation(free)[:n]
    z[at] = rng.permutation(np.resize(np.asarray(levels) + top, len(at)))
    z[0 if alone else int(rng.integers(0, V))] = top
    return z


# octaves of the others, how many, top_k, top_p: all of them to be searched in memory; a list; a list of a top_k's; a window in memory; a window's list
CUTS = {
    "row": [([33], None, 0, BELOW_ONE), ([36, 36.4], None, 0, BELOW_ONE), ([39], None, 0, BELOW_ONE)],
    "list": [([33], 5000, 0, BELOW_ONE), ([35], 5000, 0, BELOW_ONE), ([30, 33.5], 3000, 0, 1.0 - 2.0 ** -20)],
    "top_k": [([31.5], 400, 512, BELOW_ONE), ([30.25, 32], 500, 500, BELOW_ONE), ([30], 300, 512, 1.0 - 2.0 ** -23)],
    "window": [([25], None, 0, 0.999), ([20.5, 24], None, 0, 0.98), ([12, 13, 14, 28], None, 0, 0.5)],
    "window's list": [(np.arange(24, 28, 0.03), None, 0, 1.0 - 2.0 ** -12), (np.arange(14, 20, 0.05), None, 0, 0.9)],
}


@pytest.mark.parametrize("path", list(CUTS))
@pytest.mark.parametrize("V", [65536, 300001])
def test_cuts_far_below_the_largest(gpu, V, path):
    rows = [(floor_row(V, 40 + i, [down(o) for o in octaves], n), 1.0, k, p, u) for i, (octaves, n, k, p) in enumerate(CUTS[path])
            for u in (0.5, 0.9999995, 1.0)]
    check_levels(gpu, rows)


@pytest.mark.parametrize("octaves", [36, 39, 41.99, 42.6, 43.5])
def test_cuts_of_the_largest_vocabulary(gpu, octaves):
    z = floor_row(1048576, 7, [down(octaves)])
    check_levels(gpu, [(z, 1.0, 0, BELOW_ONE, u) for u in (0.5, BELOW_ONE, 1.0)])


@pytest.mark.parametrize("path", list(CUTS))
@pytest.mark.parametrize("V", [65536, 300001])
def test_cuts_beside_the_largest_in_its_own_part(gpu, V, path):
    """The others stand in the part of the largest, too, whose histogram has to hold both"""
    rows = [(floor_row(V, 60 + i, [down(o) for o in octaves], n, alone=False), 1.0, k, p, u) for i, (octaves, n, k, p) in enumerate(CUTS[path])
            for u in (0.5, 0.9999995, 1.0)]
    check_levels(gpu, rows)


@pytest.mark.parametrize("octaves", [36, 39, 41.99, 42.6, 43.5])
def test_cuts_of_the_largest_vocabulary_anywhere(gpu, octaves):
    z = floor_row(1048576, 8, [down(octaves)], alone=False)
    check_levels(gpu, [(z, 1.0, 0, BELOW_ONE, u) for u in (0.5, BELOW_ONE, 1.0)])


def test_few_parts_with_a_low_floor(gpu):
    """One part or two: what the floor's powers lose beside the largest all falls on one sum"""
    rows = [(floor_row(8000, 90 + i, [down(o)], alone=False), 1.0, 0, BELOW_ONE, u) for i, o in enumerate((33, 34, 35.5, 36.3)) for u in (0.5, 1.0)]
    check_levels(gpu, rows)


@pytest.mark.parametrize("t", [1e-4, 1e-5, 1e-6, 1e-7, 1e-20, 50.0, 1e10])
def test_cuts_at_any_temperature(gpu, t):
    """At low temperatures neighbours among the numbers lie octaves apart, and their places on the histograms' grid far behind 2^24"""
    t = float(np.float32(t))
    rows = []
    for i, octaves in enumerate((20, 33.5, 36.7)):
        for at, top in ((777, 0.0), (40000, 9.75), (65535, -30.0)):
            z = np.full(65536, top - octaves * math.log(2.0) * t, np.float32)
            z[at] = top
            if z[0] == z[at]:
                z[at] = np.nextafter(z[at], np.float32(np.inf))
            rows += [(z, t, 0, p, u) for p, u in ((BELOW_ONE, 0.5), (BELOW_ONE, 1.0), (0.75, 1.0))]
    check_levels(gpu, rows)


def ref_spread(z, t, p, u):
    """As ref_levels for rows of any values, with top_p alone: powers and sums of 64 bits behind the point (long double)"""
    ld = np.longdouble
    z, t, p, u = z.astype(ld), ld(np.float32(t)), ld(np.float32(p)), ld(np.float32(u))
    y = (z - z.max()) / t
    e = np.where(y < -1000 * math.log(2.0), ld(0), np.exp(np.maximum(y, ld(-1000))))
    order = np.lexsort((np.arange(len(z)), -z))
    upto = np.cumsum(e[order])
    total = upto[-1]
    tail = total - e[order[0]]
    slack = (1 + tail) * 32 * ld(2) ** -53 + tail * ld(1e-13)
    n = int(np.searchsorted(upto, p * total)) + 1
    assert upto[n - 1] - p * total > slack and (n == 1 or p * total - upto[n - 2] > slack), "an entry's end"
    kept = np.zeros(len(z), ld)
    kept[order[:n]] = e[order[:n]]
    upto = np.cumsum(kept)
    if u == 1:
        token = int(np.nonzero(kept)[0][-1])
    else:
        token = int(np.nonzero((upto > u * upto[-1]) & (kept > 0))[0][0])
        assert upto[token] - u * upto[-1] > slack and (token == 0 or u * upto[-1] - upto[token - 1] > slack or upto[token - 1] == 0), "a token's end"
    others = np.sort(np.delete(kept, token)).sum()
    return token, float(-np.log1p(others / kept[token]))


def check_spread(hip, rows):
    z = np.stack([r[0] for r in rows])
    t, p, u = (np.array([r[i] for r in rows], np.float32) for i in (1, 2, 3))
    want = [ref_spread(*r) for r in rows]
    got = run(hip, z, t, np.zeros(len(rows)), p, np.zeros(len(rows)), u)
    check(got, (np.array([w[0] for w in want], np.int32), np.array([w[1] for w in want])))


@pytest.mark.parametrize("V", [9000, 65536])
@pytest.mark.parametrize("ends", [(36, 39), (20, 40), (5, 45)])
def test_tails_that_are_spread(gpu, V, ends):
    rng = np.random.default_rng([V, *ends])
    rows = []
    for i, p in enumerate((BELOW_ONE, 0.9999999, 0.9999998, 0.999999, 0.9999, 0.9)):
        z = rng.uniform(-ends[1], -ends[0], V).astype(np.float32) * np.float32(math.log(2.0))
        z[rng.integers(0, V)] = 0.0
        t = (1.0, 0.7, 1.3)[i % 3]
        rows += [(z * np.float32(t), t, p, u) for u in (float(rng.random()), 1.0)]
    check_spread(gpu, rows)
