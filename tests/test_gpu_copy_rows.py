"""copy_rows against the same moves made on the host."""
import ctypes

import numpy as np
import pytest

from test_gpu_draw_tokens import Stream

pytestmark = pytest.mark.gpu

GUARD = 64


def host(src, dst, to, rows):
    out = dst.copy()
    for d, r in zip(to, rows):
        out[:, d] = 0 if r < 0 else src[:, r]
    return out


class Buffers:
    """Byte tensors [planes, rows, row_bytes] at an offset in their allocations, with guards around"""

    def __init__(self, hip, rng, shapes, rows, offset=0):
        self.hip, self.rows, self.offset, self.of = hip, rows, offset, []
        for planes, row_bytes in shapes:
            data = rng.integers(0, 256, (planes, rows, row_bytes), dtype=np.uint8)
            flat = np.concatenate([np.full(GUARD + offset, 0xAB, np.uint8), data.ravel(), np.full(GUARD, 0xAB, np.uint8)])
            self.of.append((data, hip.DeviceArray.from_numpy(flat)))

    def ptr(self, i):
        return self.of[i][1].ptr + GUARD + self.offset

    def now(self, i):
        flat = self.of[i][1].numpy()
        data = self.of[i][0]
        at = GUARD + self.offset
        assert np.all(flat[:at] == 0xAB) and np.all(flat[at + data.size:] == 0xAB)
        return flat[at:at + data.size].reshape(data.shape)


STATE = [(4, 1536), (2, 49152), (1, 4)]                              # shift, wkv, elapsed of a small model
ODD = [(3, 1), (2, 2), (1, 3), (5, 6), (1, 20), (2, 4097), (3, 40000), (1, 16)]


@pytest.mark.parametrize("shapes", [STATE, ODD], ids=["state", "odd"])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_between_two_sets_of_rows(gpu, shapes, offset, n):
    rng = np.random.default_rng(n)
    src, dst = Buffers(gpu, rng, shapes, 17, offset), Buffers(gpu, rng, shapes, 24, offset)
    to = rng.permutation(24)[:n]
    rows = rng.integers(-1, 17, n)  # some of them cleared, some twice
    gpu.copy_rows([(dst.ptr(i), src.ptr(i), p, b) for i, (p, b) in enumerate(shapes)], 24, 17, to, rows)
    gpu.device_sync()
    for i in range(len(shapes)):
        assert np.array_equal(dst.now(i), host(src.of[i][0], dst.of[i][0], to, rows)), i
        assert np.array_equal(src.now(i), src.of[i][0])


def moves_of(kind, rng, rows):
    if kind == "fork":
        return list(range(1, rows)), [0] * (rows - 1)
    if kind == "shift down":
        return list(range(rows - 1)), list(range(1, rows))
    if kind == "shift up":
        return list(range(1, rows)), list(range(rows - 1))
    if kind == "swap":
        return [2, 5], [5, 2]
    if kind == "turn":
        return list(range(rows)), [(i + 1) % rows for i in range(rows)]
    if kind == "reverse":
        return list(range(rows)), list(range(rows))[::-1]
    if kind == "compact":
        live = sorted(rng.permutation(rows)[: rows // 2].tolist())
        return list(range(rows)), live + [-1] * (rows - len(live))
    if kind == "clear":
        return [3, 0], [-1, -1]
    if kind == "stay":
        return [3, 0], [3, 0]
    to = rng.permutation(rows)
    return to.tolist(), rng.integers(-1, rows, rows).tolist()


@pytest.mark.parametrize("kind", ["fork", "shift down", "shift up", "swap", "turn", "reverse", "compact", "clear", "stay", "any", "any more"])
@pytest.mark.parametrize("shapes", [STATE, ODD], ids=["state", "odd"])
@pytest.mark.parametrize("rows", [7, 29])
def test_in_place(gpu, kind, shapes, rows):
    rng = np.random.default_rng([rows, len(kind)])
    b = Buffers(gpu, rng, shapes, rows)
    to, source = moves_of(kind, rng, rows)
    gpu.copy_rows([(b.ptr(i), b.ptr(i), p, n) for i, (p, n) in enumerate(shapes)], rows, rows, to, source)
    gpu.device_sync()
    for i in range(len(shapes)):
        assert np.array_equal(b.now(i), host(b.of[i][0], b.of[i][0], to, source)), i


def test_the_most_moves(gpu):
    rng = np.random.default_rng(3)
    for source in ([(i + 1) % 512 for i in range(512)], rng.permutation(512).tolist(), [i ^ 1 for i in range(512)]):
        b = Buffers(gpu, rng, [(2, 80), (1, 4)], 600)
        gpu.copy_rows([(b.ptr(0), b.ptr(0), 2, 80), (b.ptr(1), b.ptr(1), 1, 4)], 600, 600, list(range(512)), source)
        gpu.device_sync()
        for i in range(2):
            assert np.array_equal(b.now(i), host(b.of[i][0], b.of[i][0], range(512), source))


def test_no_moves(gpu):
    b = Buffers(gpu, np.random.default_rng(1), STATE, 5)
    gpu.copy_rows([(b.ptr(i), b.ptr(i), p, n) for i, (p, n) in enumerate(STATE)], 5, 5, [], [])
    gpu.device_sync()
    assert all(np.array_equal(b.now(i), b.of[i][0]) for i in range(3))


def test_rows_beyond_32_bits(gpu):
    """A tensor of 6 GiB: rows of 3 MiB in 4 planes of 512, the last ones behind 2^32 bytes"""
    hip = gpu
    planes, rows, row = 4, 512, 3 << 20
    big = hip.DeviceArray((planes * rows * row,), np.uint8)
    rng = np.random.default_rng(4)
    piece = {r: rng.integers(0, 256, (planes, row), dtype=np.uint8) for r in (0, 500)}
    for r, data in piece.items():
        for p in range(planes):
            big.view((p * rows + r) * row, (row,)).upload(data[p])
    hip.copy_rows([(big, big, planes, row)], rows, rows, [511, 1, 500], [0, 500, 511])
    hip.copy_rows([(big, big, planes, row)], rows, rows, [510], [-1])
    hip.device_sync()
    for p in range(planes):
        at = lambda r: big.view((p * rows + r) * row, (row,)).numpy()  # noqa: E731, B023
        assert np.array_equal(at(511), piece[0][p]) and np.array_equal(at(1), piece[500][p]) and not at(510).any() and np.array_equal(at(0), piece[0][p])
    big.free()


def test_a_captured_call_replays(gpu):
    hip = gpu
    rng = np.random.default_rng(5)
    src, dst = Buffers(hip, rng, STATE, 9), Buffers(hip, rng, STATE, 9)
    to, rows = [0, 4, 8, 2], [3, 3, -1, 1]
    s = Stream(hip)
    lib = s.lib
    graph, exe = ctypes.c_void_p(0), ctypes.c_void_p(0)
    assert lib.hipStreamBeginCapture(ctypes.c_void_p(s.ptr), ctypes.c_int(1)) == 0
    hip.copy_rows([(dst.ptr(i), src.ptr(i), p, n) for i, (p, n) in enumerate(STATE)], 9, 9, to, rows, stream=s.ptr)
    hip.copy_rows([(src.ptr(i), src.ptr(i), p, n) for i, (p, n) in enumerate(STATE)], 9, 9, [0, 1, 2], [1, 2, 0], stream=s.ptr)
    assert lib.hipStreamEndCapture(ctypes.c_void_p(s.ptr), ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    now_src, now_dst = [d for d, _ in src.of], [d for d, _ in dst.of]
    for _ in range(4):
        assert lib.hipGraphLaunch(exe, ctypes.c_void_p(s.ptr)) == 0
        s.sync()
        now_dst = [host(a, b, to, rows) for a, b in zip(now_src, now_dst)]
        now_src = [host(a, a, [0, 1, 2], [1, 2, 0]) for a in now_src]
        for i in range(3):
            assert np.array_equal(dst.now(i), now_dst[i]) and np.array_equal(src.now(i), now_src[i])
    assert lib.hipGraphExecDestroy(exe) == 0 and lib.hipGraphDestroy(graph) == 0
    s.close()


def test_two_streams_at_once(gpu):
    hip = gpu
    rng = np.random.default_rng(6)
    pools = [Buffers(hip, rng, STATE, 20) for _ in range(2)]
    streams = [Stream(hip) for _ in pools]
    turn = [(i + 1) % 20 for i in range(20)]
    for _ in range(15):
        for pool, s in zip(pools, streams):
            hip.copy_rows([(pool.ptr(i), pool.ptr(i), p, n) for i, (p, n) in enumerate(STATE)], 20, 20, list(range(20)), turn, stream=s.ptr)
    for s in streams:
        s.sync()
        s.close()
    for pool in pools:
        for i in range(3):
            assert np.array_equal(pool.now(i), np.roll(pool.of[i][0], -15, axis=1))
