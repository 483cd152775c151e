"""copy_rows of 256 MiB and more, which go past the caches: forks, gathers and cleared rows of every unit, and behind 2^32 bytes."""
import numpy as np
import pytest

from test_gpu_copy_rows import Buffers, host

pytestmark = pytest.mark.gpu

MIB = 1 << 20


def moved(shapes, to, rows):
    """Bytes that the kernel reads and writes"""
    return (len(to) + len(set(rows))) * sum(planes * size for planes, size in shapes)


@pytest.mark.parametrize("offset", [0, 4, 2, 1])
def test_every_unit(gpu, offset):
    """Rows of multiples of 16, 4, 2 and 1 bytes at several alignments, in one call"""
    rng = np.random.default_rng(offset)
    shapes = [(2, 3 * MIB), (2, 3 * MIB - 12), (1, 2 * MIB + 6), (1, 2 * MIB + 4097)]
    src, dst = Buffers(gpu, rng, shapes, 9, offset), Buffers(gpu, rng, shapes, 12, offset)
    to, rows = [11, 0, 3, 7, 4, 10, 1, 9, 5, 2, 6], [2, 8, -1, 2, 0, 5, -1, 7, 2, 1, 8]
    assert moved(shapes, to, rows) >= 256 * MIB
    gpu.copy_rows([(dst.ptr(i), src.ptr(i), p, b) for i, (p, b) in enumerate(shapes)], 12, 9, to, rows)
    gpu.device_sync()
    for i in range(len(shapes)):
        assert np.array_equal(dst.now(i), host(src.of[i][0], dst.of[i][0], to, rows)), i
        assert np.array_equal(src.now(i), src.of[i][0])


class Rows:
    """Bytes [planes, rows, size] on the device, of which some rows are known"""

    def __init__(self, hip, planes, rows, size, known, seed):
        self.planes, self.rows, self.size = planes, rows, size
        self.device = hip.DeviceArray((planes * rows * size,), np.uint8)
        rng = np.random.default_rng(seed)
        self.known = {}
        for r in known:
            self.known[r] = rng.integers(0, 256, (planes, size), dtype=np.uint8)
            for p in range(planes):
                self.device.view((p * rows + r) * size, (size,)).upload(self.known[r][p])

    def now(self, r):
        return np.stack([self.device.view((p * self.rows + r) * self.size, (self.size,)).numpy() for p in range(self.planes)])


PLANES, ROWS, SIZE = 4, 512, 3 * MIB  # 6 GiB


def test_forks_behind_32_bits(gpu):
    """Inside one tensor: three rows go on in others, two are cleared; those beside them stay"""
    big = Rows(gpu, PLANES, ROWS, SIZE, [0, 1, 30, 255, 256, 257, 300, 301, 499, 500, 501, 509, 510, 511], 1)
    to = [511, 1, 300, 256, 509, 40, 41, 42, 43, 501, *range(100, 110)]
    rows = [0, 500, 500, 0, 255, 255, 500, -1, 0, -1, *[500] * 5, *[255] * 5]
    assert moved([(PLANES, SIZE)], to, rows) >= 256 * MIB and not set(to) & set(rows)
    gpu.copy_rows([(big.device, big.device, PLANES, SIZE)], ROWS, ROWS, to, rows)
    gpu.device_sync()
    for t, r in zip(to, rows):
        got = big.now(t)
        assert np.array_equal(got, big.known[r]) if r >= 0 else not got.any(), (t, r)
    for r in (0, 30, 255, 257, 301, 499, 500, 510):
        assert np.array_equal(big.now(r), big.known[r]), r
    big.device.free()


def test_gathers_between_tensors_behind_32_bits(gpu):
    rows = [510, 3, 400, 511, -1, 257, 510, 3, 400, 511, 257, 0, 0, 0, 510]
    to = [511, 0, 509, 2, 505, 300, 4, 5, 506, 507, 508, 301, 100, 101, 102]
    src = Rows(gpu, PLANES, ROWS, SIZE, sorted(set(r for r in rows if r >= 0)), 2)
    dst = Rows(gpu, PLANES, ROWS, SIZE, [1, 3, 299, 302, 504, 510], 3)
    assert moved([(PLANES, SIZE)], to, rows) >= 256 * MIB
    gpu.copy_rows([(dst.device, src.device, PLANES, SIZE)], ROWS, ROWS, to, rows)
    gpu.device_sync()
    for t, r in zip(to, rows):
        got = dst.now(t)
        assert np.array_equal(got, src.known[r]) if r >= 0 else not got.any(), (t, r)
    for r, data in dst.known.items():
        assert np.array_equal(dst.now(r), data), r
    for r, data in src.known.items():
        assert np.array_equal(src.now(r), data), r
    src.device.free()
    dst.device.free()
