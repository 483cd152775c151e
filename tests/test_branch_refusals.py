"""What draw_tokens and copy_rows refuse, and the order of copy_rows' moves (no GPU: the calls are refused before anything is launched)."""
import pytest

from test_host_api import _run


@pytest.fixture(scope="module")
def hip():
    from rwkv_lightning_cuda_amd import hip
    hip.load()
    return hip


def test_moves_in_order():
    out = _run("copy_rows_cpu_test")
    assert "ok   any_moves_keep_what_the_rows_held" in out and "ok   the_largest_call_fits_whatever_the_cycles" in out


def test_host_side_of_branches():
    out = _run("branch_cpu_test")
    assert "ok   numbers_depend_on_their_place_alone" in out and "ok   backends_with_slices_move_runs_of_rows" in out


A = 1 << 20  # addresses that are never followed


class Workspace:
    def __init__(self, nbytes, ptr=A):
        self.nbytes, self.ptr = nbytes, ptr

    def __int__(self):
        return self.ptr


def draw(hip, rows=2, V=1000, logits=A, uniform=A, token=A, workspace=None, **kw):
    hip.draw_tokens(rows, V, logits, uniform, token, workspace, **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(rows=0), "rows must be positive"),
    (dict(rows=-1), "rows must be positive"),
    (dict(logit_rows=0), "rows must be positive"),
    (dict(V=0), "V must lie in"),
    (dict(V=1048577), "V must lie in"),
    (dict(io=2), "unknown element type"),
    (dict(logits=None), "NULL logits"),
    (dict(uniform=None), "NULL logits, uniform or token"),
    (dict(token=None), "NULL logits, uniform or token"),
    (dict(ld=999), "lie 999 apart"),
    (dict(ld=-1000), "lie -1000 apart"),
    (dict(logit_rows=1), "without their sources"),
    (dict(logits=A + 2), "misaligned logits"),
    (dict(logits=A + 1, io=0), "misaligned logits"),
    (dict(temperature=A + 2), "aligned to 4 bytes"),
    (dict(logprob=A + 1), "aligned to 4 bytes"),
    (dict(penalties_out=A), "without any"),
    (dict(decay=A), "without any"),
    (dict(penalties=A, decay=A), "without penalties_out"),
    (dict(), "workspace of"),
    (dict(workspace=Workspace(100)), "workspace of"),
    (dict(workspace=Workspace(1 << 30, A + 8)), "workspace of"),
])
def test_draws_that_are_refused(hip, kw, message):
    with pytest.raises(hip.RwkvHipError, match=message):
        draw(hip, **kw)


def test_draw_workspaces(hip):
    for V in (1, 64, 65, 50277, 65536, 1048576):
        sizes = [hip.draw_tokens_workspace(rows, V) for rows in range(1, 200)]
        assert sizes == sorted(sizes) and all(s >= rows * (-(-V // 64)) * 12 and s % 16 == 0 for rows, s in enumerate(sizes, 1))
    for rows, V in ((0, 10), (1, 0), (1, 1048577)):
        with pytest.raises(hip.RwkvHipError, match="bad arguments"):
            hip.draw_tokens_workspace(rows, V)


T = (A, 1 << 30, 2, 64)  # destination, source, planes, bytes of a row


@pytest.mark.parametrize("tensors,dst_rows,src_rows,to,rows,message", [
    ([], 4, 4, [0], [1], "1 .. 8 tensors"),
    ([T] * 9, 4, 4, [0], [1], "1 .. 8 tensors"),
    ([T], 0, 4, [0], [1], "rows, got"),
    ([T], 4, 65535, [0], [1], "rows, got"),
    ([T], 600, 600, list(range(513)), [0] * 513, "up to 512 moves"),
    ([(0, A, 2, 64)], 4, 4, [0], [1], "is NULL"),
    ([(A, None, 2, 64)], 4, 4, [0], [1], "is NULL"),
    ([(A, 1 << 30, 0, 64)], 4, 4, [0], [1], "0 planes"),
    ([(A, 1 << 30, 2, -64)], 4, 4, [0], [1], "rows of -64 bytes"),
    ([(A, 1 << 60, 1 << 40, 1 << 30)], 4, 4, [0], [1], "larger than any memory"),
    ([(A, 1 << 60, 1, 1 << 62)], 4, 4, [0], [1], "larger than any memory"),
    ([T], 4, 4, [4], [1], "goes to row 4 of 4"),
    ([T], 4, 4, [-1], [1], "goes to row -1"),
    ([T], 4, 4, [0], [4], "comes from row 4 of 4"),
    ([T], 4, 4, [0], [-2], "comes from row -2"),
    ([T], 4, 4, [2, 2], [0, 1], "two moves go to row 2"),
    ([(A, A, 2, 64)], 4, 5, [0], [1], "in place, but 4 and 5 rows"),
    ([(A, A, 2, 64), T], 4, 4, [0], [1], "in place beside"),
    ([(A, A + 64, 2, 64)], 4, 4, [0], [1], "overlaps source"),
    ([(A, 1 << 30, 2, 64), (A + 128, 1 << 31, 2, 64)], 4, 4, [0], [1], "destinations 0 and 1 overlap"),
    ([(A, 1 << 30, 2, 64), (1 << 31, A + 256, 2, 64)], 4, 4, [0], [1], "destination 0 overlaps source 1"),
    ([(A, A, 2, 64), (A + 256, A + 256, 2, 64)], 4, 4, [0], [1], "destinations 0 and 1 overlap"),
    ([(A, 1 << 45, 256, (1 << 27) + 1)], 4, 4, [0], [1], "too large for one call"),
    ([(A, A, 256, (1 << 27) + 1)], 4, 4, [0, 1], [1, 0], "too large for one call"),
])
def test_copies_that_are_refused(hip, tensors, dst_rows, src_rows, to, rows, message):
    with pytest.raises(hip.RwkvHipError, match=message):
        hip.copy_rows(tensors, dst_rows, src_rows, to, rows)


def test_lists_of_two_lengths(hip):
    with pytest.raises(ValueError):
        hip.copy_rows([T], 4, 4, [0, 1], [1])


def test_nothing_to_do_needs_no_device(hip):
    hip.copy_rows([T], 4, 4, [], [])
    hip.copy_rows([(A, A, 2, 64)], 4, 4, [1, 2], [1, 2])
