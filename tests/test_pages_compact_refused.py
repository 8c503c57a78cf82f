"""A row one of whose drafts cannot move is left as it is by compact: its length, its pages and every byte; the rows beside
it are closed up."""
import numpy as np
import pytest
import torch

from tests.test_gpu_pages import KV, Both
from tests.test_pages_shared import _held
from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import pages_b200

pytestmark = pytest.mark.gpu


def _status():
    return _lib.read_status(torch.device("cuda", 0))


def _compact(s, path, count):
    """On the GPU alone: the tests say what it has to leave."""
    pages_b200.compact(s.pools, s.table, s.lens, s.refs, s.ints(path), s.ints(count))


# many columns: several CTAs a row, of which one marks it while others may not have begun
POOLS = {"narrow": KV, "wide": [(8, 8, 128, np.float16), (8, 8, 128, np.float16)]}


@pytest.mark.parametrize("pools", POOLS, ids=str)
def test_drafts_in_a_shared_page(pools):
    """Rows 0 and 1 share a full page that holds their drafts; row 2 is alone."""
    s = Both(3, 4, 10, 64, POOLS[pools], seed=41)
    s.reserve([64, 0, 100])
    s.fork([0], [1])
    before = [_held(s.m, r) for r in range(3)]
    _compact(s, [[0, 1, 3, -1], [0, 1, 2, -1], [1, 3, -1, -1]], [3, 3, 2])
    torch.cuda.synchronize()
    assert _status() == 4
    # row 0: draft 3 would move to draft 2's place: refused.  Row 1: nothing moves, the last draft goes
    assert s.lens.tolist() == [64, 63, 98] and s.refs.sum().item() == 4
    s.m.compact(np.array([[0, -1, -1, -1], [0, 1, 2, -1], [1, 3, -1, -1]]), [-1, 3, 2])
    s.same()
    for r, n in ((0, 64), (1, 63), (2, 96)):
        assert all(np.array_equal(a[:n], b[:n]) for a, b in zip(before[r], _held(s.m, r)))
    # the refusal can be repaired: a row of its own page by page (nothing of the drafts was lost)
    s.free([64, 0, 98])
    _compact(s, [[0, 1, 3, -1]] * 3, [3, -1, -1])
    s.m.compact(np.array([[0, 1, 3, -1]] * 3), [3, -1, -1])
    s.same()
    assert s.lens.tolist() == [63, 0, 98]


@pytest.mark.parametrize("pools", POOLS, ids=str)
@pytest.mark.parametrize("path", [[0, 3, 2, -1], [1, 1, 2, -1], [0, 2, 4, -1], [0, 2, -1, -1], [3, 2, 1, 0]], ids=str)
def test_a_path_that_does_not_ascend(path, pools):
    s = Both(4, 4, 16, 16, POOLS[pools], seed=43)
    s.reserve([33, 3, 20, 4])
    # row 1 has fewer positions than there are drafts; row 3 has nothing but drafts
    _compact(s, [path, [0, 1, 2, 3], [2, 3, -1, -1], [3, -1, -1, -1]], [3, 1, 2, 1])
    s.m.compact(np.array([[0, 0, 0, 0], [0, 0, 0, 0], [2, 3, -1, -1], [3, -1, -1, -1]]), [-1, -1, 2, 1])
    s.m.status = 2
    s.same()
    assert s.lens.tolist() == [33, 3, 18, 1]


def test_a_slot_without_a_page():
    s = Both(2, 4, 8, 16, KV, seed=45)
    s.reserve([32, 32])
    held = s.table[0, 1].item()
    s.table[0, 1] = -1
    before = [p.clone() for p in s.pools]
    _compact(s, [[0, 2, -1], [0, 1, 2]], [2, 3])          # position 31 to 30, in the slot without a page; nothing moves
    torch.cuda.synchronize()
    assert _status() == 2 and s.lens.tolist() == [32, 32] and all(torch.equal(a, b) for a, b in zip(before, s.pools))
    s.table[0, 1] = held
    s.same()


def test_captured_with_rows_that_are_refused():
    s = Both(3, 4, 12, 64, KV, seed=47)
    s.reserve([128, 0, 50])
    s.fork([0], [1])
    path, count = s.ints([[0, 2, 3, -1], [0, -1, -1, -1], [1, 2, -1, -1]]), s.ints([3, -1, 2])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        pages_b200.compact(s.pools, s.table, s.lens, s.refs, path, count)
    for _ in range(8):
        g.replay()
        s.m.compact(path.cpu().numpy(), [-1, -1, 2])
        s.m.status = 4
        s.same()
    assert s.lens.tolist() == [128, 128, 34]
