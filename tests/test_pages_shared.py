"""What rows that share pages do to one another: nothing.  The statement of the page operators without a GPU, then the
operators against it, and against what every other row held before."""
import numpy as np
import pytest
import torch

from tests._pages_model import Model
from tests.test_gpu_pages import KV, Both
from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import _common, pages_b200


def _model(rows, width, pages, page_size):
    pool = np.zeros((1, pages, 1, page_size, 1), np.int64)
    return Model(np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32), page_size, [pool])


def _held(m, r):
    """What row r holds, position by position, in every pool."""
    return [np.stack([p[:, m.table[r, i // m.ps], :, i % m.ps] for i in range(int(m.lens[r]))]) if m.lens[r] else None for p in m.pools]


def test_the_statement_does_not_grow_into_a_shared_page():
    m = _model(3, 3, 6, 4)
    assert m.reserve([8, 0, 0]).tolist() == [1, 1, 1]
    m.append([np.arange(8).reshape(8, 1, 1)], [0, 8])
    m.fork([0], [1])
    m.free([8, 6, 0])
    assert m.reserve([1, 1, 0]).tolist() == [1, 0, 1] and m.status == 4 and m.lens.tolist() == [9, 6, 0]
    m.fork([1], [2])                            # a page of its own for the cut row: now it grows
    m.free([9, 0, 6])
    assert m.reserve([0, 0, 1]).tolist() == [1, 1, 1]
    m.append([np.array([[[70]]])], [0, 0, 0, 1])
    assert _held(m, 0)[0][:8].ravel().tolist() == list(range(8)) and _held(m, 2)[0].ravel().tolist() == [0, 1, 2, 3, 4, 5, 70]


def _forked(page_size=64, seed=21):
    """Row 0 of two full pages, row 1 forked from it (both pages shared), rows 2 and 3 empty."""
    s = Both(4, 6, 30, page_size, KV, seed=seed)
    s.reserve([2 * page_size, 0, 0, 0])
    s.append([2 * page_size, 0, 0, 0])
    s.fork([0], [1])
    s.same()
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("cut", [0, 1], ids=["parent", "child"])
def test_a_row_cut_inside_a_shared_page_is_not_granted_more(cut, page_size):
    s = _forked(page_size)
    keep = [2 * page_size, 2 * page_size, 0, 0]
    keep[cut] = 2 * page_size - 5
    s.free(keep)
    other = _held(s.m, 1 - cut)
    s.reserve([3, 3, 0, 0])                     # the row that was not cut gets a page, the other nothing
    assert s.m.status == 4 and s.m.lens[cut] == keep[cut] and s.m.lens[1 - cut] == 2 * page_size + 3
    s.same()
    counts = [3, 3]
    counts[cut] = 0
    s.append(counts)
    s.same()
    for a, b in zip(other, _held(s.m, 1 - cut)):
        assert np.array_equal(a, b[:2 * page_size])
    # forked into an empty row it has a page of its own, and goes on
    s.fork([cut], [2])
    keep = s.m.lens.copy()
    keep[cut] = 0
    s.free(keep)
    s.reserve([0, 0, 9, 0])
    s.append([0, 0, 9])
    s.same()
    for a, b in zip(other, _held(s.m, 1 - cut)):
        assert np.array_equal(a, b[:2 * page_size])


@pytest.mark.gpu
def test_a_page_that_is_shared_no_more_is_grown_into():
    s = _forked()
    s.free([100, 128, 0, 0])
    s.free([100, 0, 0, 0])
    s.reserve([40, 0, 0, 0])
    s.append([40])
    s.same()
    assert s.m.lens[0] == 140


@pytest.mark.gpu
def test_both_rows_cut_in_the_same_page_and_a_row_that_asks_for_nothing():
    s = _forked()
    s.free([70, 127, 0, 0])
    s.reserve([1, 64, 5, 0])
    s.same()
    assert s.m.lens.tolist() == [70, 127, 5, 0]
    s.reserve([0, 0, 0, 0])                     # no growth is always granted
    s.same()


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False], ids=["compiled", "module"])
def test_append_with_the_counts_writes_no_shared_page(compiled):
    """A row forked between its reserve and its append: the positions that are still to be written are both rows'."""
    s = Both(3, 4, 12, 64, KV, seed=23)
    s.reserve([60, 10, 0])
    s.append([60, 10])
    s.reserve([68, 5, 0])                        # to 128: two full pages, which the fork shares
    s.fork([0], [2])
    s.same()
    before = [p.clone() for p in s.pools]
    src = torch.ones(73, 2, 128, dtype=torch.float16, device="cuda")
    args = (src, src, s.pools[0][0], s.pools[1][0], s.table, s.ints([0, 68, 73]), s.lens)
    if compiled:
        assert _common.calls().append(*args, None, s.refs) is True and _common.calls().append(*args, None, s.refs[:-1].contiguous()) is None
    else:
        with pytest.raises(_lib.VmkDeviceStatusError) as e:
            pages_b200.append(*args, check=True, refs=s.refs)
        assert e.value.status == 4
    host = src[68:].cpu().numpy()
    s.m.append([host, host], [0, 0, 5])          # row 1's, and nothing else
    s.m.status = 4 if compiled else 0
    s.same()
    assert not torch.equal(before[0], s.pools[0])


def test_append_refuses_wrong_counts(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    i32 = torch.int32
    table, lens, cu = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(2, dtype=i32)
    pool, k = torch.zeros(8, 2, 16, 8, dtype=torch.float16), torch.zeros(5, 2, 8, dtype=torch.float16)
    for err, refs in ((ValueError, torch.zeros(7, dtype=i32)), (TypeError, torch.zeros(8)), (TypeError, [0] * 8)):
        with pytest.raises(err):
            pages_b200.append(k, k, pool, pool, table, cu, lens, refs=refs)
