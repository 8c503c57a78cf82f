"""The page operators on the GPU through the C ABI against the model that does one row after another: tables, lengths,
counts and every byte of the pools have to be equal."""
import numpy as np
import pytest
import torch

from tests import _verify
from tests._pages_model import Model
from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import pages_b200

pytestmark = pytest.mark.gpu


class Both:
    """The same state on the GPU and in the model."""

    def __init__(self, rows, width, pages, page_size, pools, seed):
        self.rng = np.random.default_rng(seed)
        self.ps = page_size
        made = []
        for layers, heads, w, dtype in pools:
            a = self.rng.integers(0, 255, (layers, pages, heads, page_size, w * np.dtype(dtype).itemsize), dtype=np.uint8)
            made.append(a.view(dtype) if dtype == np.uint8 else (a.view(np.uint16) & 0x3BFF).view(np.float16))
        self.m = Model(np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32), page_size, made)
        self.table, self.lens, self.refs = (torch.from_numpy(x.copy()).cuda() for x in (self.m.table, self.m.lens, self.m.refs))
        self.pools = [torch.from_numpy(p.copy()).cuda() for p in made]

    def ints(self, x):
        return torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda()

    def same(self):
        torch.cuda.synchronize()
        assert np.array_equal(self.table.cpu().numpy(), self.m.table)
        assert np.array_equal(self.lens.cpu().numpy(), self.m.lens)
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs)
        for a, b in zip(self.pools, self.m.pools):
            assert np.array_equal(a.cpu().numpy(), b)
        assert _lib.read_status(torch.device("cuda", 0)) == self.m.status
        self.m.status = 0

    def reserve(self, extra):
        got = pages_b200.reserve(self.table, self.lens, self.refs, self.ints(extra), self.ps)
        want = self.m.reserve(extra)
        assert np.array_equal(got.cpu().numpy(), want)

    def free(self, keep):
        pages_b200.free(self.table, self.lens, self.refs, self.ints(keep), self.ps)
        self.m.free(keep)

    def fork(self, parents, children):
        pages_b200.fork(self.pools, self.table, self.lens, self.refs, self.ints(parents), self.ints(children))
        self.m.fork(parents, children)

    def compact(self, path, count):
        pages_b200.compact(self.pools, self.table, self.lens, self.refs, self.ints(path), self.ints(count))
        self.m.compact(np.asarray(path), count)

    def append(self, counts, pad=0):
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        src = [self.rng.standard_normal((int(cu[-1]) + pad, p.shape[2], p.shape[4])).astype(np.float16) for p in self.m.pools]
        dev = [torch.from_numpy(s).cuda() for s in src]
        pages_b200.append(dev[0], dev[1], self.pools[0][0], self.pools[1][0], self.table, self.ints(cu), self.lens)
        self.m.append(src, cu)

    def copy(self, src, dst):
        pages_b200.copy(self.pools, self.ints(src), self.ints(dst))
        self.m.copy(src, dst)


KV = [(1, 2, 128, np.float16), (1, 2, 128, np.float16)]


@pytest.mark.parametrize("page_size,rows,pages,pools", [
    (64, 5, 40, KV), (16, 70, 300, [(2, 3, 8, np.float16)]), (1, 9, 50, [(1, 1, 16, np.uint8)]), (7, 33, 100, [(3, 1, 576, np.float16), (3, 1, 128, np.uint8)]),
    (256, 4, 30, [(1, 8, 128, np.float16)])], ids=lambda x: str(x))
def test_random_sequences_of_operators(page_size, rows, pages, pools):
    s = Both(rows, 12, pages, page_size, pools, seed=rows)
    rng = np.random.default_rng(7)
    for step in range(25):
        s.reserve(rng.integers(0, 3 * page_size + 1, rows))
        s.same()
        kd = int(min(rng.integers(1, 9), max(1, s.m.lens.min())))
        if s.m.lens.min() >= kd and step % 2:
            path = np.full((rows, kd), -1)
            # a row whose last positions lie in a page that it shares keeps all of them (path = identity moves nothing)
            count = rng.integers(0, kd + 1, rows)
            for r in range(rows):
                lo = max(0, (int(s.m.lens[r]) - kd) // page_size)
                shared = any(s.m.refs[s.m.table[r, i]] > 1 for i in range(lo, -(-int(s.m.lens[r]) // page_size)))
                path[r, :count[r]] = np.arange(count[r]) if shared else np.sort(rng.permutation(kd)[:count[r]])
            count[rng.random(rows) < 0.2] = -1
            s.compact(path, count)
            s.same()
        empty = rng.permutation(rows)[:rows // 3]
        keep = np.where(np.isin(np.arange(rows), empty), 0, rng.integers(0, 12 * page_size, rows))
        s.free(keep)
        s.same()
        if len(empty):
            s.fork(rng.integers(-1, rows, len(empty)), empty)
            s.same()
        free = np.nonzero(s.m.refs == 0)[0]
        if len(free) > 1:
            s.copy(rng.permutation(np.nonzero(s.m.refs >= 0)[0][:1]), free[-1:])
            s.same()
    s.free(np.zeros(rows))
    s.same()
    assert (s.m.refs == 0).all()


def test_append_then_what_the_pages_hold():
    s = Both(6, 8, 60, 64, KV, seed=1)
    for counts in ([1, 130, 0, 64, 63, 200], [5, 0, 7, 1, 1, 60]):
        s.reserve(counts)
        s.append(counts, pad=9)                 # rows behind the last sequence are not written anywhere
        s.same()


def test_append_takes_views_and_pools_of_different_widths():
    """dsa keeps latent rows and index keys in pools of 576 and 128, (pages, page_size, width)."""
    dev = "cuda"
    kv, ik = torch.zeros(9, 16, 576, dtype=torch.bfloat16, device=dev), torch.zeros(9, 16, 128, dtype=torch.uint8, device=dev)
    table = torch.tensor([[4, 2, -1], [7, -1, -1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([20, 3], dtype=torch.int32, device=dev)
    rows = torch.randn(23, 1, 600, device=dev).bfloat16()[:, :, 8:584]
    keys = torch.randint(0, 255, (23, 4, 128), dtype=torch.uint8, device=dev)[:, 2:3]
    pages_b200.append(rows, keys, kv, ik, table, torch.tensor([0, 20, 23], dtype=torch.int32, device=dev), lens, check=True)
    assert torch.equal(kv[4], rows[:16, 0]) and torch.equal(kv[2, :4], rows[16:20, 0]) and torch.equal(kv[7, :3], rows[20:, 0])
    assert torch.equal(ik[4], keys[:16, 0]) and torch.equal(ik[2, :4], keys[16:20, 0]) and torch.equal(ik[7, :3], keys[20:, 0])
    assert (kv[2, 4:] == 0).all() and (kv[7, 3:] == 0).all() and (kv[[0, 1, 3, 5, 6, 8]] == 0).all()


def test_append_without_a_page_writes_nothing():
    s = Both(2, 2, 8, 64, KV, seed=2)
    s.reserve([70, 3])
    s.table[0, 1] = -1                           # a slot without a page, and one outside the pool
    s.table[1, 0] = 8
    before = [p.clone() for p in s.pools]
    src = torch.ones(10, 2, 128, dtype=torch.float16, device="cuda")
    pages_b200.append(src, src, s.pools[0][0], s.pools[1][0], s.table, s.ints([0, 6, 9]), s.lens)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, s.pools)) and _lib.read_status(torch.device("cuda", 0)) == 2
    # a row that counts fewer positions than it has new tokens
    pages_b200.append(src, src, s.pools[0][0], s.pools[1][0], s.table, s.ints([0, 0, 9]), s.lens)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, s.pools)) and _lib.read_status(torch.device("cuda", 0)) == 2


def test_pages_run_out():
    s = Both(6, 10, 12, 64, [(1, 1, 8, np.float16)], seed=3)
    s.reserve([64 * 5, 0, 64 * 4, 64 * 6, 64, 10 ** 6])     # 12 pages: rows 0 and 2 get theirs, 3 and 4 do not, 5 is too long
    assert s.m.status == 4
    s.same()
    s.reserve([1, -3, 0, 64 * 2, 64, 1])
    s.same()
    s.free([0, 0, 10, 0, -1, 0])
    s.same()


def test_fork_when_pages_run_out_and_children_that_are_refused():
    s = Both(9, 4, 10, 64, [(2, 2, 16, np.float16)], seed=4)
    s.reserve([100, 64, 130, 0, 0, 0, 0, 0, 0])             # 2 + 1 + 3 pages: four are left
    s.fork([0, 1, 2, 0, 2, -1, 30, 1, 8], [3, 4, 5, 5, 0, 6, 6, 77, 7])   # 5 twice, 0 not empty, a parent and a child out of range
    assert s.m.status == 2
    s.same()
    s.fork([2, 2, 1, 2], [6, 7, 8, 1])                       # two pages are left, and row 1 is not empty
    s.same()
    s.free([100, 64, 130, 0, 0, 0, 0, 0, 0])
    s.same()
    assert s.m.refs.sum() == 6


def test_a_row_forked_in_the_call_that_forks_from_it_is_still_empty():
    s = Both(3, 4, 10, 64, [(1, 1, 8, np.float16)], seed=5)
    s.reserve([100, 0, 0])
    s.fork([0, 1], [1, 2])
    s.same()
    assert s.m.lens.tolist() == [100, 100, 0]


def test_compact_does_not_write_into_a_page_that_others_share():
    s = Both(2, 4, 10, 64, [(1, 1, 8, np.float16)], seed=6)
    s.reserve([64, 0])
    s.fork([0], [1])                                          # the full page is shared
    before = s.pools[0].clone()
    pages_b200.compact(s.pools, s.table, s.lens, s.refs, s.ints([[0, 3], [0, 1]]), s.ints([2, 2]))
    pages_b200.compact(s.pools, s.table, s.lens, s.refs, s.ints([[0, 1, 3, -1], [0, 1, 2, 3]]), s.ints([3, 4]))
    torch.cuda.synchronize()
    assert torch.equal(before, s.pools[0]) and _lib.read_status(torch.device("cuda", 0)) == 2 | 4
    assert s.lens.tolist() == [63, 64] and int(s.refs.sum()) == 2


def test_compact_longest_path_over_several_pages():
    s = Both(3, 12, 40, 16, [(2, 3, 128, np.float16), (1, 1, 16, np.uint8)], seed=8)
    s.reserve([140, 128, 131])
    path = np.full((3, 128), -1)
    path[0], path[1, :64], path[2, :1] = np.arange(128), np.arange(64) * 2, 0
    s.compact(path, [128, 64, 1])
    s.same()


@pytest.mark.parametrize("n", [1, 3, 200])
def test_copy_of_many_pages_over_all_layers(n):
    s = Both(1, 1, 2 * n + 5, 64, [(3, 8, 128, np.float16), (1, 1, 40, np.float16)], seed=n)
    ids = s.rng.permutation(2 * n + 5)
    s.copy(ids[:n], ids[n:2 * n])
    s.same()
    pages_b200.copy(s.pools, s.ints([0, -1, 10 ** 6, 2]), s.ints([-1, 0, 1, 2]))
    torch.cuda.synchronize()
    assert _lib.read_status(torch.device("cuda", 0)) == 2
    s.same()


def test_more_rows_and_pages_than_a_block_has_threads():
    s = Both(2500, 3, 9000, 16, [(1, 1, 8, np.float16)], seed=9)
    rng = np.random.default_rng(1)
    s.reserve(rng.integers(0, 40, 2500))
    s.same()
    s.free(np.where(rng.random(2500) < 0.5, 0, 100))
    s.same()
    empty = np.nonzero(s.m.lens == 0)[0]
    s.fork(rng.integers(0, 2500, len(empty)), empty)
    s.same()
    s.reserve(rng.integers(0, 5, 2500))
    s.same()
    _verify.assert_clean_status()


def test_captured_and_replayed():
    """A graph of a whole step, replayed while the state changes under it."""
    s = Both(4, 8, 40, 64, KV, seed=10)
    s.reserve([60, 100, 3, 130])
    extra, cu = s.ints([3, 3, 3, 3]), s.ints([0, 3, 6, 9, 12])
    src = torch.randn(12, 2, 128, device="cuda").half()
    path, count = s.ints([[0, 2, -1], [0, -1, -1], [0, 1, 2], [0, 1, -1]]), s.ints([2, 1, 3, 2])

    def step():
        pages_b200.reserve(s.table, s.lens, s.refs, extra, 64)
        pages_b200.append(src, src, s.pools[0][0], s.pools[1][0], s.table, cu, s.lens)
        pages_b200.compact(s.pools, s.table, s.lens, s.refs, path, count)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    host = src.cpu().numpy()
    for _ in range(30):
        g.replay()
        s.m.reserve([3] * 4)
        s.m.append([host, host], [0, 3, 6, 9, 12])
        s.m.compact(path.cpu().numpy(), [2, 1, 3, 2])
        s.same()


def test_on_another_stream():
    s = Both(3, 6, 30, 64, KV, seed=11)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        s.reserve([10, 200, 64])
        s.append([10, 200, 64])
        s.free([0, 100, 64])
    st.synchronize()
    s.same()


def test_lengths_beyond_32_bits_of_bytes():
    """A pool of over 4 GiB: pages at its end."""
    pages = 33000
    pool = torch.zeros(pages, 8, 64, 128, dtype=torch.float16, device="cuda")       # 4.3 GB
    pool[5] = torch.randn(8, 64, 128, device="cuda").half()
    ids = torch.tensor([5], dtype=torch.int32, device="cuda")
    pages_b200.copy([pool], ids, torch.tensor([pages - 1], dtype=torch.int32, device="cuda"), check=True)
    assert torch.equal(pool[5], pool[pages - 1])
    table = torch.tensor([[pages - 2, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    src = torch.randn(40, 8, 128, device="cuda").half()
    pages_b200.append(src, src, pool, pool, table, torch.tensor([0, 40], dtype=torch.int32, device="cuda"), lens, check=True)
    assert torch.equal(pool[pages - 2, :, :40], src.transpose(0, 1)) and (pool[pages - 2, :, 40:] == 0).all()
