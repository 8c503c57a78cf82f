"""The compiled form of the kernel modules' ordinary calls: it builds, loads without a GPU and hands every call that is not
ordinary back; on the GPU it takes the ordinary ones and gives what the modules' own way gives."""
import numpy as np
import pytest
import torch

from verified_metal_kernels_b200 import build
from verified_metal_kernels_b200.kernels import _common, accept_b200, pages_b200, prompt_b200


@pytest.fixture(scope="module")
def calls():
    build.build()
    build.build_calls()
    return _common.calls()


def test_build_is_keyed_by_content(calls):
    import os
    before = os.stat(build.CALLS_LIB).st_mtime_ns
    os.utime(build.CALLS_SRC)
    assert build.build_calls() == build.CALLS_LIB and os.stat(build.CALLS_LIB).st_mtime_ns == before


def test_kernels_are_reached_by_name():
    from verified_metal_kernels_b200 import load_kernel
    from verified_metal_kernels_b200.kernels import decode_b200
    assert load_kernel("prompt") is prompt_b200.kernel and load_kernel("accept") is accept_b200.kernel
    assert load_kernel("decode") is decode_b200.kernel
    with pytest.raises(KeyError):
        load_kernel("pages")                   # several functions: kernels.pages_b200


def test_calls_that_are_not_ordinary_are_handed_back(calls):
    t, i = torch.zeros(4, 2, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    table, pool = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, 2, 64, 128, dtype=torch.float16)
    for args in ((t, t, t, i, None, True), (None,) * 6, (t, t, t), (1, "x", t, i, i, True)):
        assert calls.prompt(*args) is None
    assert calls.prompt_paged(t, pool, pool, table, i, i, True) is None
    assert calls.accept(t, table, table, t, None) is None
    assert calls.reserve(table, i, i, i, 64) is None and calls.free(table, i, i, i, 64) is None
    assert calls.append(t, t, pool, pool, table, i, i) is None and calls.fork([pool], table, i, i, i, i) is None
    assert calls.compact([pool], table, i, i, table, i) is None and calls.copy([pool], i, i) is None and calls.copy(pool, i, i) is None
    with pytest.raises(ValueError):
        calls.init(1, 2)
    with pytest.raises(ValueError):
        calls.init(*[0] * 11)
    with pytest.raises(TypeError):
        calls.set_status("a", 1)


@pytest.mark.gpu
def test_ordinary_calls_are_taken(calls):
    g = torch.Generator(device="cuda").manual_seed(0)
    half = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q, k = half(60, 8, 128), half(60, 2, 128)
    cu = ints([0, 25, 60])
    want = prompt_b200.kernel(q, k, k, cu, check=True)                 # the module's own way
    assert torch.equal(calls.prompt(q, k, k, cu, None, True), want) and torch.equal(calls.prompt(q, k, k, cu, cu, 1), want)
    pool = half(3, 2, 64, 128)
    table, lens = ints([[0], [2]]), ints([30, 40])
    assert torch.equal(calls.prompt_paged(q, pool, pool, table, cu, lens, True), prompt_b200.kernel_paged(q, pool, pool, table, cu, lens, check=True))
    p = torch.softmax(torch.randn(3, 40, 50, generator=g, device="cuda"), -1)
    tok = torch.randint(0, 50, (3, 40), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(3, 40, generator=g, device="cuda")
    bits = torch.from_numpy(np.array([[[(1 << min(i + 1, 32)) - 1, (1 << max(i - 31, 0)) - 1] for i in range(40)]] * 3, dtype=np.uint32).view(np.int32)).cuda()
    for draft in (None, p.flip(0).contiguous()):
        for a, b in zip(calls.accept(p, tok, bits, u, draft), accept_b200.kernel(p, tok, bits, u, draft, check=True)):
            assert torch.equal(a, b)
    both = []
    for way in (False, True):                                          # the same page operators, by either way
        pools = [pool.clone(), torch.zeros(2, 3, 1, 64, 8, device="cuda")]
        table, lens, refs = torch.full((4, 2), -1, dtype=torch.int32, device="cuda"), ints([0] * 4), ints([0] * 3)
        one = [pools[0]]
        if way:
            assert calls.reserve(table, lens, refs, ints([70, 3, 0, 0]), 64).tolist() == [1, 1, 1, 1]
            assert calls.append(half(73, 2, 128).zero_(), half(73, 2, 128).zero_(), pools[0], pools[0], table, ints([0, 70, 73, 73, 73]), lens)
            assert calls.compact(pools, table, lens, refs, ints([[0, 2, -1]] * 4), ints([2, 1, -1, -1]))
            assert calls.fork(tuple(one), table, lens, refs, ints([1]), ints([2]))
            assert calls.copy(one, ints([0]), ints([1]))
            assert calls.free(table, lens, refs, ints([64, 0, 5, 0]), 64)
        else:
            pages_b200.reserve(table, lens, refs, ints([70, 3, 0, 0]), 64, check=True)
            pages_b200.append(half(73, 2, 128).zero_(), half(73, 2, 128).zero_(), pools[0], pools[0], table, ints([0, 70, 73, 73, 73]), lens, check=True)
            pages_b200.compact(pools, table, lens, refs, ints([[0, 2, -1]] * 4), ints([2, 1, -1, -1]), check=True)
            with pytest.raises(Exception):
                pages_b200.fork(one, table, lens, refs, ints([1]), ints([2]), check=True)      # no page is left: reported
            pages_b200.copy(one, ints([0]), ints([1]), check=True)
            pages_b200.free(table, lens, refs, ints([64, 0, 5, 0]), 64, check=True)
        both.append((*pools, table, lens, refs))
    from verified_metal_kernels_b200 import _lib
    assert _lib.read_status(torch.device("cuda", 0)) == 4             # the fork by the compiled way
    assert all(torch.equal(a, b) for a, b in zip(*both))


@pytest.mark.gpu
def test_refusals_come_from_the_module(calls):
    """A call that the entry point refuses, or whose tensors are wrong, is handed back and raises as ever."""
    q, k = torch.zeros(4, 6, 128, dtype=torch.float16, device="cuda"), torch.zeros(4, 4, 128, dtype=torch.float16, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    from verified_metal_kernels_b200._lib import VmkError
    assert calls.prompt(q, k, k, cu, None, True) is None
    with pytest.raises(VmkError):
        prompt_b200.kernel(q, k, k, cu)
    with pytest.raises(TypeError):
        prompt_b200.kernel(q, k, k, cu.long())
    p = torch.zeros(1, 140, 5, device="cuda")
    i = torch.zeros(1, 140, dtype=torch.int32, device="cuda")
    with pytest.raises(VmkError):
        accept_b200.kernel(p, i, i, torch.zeros(1, 140, device="cuda"))
    with pytest.raises(ValueError):
        pages_b200.free(cu[None].expand(3, 2), cu, cu, cu, 64)
