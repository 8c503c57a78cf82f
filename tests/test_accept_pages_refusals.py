"""What the acceptance of drafts and the page operators refuse, without a GPU, and their statements against small cases
worked by hand."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import ref64
from tests._pages_model import Model
from verified_metal_kernels_b200 import _lib, build
from verified_metal_kernels_b200.kernels import accept_b200, pages_b200
from verified_metal_kernels_b200.ops import accept as op


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _named(fn, names, base):
    return lambda **kw: fn(*[{**base, **kw}[n] for n in names])


def test_accept_refuses_before_any_launch(lib):
    names = ("p", "q", "tokens", "bits", "words", "u", "path", "count", "next", "B", "kd", "V", "dtype", "status", "stream")
    call = _named(lib.vmk_accept, names, dict(p=256, q=256, tokens=256, bits=256, words=1, u=256, path=256, count=256, next=256, B=2, kd=4, V=100,
                                              dtype=0, status=None, stream=None))
    for n in ("p", "tokens", "bits", "u", "path", "count", "next"):
        assert call(**{n: None}) == -1 and call(**{n: 258}) == -1
    assert call(q=258) == -1 and call(status=2) == -1 and call(p=257, dtype=1) == -1 and call(q=257, dtype=2) == -1
    assert call(B=-1) == -1 and call(kd=0) == -1 and call(V=0) == -1 and call(words=0) == -1 and call(dtype=3) == -1 and call(dtype=-1) == -1
    assert call(kd=33) == -2 and call(kd=129, words=5) == -2
    assert call(V=2 ** 31 - 1) == -6 and call(B=2 ** 31 - 1) == -6
    assert call(B=0, p=None) == 0


def _pool(*d):
    flat = [x for p in d for x in p]
    return (ctypes.c_int64 * len(flat))(*flat)


GOOD = (256, 1, 8, 256)


def test_page_operators_refuse_before_any_launch(lib):
    free = _named(lib.vmk_pages_free, ("t", "R", "T", "lens", "refs", "pages", "ps", "keep", "status", "stream"),
                  dict(t=256, R=2, T=4, lens=256, refs=256, pages=8, ps=64, keep=256, status=None, stream=None))
    for kw in (dict(t=None), dict(lens=257), dict(refs=264), dict(keep=None), dict(R=-1), dict(T=0), dict(pages=0), dict(ps=0), dict(status=1)):
        assert free(**kw) == -1, kw
    assert free(T=(1 << 20) + 1) == -6 and free(R=0, t=None) == 0
    ws = lib.vmk_pages_workspace_bytes(2, 3, 8)
    reserve = _named(lib.vmk_pages_reserve, ("t", "R", "T", "lens", "refs", "pages", "ps", "extra", "granted", "ws", "wsb", "status", "stream"),
                     dict(t=256, R=2, T=4, lens=256, refs=256, pages=8, ps=64, extra=256, granted=None, ws=256, wsb=ws, status=None, stream=None))
    for kw in (dict(extra=None), dict(granted=2), dict(ws=None), dict(ws=264), dict(refs=None)):
        assert reserve(**kw) == -1, kw
    assert reserve(wsb=8) == -3
    fork = _named(lib.vmk_pages_fork, ("pools", "n", "t", "R", "T", "lens", "refs", "pages", "ps", "par", "ch", "F", "ws", "wsb", "status", "stream"),
                  dict(pools=_pool(GOOD), n=1, t=256, R=2, T=4, lens=256, refs=256, pages=8, ps=64, par=256, ch=256, F=3, ws=256, wsb=ws, status=None, stream=None))
    for kw in (dict(pools=None), dict(n=0), dict(par=None), dict(ch=258), dict(F=-1), dict(ws=None), dict(pools=_pool((264, 1, 8, 256))), dict(pools=_pool((0, 1, 8, 256))),
               dict(pools=_pool((256, 0, 8, 256))), dict(pools=_pool((256, 1, 0, 256))), dict(pools=_pool((256, 1, 8, 24)))):
        assert fork(**kw) == -1, kw
    assert fork(n=9, pools=_pool(*[GOOD] * 9)) == -2 and fork(wsb=16) == -3 and fork(F=0, par=None) == 0
    assert fork(pools=_pool((256, 1, 8, 1 << 24)), ps=1 << 20) == -6
    compact = _named(lib.vmk_pages_compact, ("pools", "n", "t", "R", "T", "lens", "refs", "pages", "ps", "path", "count", "kd", "status", "stream"),
                     dict(pools=_pool(GOOD), n=1, t=256, R=2, T=4, lens=256, refs=256, pages=8, ps=64, path=256, count=256, kd=4, status=None, stream=None))
    assert compact(path=None) == -1 and compact(count=None) == -1 and compact(kd=0) == -1 and compact(kd=129) == -2
    copy = _named(lib.vmk_pages_copy, ("pools", "n", "pages", "ps", "src", "dst", "m", "status", "stream"),
                  dict(pools=_pool(GOOD), n=1, pages=8, ps=64, src=256, dst=256, m=3, status=None, stream=None))
    assert copy(src=None) == -1 and copy(dst=257) == -1 and copy(m=-1) == -1 and copy(m=0, src=None) == 0
    src = (ctypes.c_int64 * 6)(256, 2048, 256, 256, 2048, 256)
    append = _named(lib.vmk_pages_append, ("pools", "src", "pages", "ps", "t", "T", "cu", "lens", "S", "tokens", "status", "stream"),
                    dict(pools=_pool(GOOD, GOOD), src=src, pages=8, ps=64, t=256, T=4, cu=256, lens=256, S=2, tokens=9, status=None, stream=None))
    for kw in (dict(src=None), dict(t=None), dict(cu=None), dict(lens=None), dict(S=-1), dict(tokens=-1), dict(T=0),
               dict(src=(ctypes.c_int64 * 6)(264, 2048, 256, 256, 2048, 256)), dict(src=(ctypes.c_int64 * 6)(256, 2048, 256, 256, -16, 256)),
               dict(src=(ctypes.c_int64 * 6)(256, 2048, 250, 256, 2048, 256))):
        assert append(**kw) == -1, kw
    assert append(pools=_pool((256, 2, 8, 256), GOOD)) == -2 and append(tokens=0) == 0


def test_modules_refuse_by_their_checks(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    i32 = torch.int32
    p, tok, u = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=i32), torch.zeros(2, 3)
    good = dict(target_probs=p, tokens=tok, bits=tok, u=u, draft_probs=p)
    for err, kw in ((TypeError, dict(target_probs=p.double())), (TypeError, dict(draft_probs=p.half())), (ValueError, dict(target_probs=p[0])),
                    (ValueError, dict(tokens=tok[:1])), (TypeError, dict(tokens=tok.long())), (TypeError, dict(bits=tok.long())), (ValueError, dict(bits=tok[0])),
                    (ValueError, dict(u=u[:, :2])), (TypeError, dict(u=u.double())), (ValueError, dict(draft_probs=p[:1])),
                    (ValueError, dict(target_probs=p.transpose(0, 1).contiguous().transpose(0, 1)))):
        with pytest.raises(err):
            accept_b200.kernel(**{**good, **kw})
    table, lens, refs = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(8, dtype=i32)
    pool = torch.zeros(8, 2, 16, 8, dtype=torch.float16)
    two = torch.zeros(2, dtype=i32)
    k = torch.zeros(5, 2, 8, dtype=torch.float16)
    cu = torch.zeros(3, dtype=i32)
    bad = [(TypeError, pages_b200.reserve, (table.long(), lens, refs, two, 16)), (ValueError, pages_b200.reserve, (table, lens[:1], refs, two, 16)),
           (ValueError, pages_b200.reserve, (table, lens, refs, two[:1], 16)), (TypeError, pages_b200.free, (table, lens, refs, two.float(), 16)),
           (ValueError, pages_b200.fork, (pool, table, lens, refs, two, two)), (ValueError, pages_b200.fork, ([], table, lens, refs, two, two)),
           (ValueError, pages_b200.fork, ([pool], table, lens, refs[:7], two, two)), (ValueError, pages_b200.fork, ([pool], table, lens, refs, two, two[:1])),
           (ValueError, pages_b200.fork, ([pool, pool[:7].contiguous()], table, lens, refs, two, two)),
           (ValueError, pages_b200.fork, ([pool[:, :, :, :4].contiguous()], table, lens, refs, two, two)),
           (ValueError, pages_b200.fork, ([pool.transpose(1, 2)], table, lens, refs, two, two)),
           (ValueError, pages_b200.compact, ([pool], table, lens, refs, two, two)), (ValueError, pages_b200.compact, ([pool], table, lens, refs, table[:1], two)),
           (ValueError, pages_b200.copy, ([pool], two, two[:1])), (ValueError, pages_b200.copy, ([], two, two)), (ValueError, pages_b200.copy, ([pool] * 9, two, two)),
           (TypeError, pages_b200.append, (k.float(), k, pool, pool, table, cu, lens)), (ValueError, pages_b200.append, (k[:, :1], k, pool, pool, table, cu, lens)),
           (ValueError, pages_b200.append, (k, k[:4], pool, pool, table, cu, lens)), (ValueError, pages_b200.append, (k, k, pool[None], pool[None], table, cu, lens)),
           (ValueError, pages_b200.append, (k, k, pool, pool, table, torch.zeros(4, dtype=i32), lens)),
           (ValueError, pages_b200.append, (torch.zeros(5, 2, 12, dtype=torch.float16)[:, :, :8], k, pool, pool, table, cu, lens))]
    for err, fn, args in bad:
        with pytest.raises(err):
            fn(*args)


def test_statement_of_the_acceptance_by_hand():
    p, q = np.array([[[0.5, 0.3, 0.2]] * 2]), np.array([[[0.2, 0.6, 0.2]] * 2])
    base = dict(target_probs=p, draft_probs=q, bits=np.array([[1, 3]]), tokens=np.array([[0, 1]]))
    # token 1 stands with probability 0.3 / 0.6; refused, the residual is (0.3, 0, 0): token 0
    path, count, nxt, _ = ref64.accept_ref64(u=np.array([[0.9, 0.49]]), **base)
    assert path.tolist() == [[0, 1]] and count.tolist() == [2] and nxt.tolist() == [2]
    path, count, nxt, _ = ref64.accept_ref64(u=np.array([[0.9, 0.51]]), **base)
    assert path.tolist() == [[0, -1]] and count.tolist() == [1] and nxt.tolist() == [0]
    # chosen drafts: token 1 stands with probability 0.3; refused, the rest is (0.5, 0, 0.2) of 0.7
    base["draft_probs"] = None
    assert ref64.accept_ref64(u=np.array([[0.72, 0.31]]), **base)[2].tolist() == [2]
    assert ref64.accept_ref64(u=np.array([[0.70, 0.31]]), **base)[2].tolist() == [0]
    # a second child that repeats the refused token cannot stand
    base.update(bits=np.array([[1, 3, 5]]), tokens=np.array([[0, 1, 1]]), target_probs=np.array([[[0.5, 0.3, 0.2]] * 3]))
    assert ref64.accept_ref64(u=np.array([[0.70, 0.31, 0.0]]), **base)[1].tolist() == [1]


def test_the_closed_form_is_the_recursion():
    """S and M against the residual that is normalised again, over several refusals."""
    rng = np.random.default_rng(0)
    p, q = rng.random(50), rng.random(50)
    p, q = p / p.sum(), q / q.sum()
    r, mass, S, M = p.copy(), 1.0, 0.0, 1.0
    for _ in range(6):
        r = np.maximum(r / mass - q, 0) * 1.0
        mass = r.sum()
        S += M
        closed = np.maximum(p - S * q, 0)
        M = closed.sum()
        assert M > 0
        np.testing.assert_allclose(r / mass, closed / M, rtol=1e-9, atol=1e-12)


def test_generated_trees_have_parents_below():
    inp = op.make_inputs(2, 40, 30, 3, seed=1)
    assert inp["bits"].shape == (2, 40, 2) and inp["draft_probs"].shape == (2, 40, 30)


def test_the_page_model_by_hand():
    m = Model(np.full((3, 3), -1, np.int32), np.zeros(3, np.int32), np.zeros(5, np.int32), 4, [np.arange(5 * 4).reshape(1, 5, 1, 4, 1).astype(np.int64)])
    assert m.reserve([5, 8, 9]).tolist() == [1, 1, 0] and m.status == 4 and m.table.tolist() == [[0, 1, -1], [2, 3, -1], [-1, -1, -1]]
    m.fork([0], [2])
    assert m.table[2].tolist() == [0, 4, -1] and m.refs.tolist() == [2, 1, 1, 1, 1] and m.pools[0][0, 4, 0, :, 0].tolist() == [4, 17, 18, 19]
    m.compact(np.array([[0, -1], [1, -1], [0, 1]]), [-1, 1, 0])
    assert m.lens.tolist() == [5, 7, 3] and m.table[2].tolist() == [0, -1, -1] and m.refs.tolist() == [2, 1, 1, 1, 0]
    assert m.pools[0][0, 3, 0, :, 0].tolist() == [12, 13, 15, 15]
    m.free([0, 4, 0])
    assert m.refs.tolist() == [0, 0, 1, 0, 0] and m.lens.tolist() == [0, 4, 0]
