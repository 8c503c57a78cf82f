"""Acceptance of drafts on the GPU through the C ABI against the float64 statement.  The answers are whole numbers and have to
be equal, except where a comparison of the statement is nearer to its border than the order of 64-bit sums can move it:
a sum of V numbers in another order moves by less than V 2^-53 of itself."""
import numpy as np
import pytest
import torch

from oracle import ref64
from verified_metal_kernels_b200 import _lib, check_status
from verified_metal_kernels_b200.kernels import accept_b200
from verified_metal_kernels_b200.ops import accept as op

pytestmark = pytest.mark.gpu


def _dev(inp, dtype=torch.float32):
    d = {k: None if v is None else torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in inp.items()}
    for k in ("target_probs", "draft_probs"):
        if d[k] is not None:
            d[k] = d[k].to(dtype)
    return d


def _truth(d):
    host = {k: None if v is None else (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in d.items()}
    return ref64.accept_ref64(**host)


def _check(got, d):
    path, count, nxt, near = _truth(d)
    sure = near > d["target_probs"].shape[2] * 2.0 ** -50
    assert sure.mean() > 0.9
    for g, w in zip(got, (path, count, nxt)):
        assert g.dtype == torch.int32
        assert np.array_equal(g.cpu().numpy()[sure], w[sure])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(op.FUZZ)))
def test_against_the_float64_statement(case, dtype):
    B, kd, V, depth, draft, dist = op.FUZZ[case]
    d = _dev(op.make_inputs(B, kd, V, depth, draft, dist, seed=100 + case), dtype)
    got = accept_b200.kernel(**d, check=True)
    _check(got, d)
    for a, b in zip(got, accept_b200.kernel(**d)):
        assert torch.equal(a, b)


def test_a_draft_equal_to_the_target_always_stands():
    B, kd, V, depth, draft, dist = 20, 12, 500, 0, True, "same"
    d = _dev(op.make_inputs(B, kd, V, depth, draft, dist, seed=3))
    path, count, nxt = accept_b200.kernel(**d, check=True)
    assert (count == kd).all() and torch.equal(path, torch.arange(kd, dtype=torch.int32, device="cuda").expand(B, kd))


def test_the_tokens_are_distributed_as_the_target():
    """200000 requests with one draft each over five tokens: the first token that comes out has the target's frequencies.
    A frequency of n draws is off by more than 6 sqrt(f (1 - f) / n) once in 5e8 times."""
    n, V = 200000, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.tensor([0.05, 0.4, 0.3, 0.0, 0.25], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.3, 0.2, 0.1], device="cuda")
    for draft in (True, False):
        tok = torch.zeros(n, 3, dtype=torch.int32, device="cuda")
        tok[:, 1:] = torch.multinomial(q, 2 * n, replacement=True, generator=g).view(n, 2).int()
        bits = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda").expand(n, 3).contiguous()      # two children of the root
        u = torch.rand(n, 3, generator=g, device="cuda")
        path, count, nxt = accept_b200.kernel(p.expand(n, 3, V).contiguous(), tok, bits, u, draft_probs=q.expand(n, 3, V).contiguous() if draft else None, check=True)
        first = torch.where(count > 1, tok.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
        f = torch.bincount(first.long(), minlength=V).double() / n
        assert ((f - p.double()).abs() <= 6 * (p.double() * (1 - p.double()) / n).sqrt() + 1e-12).all(), f


def test_rows_of_nothing_and_values_that_are_none():
    B, kd, V = 6, 4, 3001
    inp = op.make_inputs(B, kd, V, 2, True, "near", seed=5)
    p = inp["target_probs"]
    p[0] = 0
    p[1] = np.nan
    p[2, :, ::3] = np.inf
    p[2, :, 1::3] = -1.0
    p[3, :, :] = 0
    p[3, :, 2999] = 1e-30
    inp["draft_probs"][4] = 0
    inp["draft_probs"][5, :, 5:] = np.nan
    for draft in (True, False):
        d = _dev(inp if draft else dict(inp, draft_probs=None))
        got = accept_b200.kernel(**d, check=True)
        _check(got, d)
        assert got[2].tolist()[:2] == [-1, -1] and got[2].tolist()[3] == 2999


def test_numbers_at_the_ends_of_their_range():
    B, kd, V = 5, 3, 700
    inp = op.make_inputs(B, kd, V, 0, True, "near", seed=6)
    inp["u"][0], inp["u"][1], inp["u"][2] = 0.0, 1.0 - 2.0 ** -24, 1.0
    inp["u"][3], inp["u"][4] = np.nan, -0.5
    d = _dev(inp)
    path, count, nxt = accept_b200.kernel(**d, check=True)
    assert count[0] == kd and nxt[0] == 0
    assert count[3] == 1 and count[4] == kd and ((nxt >= 0) & (nxt < V)).all()
    want = ref64.accept_ref64(**{k: v[:3] for k, v in inp.items()})
    assert np.array_equal(count.cpu().numpy()[:3], want[1]) and np.array_equal(nxt.cpu().numpy()[:2], want[2][:2])


def test_several_roots_and_bits_of_later_nodes():
    """Only the highest node below i in bits[i] is its parent: later bits say nothing, a node without one is no child."""
    V = 40
    inp = op.make_inputs(2, 5, V, 0, True, "same", seed=7)
    inp["bits"][:] = np.array([0x1F, 2, 0x1D, 8 | 4, 16 | 8], dtype=np.int32)      # node 1 has no parent, node 2 is the root's
    inp["tokens"][:, 2] = inp["target_probs"][:, 0].argmax(-1)
    inp["tokens"][:, 3] = inp["target_probs"][:, 2].argmax(-1)
    inp["tokens"][:, 4] = inp["target_probs"][:, 3].argmax(-1)
    d = _dev(inp)
    path, count, _ = accept_b200.kernel(**d, check=True)
    assert path.tolist() == [[0, 2, 3, 4, -1]] * 2 and count.tolist() == [4, 4]
    _check(accept_b200.kernel(**d), d)


def test_tokens_outside_the_vocabulary_are_refused_and_reported():
    inp = op.make_inputs(3, 4, 100, 0, True, "same", seed=8)
    inp["tokens"][0, 1], inp["tokens"][1, 2], inp["tokens"][2, 0] = 100, -1, 10 ** 9      # the root's is not read
    for draft in (True, False):
        d = _dev(inp if draft else dict(inp, draft_probs=None))
        got = accept_b200.kernel(**d)
        with pytest.raises(_lib.VmkDeviceStatusError) as e:
            check_status("cuda:0")
        assert e.value.status == 2
        _check(got, d)
        assert got[1][0] == 1 and got[1][1] <= 2


def test_independent_of_the_batch_under_the_invariant_switch():
    lib = _lib.lib()
    d = _dev(op.make_inputs(120, 6, 20011, 2, True, "near", seed=9))
    lib.vmk_set_batch_invariant(1)
    try:
        whole = accept_b200.kernel(**d)
        for b in (0, 50, 119):
            for a, w in zip(accept_b200.kernel(**{k: v[b:b + 1].contiguous() for k, v in d.items()}), whole):
                assert torch.equal(a[0], w[b])
    finally:
        lib.vmk_set_batch_invariant(0)


def test_tensors_that_begin_anywhere():
    """Slices of a batch of odd rows: the two tensors begin at different places of a 16-byte vector."""
    for dtype in (torch.float32, torch.bfloat16):
        d = _dev(op.make_inputs(3, 5, 1009, 2, True, "near", seed=11), dtype)
        e = dict(d, target_probs=torch.empty(3 * 5 * 1009 + 3, dtype=dtype, device="cuda")[3:].view(3, 5, 1009))
        e["target_probs"].copy_(d["target_probs"])
        for a, b in zip(accept_b200.kernel(**e, check=True), accept_b200.kernel(**d)):
            assert torch.equal(a, b)


def test_empty_batch():
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")
    path, count, nxt = accept_b200.kernel(z(0, 4, 10, dtype=torch.float32), z(0, 4), z(0, 4), z(0, 4, dtype=torch.float32), check=True)
    assert path.shape == (0, 4) and count.shape == (0,) and nxt.shape == (0,)


def test_streams_graphs_and_host_tensors():
    inp = op.make_inputs(4, 8, 5003, 3, True, "near", seed=10)
    d = _dev(inp)
    want = accept_b200.kernel(**d)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, accept_b200.kernel(**d)))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = accept_b200.kernel(**d)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got in [other] + [o for _, o in graphs]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    d["u"].copy_(torch.rand(4, 8, device="cuda"))
    new = accept_b200.kernel(**d)
    for g, out in graphs:
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, new))
    host = accept_b200.kernel(**{k: torch.from_numpy(v) for k, v in inp.items()})
    assert all(not a.is_cuda and torch.equal(a, b.cpu()) for a, b in zip(host, want))
