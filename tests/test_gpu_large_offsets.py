"""Prompt, accept and page operators where byte and element offsets pass 32 bits: pools and inputs of more than 4 GiB of which a
call touches the far end, against the same call on small tensors (the same bits, the arithmetic being the same)."""
import pytest
import torch

from verified_metal_kernels_b200.kernels import accept_b200, pages_b200, prompt_b200

pytestmark = pytest.mark.gpu
PAGE, HEADS, D = 64, 8, 128
FAR = 35000                                    # pages of 128 KiB before the ones in use: 4.6 GB


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _half(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").half()


def test_pages_far_into_their_pools():
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, q = _half(g, 300, HEADS, D), _half(g, 300, HEADS, D), _half(g, 300, 32, D)
    got = []
    for before in (0, FAR):
        pools = [torch.empty(before + 12, HEADS, PAGE, D, dtype=torch.float16, device="cuda") for _ in range(2)]
        for p in pools:
            p[before:].zero_()
        table, lens = torch.full((3, 5), -1, dtype=torch.int32, device="cuda"), _ints([0, 0, 0])
        refs = torch.ones(before + 12, dtype=torch.int32, device="cuda")
        refs[before:] = 0
        assert pages_b200.reserve(table, lens, refs, _ints([200, 100, 0]), PAGE, check=True).tolist() == [1, 1, 1]
        pages_b200.append(k, v, *pools, table, _ints([0, 200, 300]), lens, check=True)
        pages_b200.fork(pools, table, lens, refs, _ints([1]), _ints([2]), check=True)
        pages_b200.compact(pools, table, lens, refs, _ints([[0, 2, 4, -1, -1]] * 3), _ints([3, 3, -1]), check=True)
        pages_b200.copy(pools, _ints([before]), _ints([before + 11]), check=True)
        out = prompt_b200.kernel_paged(q[:60], *pools, table[:2], _ints([0, 20, 60]), lens[:2], check=True)
        pages_b200.free(table, lens, refs, _ints([64, 0, 100]), PAGE, check=True)
        got.append((out, table - before * (table >= 0), lens, refs[before:], *[p[before:].clone() for p in pools]))
        del pools
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_queries_far_into_their_tensor():
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = _half(g, 50, 64, D), _half(g, 50, HEADS, D)
    want = prompt_b200.kernel(q, k, k, _ints([0, 50]), check=True)
    n = (1 << 18) + 50                         # 64 heads of 128: 2^31 elements and more
    far = torch.empty(n, 64, D, dtype=torch.float16, device="cuda")
    far[-50:] = q
    out = prompt_b200.kernel(far, k, k, _ints([n - 50, n]), _ints([0, 50]), check=True)
    assert torch.equal(out[-50:], want) and not out[:-50].any()


def test_requests_far_into_the_probabilities():
    g = torch.Generator(device="cuda").manual_seed(2)
    V, kd = 131072, 64
    p = torch.softmax(2 * torch.randn(1, kd, V, generator=g, device="cuda"), -1).half()
    tok = torch.randint(0, V, (1, kd), generator=g, device="cuda", dtype=torch.int32)
    tok[0, 1] = p[0, 0].argmax()
    u = torch.rand(1, kd, generator=g, device="cuda") * 1e-4
    bits = torch.zeros(1, kd, 2, dtype=torch.int32, device="cuda")
    bits[0, :, 0] = 3                          # nodes 0 and 1 are everybody's ancestors
    bits[0, 0, 0] = 1
    B = 260                                    # 260 x 64 x 131072: 2^31 elements and more
    far = torch.zeros(B, kd, V, dtype=torch.float16, device="cuda")
    far[-1] = p[0]
    want = accept_b200.kernel(p, tok, bits, u, check=True)
    got = accept_b200.kernel(far, tok.expand(B, kd).contiguous(), bits.expand(B, kd, 2).contiguous(), u.expand(B, kd).contiguous(), check=True)
    assert want[1].item() >= 2
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[-1])
    assert (got[1][:-1] == 1).all() and (got[2][:-1] == -1).all()
