"""The operators together, as a serving loop uses them: pages reserved and filled, prompts answered from them, a draft tree
verified, accepted and closed up, single tokens decoded, requests forked and freed.  Every attention call over the pages
equals the same call over contiguous caches that the test keeps beside them."""
import numpy as np
import pytest
import torch

from tests import _verify
from verified_metal_kernels_b200.kernels import accept_b200, decode_b200, pages_b200, prompt_b200, spec_b200
from verified_metal_kernels_b200.ops import spec

pytestmark = pytest.mark.gpu
HQ, HKV, D, PS = 8, 2, 128, 64


def _dense(rows):
    """(keys, values) of each row, lists of (n, Hkv, D), padded to (R, Hkv, L, D)."""
    L = max(k.shape[0] for k, _ in rows)
    pad = lambda x: torch.cat([x, x.new_zeros(L - x.shape[0], HKV, D)]).transpose(0, 1)
    return torch.stack([pad(k) for k, _ in rows]), torch.stack([pad(v) for _, v in rows])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_prompt_verify_accept_compact_decode_fork_free(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    R, B, n, kd = 7, 3, 190, 40                       # three requests, four rows to fork into
    pools = [torch.full((40, HKV, PS, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    table, lens, refs = torch.full((R, 8), -1, dtype=torch.int32, device="cuda"), ints([0] * R), ints([0] * 40)
    # the prompts, in two chunks
    rows = [(randn(n, HKV, D), randn(n, HKV, D)) for _ in range(B)]
    q = [randn(n, HQ, D) for _ in range(B)]
    whole = prompt_b200.kernel(torch.cat(q), torch.cat([k for k, _ in rows]), torch.cat([v for _, v in rows]), ints([0, n, 2 * n, 3 * n]))
    for lo, hi in ((0, 77), (77, n)):
        c = hi - lo
        cu = ints([0, c, 2 * c, 3 * c])
        pages_b200.reserve(table, lens, refs, ints([c] * B + [0] * (R - B)), PS, check=True)
        pages_b200.append(torch.cat([k[lo:hi] for k, _ in rows]), torch.cat([v[lo:hi] for _, v in rows]), *pools, table, cu, lens, check=True)
        out = prompt_b200.kernel_paged(torch.cat([x[lo:hi] for x in q]), *pools, table[:B], cu, lens[:B], check=True)
        for b in range(B):
            # the same keys in other tiles of queries: the rounding of P and of the output, with values of size about 1
            assert (out[b * c:(b + 1) * c].float() - whole[b * n + lo:b * n + hi].float()).abs().max() <= 16 * torch.finfo(dtype).eps
    # a tree of drafts at the end of each row
    pages_b200.reserve(table, lens, refs, ints([kd] * B + [0] * (R - B)), PS, check=True)
    new = [(randn(kd, HKV, D), randn(kd, HKV, D)) for _ in range(B)]
    pages_b200.append(torch.cat([k for k, _ in new]), torch.cat([v for _, v in new]), *pools, table, ints([0, kd, 2 * kd, 3 * kd]), lens, check=True)
    rows = [(torch.cat([a, c]), torch.cat([b, d])) for (a, b), (c, d) in zip(rows, new)]
    rng = np.random.default_rng(5)
    masks = [spec.tree_bits(kd, rng, 5) for _ in range(B)]
    bits = torch.from_numpy(spec.pack_bits(masks, kd)).cuda()
    qd = randn(B, kd, HQ, D)
    k, v = (x.contiguous() for x in _dense(rows))
    assert torch.equal(spec_b200.kernel_paged(qd, *pools, table[:B].contiguous(), n + kd, bits, check=True), spec_b200.kernel(qd, k, v, bits))
    # what stands of it
    V = 300
    p = torch.softmax(torch.randn(B, kd, V, generator=g, device="cuda"), -1)
    tok = torch.randint(0, V, (B, kd), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(B, kd, generator=g, device="cuda") * 0.002          # small numbers: chosen drafts of this target stand often
    path, count, nxt = accept_b200.kernel(p, tok, bits, u, check=True)
    assert count.max() > 2
    full = torch.full((R, kd), -1, dtype=torch.int32, device="cuda")
    full[:B] = path
    pages_b200.compact(pools, table, lens, refs, full, torch.cat([count, ints([-1] * (R - B))]), check=True)
    at = [[n + j for j in path[b, :count[b]].tolist()] for b in range(B)]
    rows = [(torch.cat([k[:n], k[a]]), torch.cat([v[:n], v[a]])) for (k, v), a in zip(rows, at)]
    assert lens.tolist() == [n + int(c) for c in count] + [0] * (R - B)
    # single tokens over what is left, and over forked rows that grow by a token each
    one = randn(B, HQ, D)
    k, v = (x.contiguous() for x in _dense(rows))
    assert torch.equal(decode_b200.kernel_paged(one, *pools, table[:B].contiguous(), lens[:B].contiguous(), check=True), decode_b200.kernel(one, k, v, lens[:B].contiguous()))
    pages_b200.fork(pools, table, lens, refs, ints([0, 0, 2, 1]), ints([3, 4, 5, 6]), check=True)
    rows += [rows[0], rows[0], rows[2], rows[1]]
    pages_b200.reserve(table, lens, refs, ints([1] * R), PS, check=True)
    k1, v1 = randn(R, HKV, D), randn(R, HKV, D)
    pages_b200.append(k1, v1, *pools, table, ints(range(R + 1)), lens, check=True)
    rows = [(torch.cat([k, k1[r:r + 1]]), torch.cat([v, v1[r:r + 1]])) for r, (k, v) in enumerate(rows)]
    one = randn(R, HQ, D)
    k, v = (x.contiguous() for x in _dense(rows))
    assert torch.equal(decode_b200.kernel_paged(one, *pools, table, lens, check=True), decode_b200.kernel(one, k, v, lens))
    assert int(refs.max()) > 1
    pages_b200.free(table, lens, refs, ints([0] * R), PS, check=True)
    assert int(refs.abs().sum()) == 0 and int(lens.sum()) == 0 and (table == -1).all()
    _verify.assert_clean_status()
