"""Units whose keys several CTAs share: a NaN or infinity in V reaches the rows that see its key also where the weight of the
share that holds it comes to 0, and no other element changes by a bit."""
import numpy as np
import pytest
import torch

from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import prompt_b200
from verified_metal_kernels_b200.ops import prompt as op

pytestmark = pytest.mark.gpu


# one 128-row tile in both tiles of a share, two tiles, and one sequence of each
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("seqs", [[(5, 6000)], [(60, 6000)], [(1, 5600), (40, 5900)]], ids=str)
def test_special_values_in_a_share_without_weight(seqs, dtype):
    """Scores of the first 5000 keys are 636 below the others (918 steps of a power of two): their share of the sum is 0 in fp32."""
    nq, nk = [n for n, _ in seqs], [m for _, m in seqs]
    g = torch.Generator(device="cuda").manual_seed(1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = torch.zeros(sum(nq), 8, 128, dtype=dtype, device="cuda")
    q[..., 0] = 60
    k = torch.zeros(sum(nk), 2, 128, dtype=dtype, device="cuda")
    v = torch.randn(sum(nk), 2, 128, generator=g, device="cuda").to(dtype)
    marked = v.clone()
    want = torch.zeros(sum(nq), 8, 128, dtype=torch.bool, device="cuda")
    for s, (n, m) in enumerate(seqs):
        at, to = sum(nk[:s]), sum(nq[:s])
        k[at:at + m, :, 0] = 60
        k[at:at + 5000, :, 0] = -60
        for key, head, col, x in ((100, 0, 3, float("nan")), (2000, 1, 5, float("inf")), (4999, 1, 127, float("-inf")), (m - 1, 0, 9, float("inf"))):
            marked[at + key, head, col] = x
            want[max(to, to + n - (m - key)):to + n, head * 4:head * 4 + 4, col] = True
    cu = ints(np.concatenate([[0], np.cumsum(nq)])), ints(np.concatenate([[0], np.cumsum(nk)]))

    def both(v):
        kp, vp, table = op.to_pages(k.float().cpu().numpy(), v.float().cpu().numpy(), nk, 64, seed=2)
        yield prompt_b200.kernel(q, k, v, *cu, check=True)
        yield prompt_b200.kernel_paged(q, torch.from_numpy(kp).cuda().to(dtype), torch.from_numpy(vp).cuda().to(dtype), torch.from_numpy(table).cuda(),
                                       cu[0], ints(nk), check=True)

    for clean, got in zip(both(v), both(marked)):
        assert torch.isfinite(clean).all()
        assert not torch.isfinite(got[want]).any() and torch.equal(got[~want], clean[~want])
    # where one CTA takes all keys the same rows are reached
    _lib.lib().vmk_set_batch_invariant(1)
    try:
        alone = prompt_b200.kernel(q, k, marked, *cu, check=True)
    finally:
        _lib.lib().vmk_set_batch_invariant(0)
    assert torch.equal(~torch.isfinite(alone), want)
