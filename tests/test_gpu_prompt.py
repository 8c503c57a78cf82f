"""Prompt attention on the GPU through the C ABI against the float64 statement: lengths around the tiles, rows that see
nothing, grouped heads of every kind, pages, views, other streams, captured graphs, bad lengths.

Tolerance of an output element, from the roundings that the kernel makes (u = half a step of the 16-bit type, relative):
  u |o|                 the output's own rounding,
  u a                   P rounded to 16 bits before P.V, where a = sum_j p_j |v_j| (fp16: P below 2^-14 is off by up to
                        2^-25 instead, and P of the largest score is at least 1: 2^-25 sum |v_j| <= 2^-25 n max|v|),
  a (2^-20 s + 2^-18)   scores, exponentials and sums in fp32: a score is a sum of 128 products, off by at most
                        2^-20 s with s = sum |q_d k_d| / sqrt(D) (128 additions of 2^-24, each of at most s, and the
                        rounding of the scaled maximum), an error e of a score changes p by a factor of 1 + e twice
                        (in p and in the sum: the factor two is in the 2^-20); exponentials and the sum over n keys
                        are off by less than 2^-18 for n up to some thousands of keys."""
import numpy as np
import pytest
import torch

from oracle import ref64
from tests import _verify
from verified_metal_kernels_b200 import _lib, check_status, ops
from verified_metal_kernels_b200.kernels import prompt_b200
from verified_metal_kernels_b200.ops import prompt as op

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _dev(inp, dtype):
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in inp.items()}
    for k in ("q", "k", "v"):
        d[k] = d[k].to(dtype)
    return d


def _inputs(seqs, hq, hkv, dtype, **kw):
    inp = op.make_inputs(seqs, hq, hkv, **kw)
    if dtype == torch.bfloat16:
        for k in ("q", "k", "v"):
            inp[k] = ops.round_bf16(inp[k])
    return inp


def _check(out, inp, seqs, dtype, causal=True):
    nq, nk = [n for n, _ in seqs], [m for _, m in seqs]
    truth, a, s = ref64.prompt_ref64(inp["q"], inp["k"], inp["v"], nq, nk, causal)
    got = out.float().cpu().numpy().astype(np.float64)
    u = HALF[dtype]
    n = max(nk, default=0)
    vmax = np.abs(np.asarray(inp["v"], dtype=np.float64)[:sum(nk)]).max(initial=0.0)
    floor = n * vmax * 2.0 ** -25 + 2.0 ** -25 if dtype == torch.float16 else 1e-38
    tol = u * np.abs(truth) + (u + 2.0 ** -20 * s[:, :, None] + 2.0 ** -18) * a + floor
    assert np.isfinite(got).all()
    bad = np.abs(got - truth) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - truth) / np.maximum(tol, 1e-30)).max()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(op.FUZZ)))
def test_against_the_float64_statement(case, dtype):
    seqs, hq, hkv, dist = op.FUZZ[case]
    inp = _inputs(seqs, hq, hkv, dtype, seed=71 + case, dist=dist)
    d = _dev(inp, dtype)
    out = prompt_b200.kernel(**d, check=True)
    assert out.dtype == dtype and out.shape == d["q"].shape
    _check(out, inp, seqs, dtype)
    full = prompt_b200.kernel(**d, causal=False, check=True)
    _check(full, inp, seqs, dtype, causal=False)


@pytest.mark.parametrize("page_size", [64, 128, 192])
@pytest.mark.parametrize("case", [2, 3, 4, 5, 9, 12])
def test_paged_equals_contiguous_bit_for_bit(case, page_size):
    """The same tiles in the same order; pages hold NaN behind the sequences, the table -1."""
    seqs, hq, hkv, dist = op.FUZZ[case]
    inp = _inputs(seqs, hq, hkv, torch.float16, seed=5 + case, dist=dist)
    d = _dev(inp, torch.float16)
    nk = [m for _, m in seqs]
    kp, vp, table = op.to_pages(inp["k"], inp["v"], nk, page_size, seed=3)
    out = prompt_b200.kernel_paged(d["q"], torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), torch.from_numpy(table).cuda(),
                                   d["cu_q"], torch.tensor(nk, dtype=torch.int32, device="cuda"), check=True)
    _check(out, inp, seqs, torch.float16)
    assert torch.equal(out, prompt_b200.kernel(**d))


def test_padding_is_zero_and_what_lies_behind_the_keys_does_not_matter():
    seqs = [(50, 50), (77, 77)]
    inp = _inputs(seqs, 8, 2, torch.bfloat16, seed=9, pad_q=300, pad_k=200, fill=np.nan)
    d = _dev(inp, torch.bfloat16)
    junk = torch.full((4 << 20,), float("nan"), device="cuda")          # what the allocator hands out next is not zero
    del junk
    out = prompt_b200.kernel(**d, check=True)
    _check(out, inp, seqs, torch.bfloat16)
    assert (out[127:] == 0).all()
    # a first sequence that does not begin at row 0: the rows before it are zero too
    shifted = prompt_b200.kernel(d["q"], d["k"], d["v"], d["cu_q"][1:].contiguous(), d["cu_k"][1:].contiguous(), check=True)
    assert (shifted[:50] == 0).all() and torch.equal(shifted[50:127], out[50:127])


def test_keys_of_another_sequence_may_be_nan_or_infinite():
    seqs = [(70, 70), (61, 61), (90, 90)]
    inp = _inputs(seqs, 8, 2, torch.float16, seed=19)
    inp["k"][70:131], inp["v"][70:131] = np.nan, np.inf
    d = _dev(inp, torch.float16)
    out = prompt_b200.kernel(**d, check=True)
    assert not torch.isfinite(out[70:131]).any()
    clean = dict(inp, k=inp["k"].copy(), v=inp["v"].copy())
    clean["k"][70:131], clean["v"][70:131] = 0, 0
    out[70:131] = prompt_b200.kernel(**_dev(clean, torch.float16))[70:131]
    _check(out, clean, seqs, torch.float16)


def test_a_nan_key_reaches_the_rows_that_see_it_and_no_other():
    seqs = [(300, 300)]
    inp = _inputs(seqs, 4, 2, torch.float16, seed=23)
    clean = prompt_b200.kernel(**_dev(inp, torch.float16))
    inp["k"][201, 1] = np.nan
    out = prompt_b200.kernel(**_dev(inp, torch.float16), check=True)
    assert torch.isnan(out[201:, 2:]).all()
    assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[:201], clean[:201])


def test_views_of_a_fused_projection():
    seqs = [(100, 100), (33, 33)]
    inp = _inputs(seqs, 12, 4, torch.bfloat16, seed=29)
    d = _dev(inp, torch.bfloat16)
    fused = torch.cat([d["q"], d["k"], d["v"]], dim=1)                     # (T, 12 + 4 + 4, 128)
    out = prompt_b200.kernel(fused[:, :12], fused[:, 12:16], fused[:, 16:], d["cu_q"], check=True)
    ref = prompt_b200.kernel(**d)
    assert torch.equal(out, ref)
    by_head = {k: d[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("q", "k", "v")}
    assert torch.equal(prompt_b200.kernel(**by_head, cu_q=d["cu_q"], check=True), ref)


def test_a_row_does_not_depend_on_what_else_is_in_the_batch():
    seqs = [(40, 40), (513, 513), (7, 260)]
    inp = _inputs(seqs, 8, 2, torch.float16, seed=31)
    d = _dev(inp, torch.float16)
    out = prompt_b200.kernel(**d)
    q, k, v = d["q"][40:553], d["k"][40:553], d["v"][40:553]
    alone = prompt_b200.kernel(q, k, v, torch.tensor([0, 513], dtype=torch.int32, device="cuda"))
    assert torch.equal(out[40:553], alone)


def test_more_sequences_than_the_planner_has_threads():
    rng = np.random.default_rng(3)
    seqs = [(int(n), int(n)) for n in rng.integers(0, 4, 2500)]
    inp = _inputs(seqs, 4, 4, torch.float16, seed=37)
    out = prompt_b200.kernel(**_dev(inp, torch.float16), check=True)
    _check(out, inp, seqs, torch.float16)


def test_many_units_for_each_multiprocessor():
    """Thousands of units of different costs, against single calls of some of the sequences."""
    rng = np.random.default_rng(4)
    seqs = [(int(n), int(n)) for n in rng.integers(1, 1200, 40)]
    inp = _inputs(seqs, 32, 8, torch.bfloat16, seed=41)
    d = _dev(inp, torch.bfloat16)
    out = prompt_b200.kernel(**d, check=True)
    at = 0
    for i, (n, _) in enumerate(seqs):
        if i % 9 == 0:
            alone = prompt_b200.kernel(d["q"][at:at + n], d["k"][at:at + n], d["v"][at:at + n], torch.tensor([0, n], dtype=torch.int32, device="cuda"))
            assert torch.equal(out[at:at + n], alone)
            sub = {k: inp[k][at:at + min(n, 70)] for k in ("q", "k", "v")}
            _check(out[at:at + min(n, 70)], sub, [(min(n, 70), min(n, 70))], torch.bfloat16)
        at += n


def test_last_position_equals_single_token_decode():
    """The single-token form is `decode`: the last query of a prompt against a decode step over the same cache."""
    from verified_metal_kernels_b200.kernels import decode_b200
    n = 777
    inp = _inputs([(n, n)], 32, 8, torch.float16, seed=43)
    d = _dev(inp, torch.float16)
    out = prompt_b200.kernel(**d)
    cache = {k: d[k].transpose(0, 1)[None].contiguous() for k in ("k", "v")}
    step = decode_b200.kernel(d["q"][-1:].contiguous(), cache["k"], cache["v"], torch.tensor([n], dtype=torch.int32, device="cuda"))
    a = np.abs(inp["v"].astype(np.float64)).max()
    assert (out[-1] - step[0]).abs().max().item() <= 4 * HALF[torch.float16] * a


def test_no_queries_and_no_sequences():
    q = torch.empty(0, 8, 128, dtype=torch.float16, device="cuda")
    k = torch.empty(0, 2, 128, dtype=torch.float16, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert prompt_b200.kernel(q, k, k, cu, check=True).shape == (0, 8, 128)
    q = torch.randn(9, 8, 128, device="cuda").half()
    assert (prompt_b200.kernel(q, k, k, cu[:1], check=True) == 0).all()
    assert (prompt_b200.kernel(q, k, k, torch.tensor([0, 9], dtype=torch.int32, device="cuda"), cu[:2].contiguous(), check=True) == 0).all()


def test_lengths_outside_their_tensors_are_clamped_and_reported():
    inp = _inputs([(60, 60)], 8, 2, torch.float16, seed=47)
    d = _dev(inp, torch.float16)
    ref = prompt_b200.kernel(**d, check=True)
    out = prompt_b200.kernel(d["q"], d["k"], d["v"], torch.tensor([-5, 4000], dtype=torch.int32, device="cuda"))
    with pytest.raises(_lib.VmkDeviceStatusError) as e:
        check_status(out.device)
    assert e.value.status == 2
    assert torch.equal(out, ref)
    prompt_b200.kernel(d["q"], d["k"], d["v"], torch.tensor([0, 60, 20, 60, 0], dtype=torch.int32, device="cuda"))
    with pytest.raises(_lib.VmkDeviceStatusError):
        check_status(out.device)


def test_on_another_stream_and_twice_at_once():
    seqs = [(400, 400), (90, 90)]
    inp = _inputs(seqs, 16, 4, torch.bfloat16, seed=53)
    other = _inputs(seqs, 16, 4, torch.bfloat16, seed=59)
    d, e = _dev(inp, torch.bfloat16), _dev(other, torch.bfloat16)
    ref, ref2 = prompt_b200.kernel(**d), prompt_b200.kernel(**e)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            outs.append((prompt_b200.kernel(**d), ref))
        with torch.cuda.stream(s2):
            outs.append((prompt_b200.kernel(**e), ref2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    _verify.assert_clean_status()


def test_captured_twice_and_replayed_with_other_lengths():
    seqs = [(100, 100), (30, 30)]
    inp = _inputs(seqs, 8, 2, torch.float16, seed=61, pad_q=70, pad_k=70)
    d = _dev(inp, torch.float16)
    prompt_b200.kernel(**d)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(prompt_b200.kernel(**d))
        graphs.append(g)
    for new in ([(100, 100), (30, 30)], [(3, 3), (190, 190)]):
        inp["cu_q"] = np.array([0, new[0][0], new[0][0] + new[1][0]], dtype=np.int32)
        d["cu_q"].copy_(torch.from_numpy(inp["cu_q"]))
        d["cu_k"].copy_(torch.from_numpy(inp["cu_q"]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            _check(o, inp, new, torch.float16)
    _verify.assert_clean_status()


def test_host_tensors_come_back_on_the_host():
    seqs = [(44, 44)]
    inp = _inputs(seqs, 8, 2, torch.float16, seed=67)
    out = prompt_b200.kernel(**{k: torch.from_numpy(v) for k, v in inp.items()})
    assert not out.is_cuda
    _check(out, inp, seqs, torch.float16)


def test_page_ids_outside_the_pool_read_as_zeros():
    seqs = [(20, 200)]
    inp = _inputs(seqs, 8, 2, torch.float16, seed=73)
    kp, vp, table = op.to_pages(inp["k"], inp["v"], [200], 64, seed=1)
    table[0, 1] = 1 << 30
    d = _dev(inp, torch.float16)
    out = prompt_b200.kernel_paged(d["q"], torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), torch.from_numpy(table).cuda(),
                                   d["cu_q"], torch.tensor([200], dtype=torch.int32, device="cuda"), check=True)
    inp["k"][64:128], inp["v"][64:128] = 0, 0
    _check(out, inp, seqs, torch.float16)


@pytest.mark.parametrize("paged", [False, True], ids=["packed", "paged"])
@pytest.mark.parametrize("seqs", [[(17, 9001)], [(1, 5000), (3, 700), (2, 0), (5, 2048)], [(64, 1500)], [(40, 513)], [(9, 512), (9, 1024)]], ids=str)
def test_few_rows_over_many_keys_shared_by_several_ctas(seqs, paged):
    for dtype in (torch.float16, torch.bfloat16):
        inp = _inputs(seqs, 8, 2, dtype, seed=83)
        d = _dev(inp, dtype)
        if paged:
            nk = [m for _, m in seqs]
            kp, vp, table = op.to_pages(inp["k"].astype(np.float32), inp["v"].astype(np.float32), nk, 64, seed=4)
            out = prompt_b200.kernel_paged(d["q"], torch.from_numpy(kp).cuda().to(dtype), torch.from_numpy(vp).cuda().to(dtype), torch.from_numpy(table).cuda(),
                                           d["cu_q"], torch.tensor(nk, dtype=torch.int32, device="cuda"), check=True)
        else:
            out = prompt_b200.kernel(**d, check=True)
        _check(out, inp, seqs, dtype)
        if not paged:
            _check(prompt_b200.kernel(**d, causal=False, check=True), inp, seqs, dtype, causal=False)


def test_batch_invariant_mode_does_not_share():
    lib = _lib.lib()
    seqs = [(17, 9001)] + [(30, 30)] * 60
    inp = _inputs(seqs, 8, 2, torch.float16, seed=89)
    d = _dev(inp, torch.float16)
    lib.vmk_set_batch_invariant(1)
    try:
        whole = prompt_b200.kernel(**d, check=True)
        alone = prompt_b200.kernel(d["q"][:17], d["k"][:9001], d["v"][:9001], *(torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (17, 9001)))
        assert torch.equal(whole[:17], alone)
    finally:
        lib.vmk_set_batch_invariant(0)


def test_a_nan_key_in_one_share_reaches_every_row():
    inp = _inputs([(5, 6000)], 4, 2, torch.float16, seed=97)
    clean = prompt_b200.kernel(**_dev(inp, torch.float16))
    inp["k"][3000, 0] = np.nan
    out = prompt_b200.kernel(**_dev(inp, torch.float16), check=True)
    assert torch.isnan(out[:, :2]).all() and torch.equal(out[:, 2:], clean[:, 2:])


def test_sequences_that_overlap_are_reported_and_stay_inside_their_tensors():
    """More tiles than the rows of q come to: a list of lengths that goes up and down, long enough for the planner."""
    q = torch.randn(5000, 4, 128, device="cuda").half()
    k = torch.randn(5000, 1, 128, device="cuda").half()
    cu = torch.tensor([0, 5000] * 600 + [0], dtype=torch.int32, device="cuda")
    out = prompt_b200.kernel(q, k, k, cu)
    with pytest.raises(_lib.VmkDeviceStatusError) as e:
        check_status(out.device)
    assert e.value.status == 2 and out.shape == q.shape


@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1), (16, 1), (4, 4)])
def test_sequences_of_one_and_of_two_tiles_share_in_one_call(hq, hkv):
    """A sequence whose rows fit one 128-row tile has them in both, which take its blocks in turn; odd and even numbers of
    blocks to a share, shares of one block, NaN behind the last key."""
    tpt = 128 // (hq // hkv)
    for seqs in ([(tpt + 3, 2000), (tpt, 2000)], [(1, 513), (2 * tpt, 1153), (tpt - 1, 640)], [(3, 4096 + 65)], [(5, 1), (2, 1037)]):
        inp = _inputs(seqs, hq, hkv, torch.float16, seed=101, pad_q=3, pad_k=70, fill=np.nan)
        out = prompt_b200.kernel(**_dev(inp, torch.float16), check=True)
        n = sum(a for a, _ in seqs)
        assert (out[n:] == 0).all()
        inp = {**inp, "q": inp["q"][:n], "k": inp["k"][:sum(m for _, m in seqs)], "v": inp["v"][:sum(m for _, m in seqs)]}
        _check(out[:n], inp, seqs, torch.float16)


def test_a_short_list_that_does_not_ascend_is_reported():
    q = torch.randn(40, 8, 128, device="cuda").half()
    k = torch.randn(40, 2, 128, device="cuda").half()
    prompt_b200.kernel(q, k, k, torch.tensor([0, 10, 30, 40], dtype=torch.int32, device="cuda"), check=True)
    with pytest.raises(_lib.VmkDeviceStatusError) as e:
        prompt_b200.kernel(q, k, k, torch.tensor([0, 30, 10, 40], dtype=torch.int32, device="cuda"), check=True)
    assert e.value.status == 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("seqs", [[(300, 300)], [(40, 1100)], [(9, 1500), (70, 500)], [(513, 513)] * 3, [(100, 100)] * 40, [(5, 5)]], ids=str)
def test_special_values_in_v_reach_the_rows_that_see_them_and_no_other(seqs, dtype):
    """NaN in one column and infinity in another, at keys that rows before them share a block with: every other element
    keeps its bits, packed or paged, shared by several CTAs or not."""
    inp = _inputs(seqs, 8, 2, dtype, seed=103)
    d = _dev(inp, dtype)
    nk = [m for _, m in seqs]
    rng = np.random.default_rng(5)
    v, hit = inp["v"].copy(), []
    for s, (nq, m) in enumerate(seqs):
        for at in sorted({m - 1, m - 2, m - nq, int(rng.integers(m - nq, m)), int(rng.integers(0, m))}):
            col, head = int(rng.integers(0, 128)), int(rng.integers(0, 2))
            v[sum(nk[:s]) + at, head, col] = rng.choice([np.nan, np.inf, -np.inf])
            hit.append((s, at, head, col))

    def run(v):
        kp, vp, table = op.to_pages(inp["k"].astype(np.float32), np.asarray(v, dtype=np.float32), nk, 64, seed=4)
        paged = prompt_b200.kernel_paged(d["q"], torch.from_numpy(kp).cuda().to(dtype), torch.from_numpy(vp).cuda().to(dtype), torch.from_numpy(table).cuda(),
                                         d["cu_q"], torch.tensor(nk, dtype=torch.int32, device="cuda"), check=True)
        return prompt_b200.kernel(**{**d, "v": torch.from_numpy(np.ascontiguousarray(v)).cuda().to(dtype)}, check=True), paged

    clean, _ = run(inp["v"])
    for out in run(v):
        want = clean.float()
        for s, at, head, col in hit:
            nq, m = seqs[s]
            q0 = sum(n for n, _ in seqs[:s])
            first = max(0, at - (m - nq))
            want[q0 + first:q0 + nq, head * 4:head * 4 + 4, col] += float(v[sum(nk[:s]) + at, head, col])
        same = torch.isfinite(want)
        assert torch.equal(out.float()[same], want[same])
        assert (torch.isnan(out.float()[~same]) | (out.float()[~same] == want[~same])).all() and not torch.isfinite(out.float()[~same]).any()
