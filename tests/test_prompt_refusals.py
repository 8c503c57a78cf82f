"""What prompt attention refuses, without a GPU: the C entry points before any launch, the kernel module by its checks."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import ref64
from verified_metal_kernels_b200 import _lib, build
from verified_metal_kernels_b200.kernels import prompt_b200
from verified_metal_kernels_b200.ops import prompt as op


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _call(lib, q=256, k=256, v=256, cu_q=256, cu_k=256, strides=None, out=256, S=1, Tq=64, Tk=64, Hq=8, Hkv=2, D=128, causal=1,
          bf16=0, ws=256, ws_bytes=1 << 20, status=None):
    return lib.vmk_prompt(q, k, v, cu_q, cu_k, strides, out, S, Tq, Tk, Hq, Hkv, D, causal, bf16, ws, ws_bytes, status, None)


def test_c_entry_refuses_before_any_launch(lib):
    for name in ("q", "k", "v", "cu_q", "cu_k", "out", "ws"):
        assert _call(lib, **{name: None}) == -1, name
        assert _call(lib, **{name: 258 if not name.startswith("cu") else 257}) == -1, name
    assert _call(lib, status=2) == -1 and _call(lib, out=272) == -1
    for name in ("S", "Tq", "Tk"):
        assert _call(lib, **{name: -1}) == -1
    assert _call(lib, Hq=0) == -1 and _call(lib, Hkv=0) == -1 and _call(lib, bf16=2) == -1 and _call(lib, causal=5) == -1
    assert _call(lib, D=64) == -2 and _call(lib, Hq=9) == -2 and _call(lib, Hq=34) == -2
    assert _call(lib, ws_bytes=64) == -3
    assert _call(lib, Tq=2 ** 31 - 1) == -6 and _call(lib, Tk=2 ** 31 - 1) == -6
    assert _call(lib, Tq=0) == 0
    paged = lambda **kw: lib.vmk_prompt_paged(*[{**dict(q=256, k=256, v=256, table=256, pages=4, page_size=64, stride=2, cu_q=256, lens=256,
                                              strides=None, out=256, S=1, Tq=64, Hq=8, Hkv=2, D=128, causal=1, bf16=0, ws=256, wsb=1 << 20,
                                              status=None, stream=None), **kw}[n] for n in ("q", "k", "v", "table", "pages", "page_size", "stride",
                                              "cu_q", "lens", "strides", "out", "S", "Tq", "Hq", "Hkv", "D", "causal", "bf16", "ws", "wsb", "status", "stream")])
    for kw in (dict(table=None), dict(lens=None), dict(page_size=96), dict(page_size=0), dict(stride=0), dict(pages=-1), dict(k=None), dict(lens=257)):
        assert paged(**kw) == -1, kw
    assert paged(pages=2 ** 31 - 1) == -6


def test_workspace_sizes(lib):
    f = lib.vmk_prompt_workspace_bytes
    assert f(1, 128, 128, 32, 8, 128) >= 256 and f(0, 0, 0, 32, 8, 128) >= 256
    assert f(1, 128, 128, 32, 8, 64) == 0 and f(1, 128, 128, 33, 8, 128) == 0 and f(1, 128, 128, 34, 2, 128) == 0
    assert f(-1, 1, 1, 8, 8, 128) == 0 and f(1, 1, -1, 8, 8, 128) == 0
    assert f(1, 1 << 17, 1 << 17, 32, 8, 128) < 1 << 20
    assert 1 << 20 < f(1, 17, 1 << 20, 32, 8, 128) < 1 << 25             # few rows over many keys: the shares' partials


def test_module_refuses_by_its_checks(monkeypatch):
    """Everything that a wrong call can be refused for before the library is reached (the CUDA check is taken out)."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    q, k = torch.zeros(6, 4, 128, dtype=torch.float16), torch.zeros(6, 2, 128, dtype=torch.float16)
    cu = torch.zeros(2, dtype=torch.int32)
    bad = [(TypeError, dict(q=q.float())), (TypeError, dict(k=k.bfloat16())), (TypeError, dict(cu_q=cu.long())), (TypeError, dict(q=None)),
           (ValueError, dict(q=q[0])), (ValueError, dict(k=k[:, :, :64])), (ValueError, dict(v=k[:5])), (ValueError, dict(cu_q=cu[:0])),
           (ValueError, dict(cu_k=torch.zeros(3, dtype=torch.int32))),
           (ValueError, dict(q=torch.zeros(6, 4, 256, dtype=torch.float16)[:, :, ::2])),
           (ValueError, dict(k=torch.zeros(6, 2, 132, dtype=torch.float16)[:, :, :128])),
           (ValueError, dict(k=k[:1].expand(6, 2, 128))),
           (ValueError, dict(q=torch.zeros(6 * 4 * 128 + 8, dtype=torch.float16)[1:1 + 6 * 4 * 128].view(6, 4, 128)))]
    for err, kw in bad:
        with pytest.raises(err):
            prompt_b200.kernel(**{**dict(q=q, k=k, v=k, cu_q=cu), **kw})
    pool, table = torch.zeros(3, 2, 64, 128, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    lens = torch.zeros(1, dtype=torch.int32)
    for kw in (dict(k_pages=pool[:, :, :32].contiguous(), v_pages=pool[:, :, :32].contiguous()), dict(page_table=table[0]), dict(lens=lens[:0]),
               dict(v_pages=pool[:2]), dict(page_table=torch.zeros(2, 2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            prompt_b200.kernel_paged(**{**dict(q=q, k_pages=pool, v_pages=pool, page_table=table, cu_q=cu, lens=lens), **kw})


def test_cpu_tensors_need_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    inp = op.make_inputs([(4, 4)], 4, 2)
    with pytest.raises((RuntimeError, AssertionError)):
        prompt_b200.kernel(**{k: torch.from_numpy(v) for k, v in inp.items()})


def test_the_statement_is_that_of_the_tree_verification():
    """A chunk over a context is spec's chain: the last kd positions of a cache, causal among themselves."""
    from verified_metal_kernels_b200.ops import spec
    inp = spec.make_inputs(dict(B=1, L=40, k=8, Hq=4, Hkv=2), seed=1, dist="chain")
    want = ref64.spec_ref64(**inp)[0]
    out, _, _ = ref64.prompt_ref64(inp["q"][0], inp["k"][0].swapaxes(0, 1), inp["v"][0].swapaxes(0, 1), [8], [40])
    np.testing.assert_allclose(out, want, rtol=1e-12, atol=1e-12)


def test_pages_hold_what_the_packed_keys_hold():
    inp = op.make_inputs([(3, 100), (2, 0), (1, 64)], 4, 2, seed=2)
    kp, vp, table = op.to_pages(inp["k"], inp["v"], [100, 0, 64], 64)
    got = np.concatenate([kp[table[0, 0], :, :64], kp[table[0, 1], :, :36]], axis=1).swapaxes(0, 1)
    assert np.array_equal(got, inp["k"][:100]) and np.array_equal(vp[table[2, 0]].swapaxes(0, 1), inp["v"][100:])
    assert (table[1] == -1).all()
