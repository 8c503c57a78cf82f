"""Scratch of a captured call is the graph's own: it is not the stream's, which a larger call replaces and other graphs use."""
import pytest
import torch

from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import decode_b200, spec_b200
from verified_metal_kernels_b200.ops import load_op, to_torch


def test_not_kept_under_capture(monkeypatch):
    cpu = torch.device("cpu")
    monkeypatch.setattr(_lib, "_workspace", _lib.Workspace())
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    eager = _lib.workspace(1000, cpu, 5)
    assert _lib.workspace(500, cpu, 5) is eager
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True, raising=False)
    a, b = _lib.workspace(500, cpu, 5), _lib.workspace(500, cpu, 5)
    assert len({x.data_ptr() for x in (eager, a, b)}) == 3 and a.numel() >= 500
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    assert _lib.workspace(500, cpu, 5) is eager


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "spec"])
def test_a_replay_after_a_larger_call_writes_into_nobody_elses_memory(which):
    """Split calls, whose partials go through the scratch: captured, then a larger eager call on the same stream, then tensors in
    whatever memory is free."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device="cuda").manual_seed(3)
    half = lambda *s: torch.randn(*s, generator=g, device=dev).half()

    def call(B, L):
        if which == "decode":
            q, k, v = half(B, 32, 128), half(B, 8, L, 128), half(B, 8, L, 128)
            lens = torch.full((B,), L, dtype=torch.int32, device=dev)
            return lambda: decode_b200.kernel(q, k, v, lens)
        inp = to_torch(load_op("spec").make_inputs(dict(B=B, L=L, k=8), seed=B), "cuda")
        return lambda: spec_b200.kernel(**inp)

    small, large = call(1, 8000), call(8, 16000)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = small()
    st.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            graphs.append((gr, small()))
    with torch.cuda.stream(st):
        big = large()
        others = [torch.full((n,), 7, dtype=torch.uint8, device=dev) for n in (1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 21, 1 << 22) for _ in range(4)]
    st.synchronize()
    lone = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (gr, _) in zip(lone, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs)
    assert all(bool((x == 7).all()) for x in others)
    with torch.cuda.stream(st):
        assert torch.equal(large(), big)
    assert _lib.read_status(dev) == 0
