"""Kernel module for the acceptance of drafts on B200: which nodes of a speculative tree stand, and the token after them.

Not one of the reference's ops, which verify the attention of the drafts (reference ops/spec.py:14-25 builds the trees):
it is the step after `spec`, once the target's probabilities of every draft row are known."""
import torch

from .. import _lib
from ._common import calls, elsewhere, handles, need, need_on, stage_in

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def kernel(target_probs, tokens, bits, u, draft_probs=None, check=False):
    """target_probs (B,kd,V) fp32, fp16 or bf16, tokens (B,kd) int32, bits (B,kd) int32 -- or (B,kd,W) words for kd > 32 --
    as `spec` takes them, u (B,kd) float32 in [0, 1), draft_probs like target_probs or None -> (path (B,kd) int32, count
    (B,) int32, next_token (B,) int32).

    Node 0 is the root: the token that is decided already.  Node i's parent is the highest node below i in bits[i].  Row c
    of target_probs is the target's distribution after node c, row c of draft_probs the one that the children of c were
    drawn from, each by itself; draft_probs=None: the drafts were chosen, not drawn (looked up, or the likeliest).  A
    node's children are tried in ascending order, child i with the number u[:, i]; u[:, 0] draws the next token, from
    what is left of the target where the walk ends.  The tokens that come out are distributed as the target's own.

    path: the accepted nodes in order (path[:, 0] = 0), -1 behind them; count: how many.  Differences are
    pairs of fp32 numbers, sums fp64 (include/vmk_b200.h has the bound of what that is off by).  Entries that are NaN,
    infinite or negative count as 0; a row of nothing but those gives next_token -1.  A draft token outside [0, V) is refused
    (and reported in the device status word).  Host tensors are copied in and the results returned on the host."""
    if not check:
        out = calls().accept(target_probs, tokens, bits, u, draft_probs)
        if out is not None:
            return out
    (target_probs, tokens, bits, u, draft_probs), host = stage_in([target_probs, tokens, bits, u, draft_probs])
    if not isinstance(target_probs, torch.Tensor) or target_probs.dtype not in DTYPES:
        raise TypeError("target_probs: expected a float32, float16 or bfloat16 tensor")
    dt = target_probs.dtype
    need(target_probs, "target_probs", dt, dims=3)
    B, kd, V = target_probs.shape
    dev = target_probs.device
    need_on(tokens, "tokens", torch.int32, (B, kd), dev)
    if not isinstance(bits, torch.Tensor) or bits.dtype != torch.int32:
        raise TypeError("bits: expected an int32 tensor")
    words = 1 if bits.dim() == 2 else bits.shape[2] if bits.dim() == 3 else 0
    need_on(bits, "bits", torch.int32, (B, kd) if bits.dim() == 2 else (B, kd, words), dev)
    need_on(u, "u", torch.float32, (B, kd), dev)
    if draft_probs is not None:
        need_on(draft_probs, "draft_probs", dt, (B, kd, V), dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return kernel(target_probs, tokens, bits, u, draft_probs, check)
    stream, status = handles(dev)
    path, count, token = torch.empty_like(tokens), tokens.new_empty(B), tokens.new_empty(B)
    rc = lib.vmk_accept(target_probs.data_ptr(), _lib.ptr(draft_probs), tokens.data_ptr(), bits.data_ptr(), words, u.data_ptr(),
                        path.data_ptr(), count.data_ptr(), token.data_ptr(), B, kd, V, DTYPES[dt],
                        status, stream)
    _lib.check(rc, "vmk_accept")
    if host:
        path, count, token = path.cpu(), count.cpu(), token.cpu()
    if host or check:
        _lib.raise_on_status(dev, "vmk_accept")
    return path, count, token
