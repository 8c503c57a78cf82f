"""Op definition of the acceptance of drafts (an extension: the reference verifies the drafts' attention, ops/spec.py; the
trees and their bits are that op's).  target_probs, draft_probs (B,kd,V), tokens (B,kd) int32, bits (B,kd[,W]) int32,
u (B,kd) float32."""
import numpy as np

from . import spec

NAME = "accept"
# (B, kd, V, max_depth: 0 a chain, draft probabilities or none, distribution)
FUZZ = [(1, 1, 5, 0, True, "near"), (3, 8, 1000, 0, True, "near"), (4, 31, 4097, 4, True, "near"), (2, 64, 9001, 3, True, "near"),
        (5, 33, 777, 2, True, "far"), (2, 128, 50021, 5, True, "near"), (6, 16, 2050, 2, True, "same"), (3, 12, 64, 2, True, "disjoint"),
        (1, 1, 1, 0, False, "near"), (7, 9, 1003, 0, False, "near"), (2, 70, 30011, 3, False, "near"), (40, 6, 257, 2, False, "repeated"),
        (9, 24, 513, 2, True, "repeated"), (150, 4, 8200, 0, True, "near")]


def make_inputs(B, kd, V, depth=0, with_draft=True, dist="near", seed=0, dtype=np.float32):
    """Seeded inputs: a target, a draft near it, tokens drawn from the draft's row of the parent.  "far": another draft;
    "same": the draft is the target (every drawn token stands); "disjoint": the two share no token; "repeated": siblings
    repeat tokens."""
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((B, kd, V)) * 2
    y = z + rng.standard_normal((B, kd, V)) * (0 if dist == "same" else 4 if dist == "far" else 0.7)
    p, q = np.exp(z), np.exp(y)
    if dist == "disjoint":
        p[..., ::2], q[..., 1::2] = 0, 0
    p, q = ((x / x.sum(-1, keepdims=True)).astype(dtype) for x in (p, q))
    masks = [spec.chain_bits(kd) if depth == 0 else spec.tree_bits(kd, rng, depth) for _ in range(B)]
    tokens = np.zeros((B, kd), dtype=np.int32)
    for b in range(B):
        for i in range(1, kd):
            par = (masks[b][i] & ((1 << i) - 1)).bit_length() - 1
            c = np.cumsum(q[b, max(par, 0)].astype(np.float64))
            x = int(np.searchsorted(c, rng.random() * c[-1], side="right"))
            tokens[b, i] = min(x, V - 1) if dist != "repeated" else min(x, V - 1) % 3
    u = rng.random((B, kd), dtype=np.float32)
    return dict(target_probs=p, tokens=tokens, bits=spec.pack_bits(masks, kd), u=u, draft_probs=q if with_draft else None)
