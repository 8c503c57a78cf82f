"""Acceptance where the draft is nearly the target and several children are refused: what is left of the target is then small
against the numbers that it is the difference of.  The answers have to be those of the statement wherever its comparisons
are further from their border than the kernel's arithmetic can be off.

The bound, at a node's k-th refusal, of what the sum M of the residual is off by (sum of p = 1, n entries to a thread): an
entry's difference p - S q is a pair of fp32 numbers whose smaller one is off by less than 3 x 2^-47 of p (its two roundings,
and S to 49 bits), the smaller ones are summed in fp32 (n additions of 2^-24 each, of numbers below 2^-22 of p): less than
(2 n + 3) 2^-47 in all.  S is the sum of the Ms before, and an error of S moves the next M by as much at most: so it
doubles with every refusal, d_k = 2^k (2 n + 3) 2^-47."""
import numpy as np
import pytest
import torch

from verified_metal_kernels_b200.kernels import accept_b200

KD = 7


def _inputs(V, eps, B, seed):
    """One root with six children.  The first token lies where the draft is above the target and has a number near 1: refused."""
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((B, KD, V)) * 2
    p, q = np.exp(z), np.exp(z + eps * rng.standard_normal((B, KD, V)))
    p, q = ((x / x.sum(-1, keepdims=True)).astype(np.float32) for x in (p, q))
    tokens, u = rng.integers(0, V, (B, KD)).astype(np.int32), rng.random((B, KD), dtype=np.float32)
    for b in range(B):
        ratio = q[b, 0].astype(np.float64) / p[b, 0]
        tokens[b, 1:4] = rng.permutation(np.nonzero(ratio > 1 + eps / 2)[0])[:3]
    u[:, 1] = 1 - 2.0 ** -24
    bits = np.tile(np.array([1] + [1 | 1 << i for i in range(1, KD)], dtype=np.int32), (B, 1))
    return dict(target_probs=p, draft_probs=q, tokens=tokens, u=u, bits=bits)


def _statement(inp, b, n):
    """(path, count, next) of request b in long doubles, how many children were refused, and whether every comparison is clear of its border."""
    p, q = (inp[k][b].astype(np.longdouble) for k in ("target_probs", "draft_probs"))
    u = inp["u"][b].astype(np.longdouble)
    S, M, off, clear, at, path, refused = np.longdouble(0), np.longdouble(1), np.longdouble(0), True, 0, [0], 0
    left = p[0]
    for i in range(1, KD):
        x = inp["tokens"][b, i]
        r, bar = p[0, x] - S * q[0, x], u[i] * M * q[0, x]
        clear &= bool(abs(bar - r) > 2 * off * q[0, x] + 2.0 ** -50 * p[0, x])
        if r > 0 and bar < r:
            at, left = i, p[i]
            path.append(i)
            break
        refused += 1
        S += M
        left = np.maximum(p[0] - S * q[0], 0)
        M = left.sum()
        off = 2.0 ** refused * (2 * n + 3) * 2.0 ** -47
    if at:
        off = np.longdouble(2.0 ** -50) * p.shape[1]
    c = left.cumsum()
    nxt = int(np.nonzero((c > u[0] * c[-1]) & (left > 0))[0][0])
    clear &= bool(np.abs(c - u[0] * c[-1]).min() > 2 * off)
    return path + [-1] * (KD - len(path)), len(path), nxt, refused, clear


# (a thread's entries: 512 threads a CTA, 8 CTAs from 32768 entries and 1 below 8192, by vectors of 4)
CASES = [(32768, 1e-2, 8 + 4), (32768, 1e-4, 8 + 4), (2048, 1e-6, 4 + 4)]


@pytest.mark.parametrize("V,eps,n", CASES, ids=str)
def test_the_statement_decides(V, eps, n):
    """The cases are worth something: several refusals, and most requests clear of their borders."""
    inp = _inputs(V, eps, 24, seed=5)
    got = [_statement(inp, b, n) for b in range(24)]
    assert np.mean([g[4] for g in got]) > 0.6 and sum(g[3] >= 3 for g in got) > 12


@pytest.mark.gpu
@pytest.mark.parametrize("V,eps,n", CASES, ids=str)
def test_a_draft_that_is_nearly_the_target(V, eps, n):
    inp = _inputs(V, eps, 24, seed=5)
    path, count, nxt = (x.cpu() for x in accept_b200.kernel(**{k: torch.from_numpy(v).cuda() for k, v in inp.items()}, check=True))
    for b in range(24):
        want = _statement(inp, b, n)
        if want[4]:
            assert (path[b].tolist(), int(count[b]), int(nxt[b])) == (want[0], want[1], want[2]), b
