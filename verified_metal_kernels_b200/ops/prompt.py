"""Op definition of prompt attention (an extension: the reference's ops decode; head counts follow them, ops/spec.py:9).
q (Tq,Hq,D), k/v (Tk,Hkv,D) fp16 packed by cu_q, cu_k (S+1,) int32; query i of a sequence with nq queries and nk keys
sees its keys j <= nk - nq + i."""
import numpy as np

NAME = "prompt"
HQ, HKV, D = 32, 8, 128
# (queries and keys of each sequence, query heads, kv heads, distribution).  Lengths around the tiles (128 keys, and
# 128 // group tokens to a tile), of zero and one, more queries than keys (rows that see nothing), contexts.
FUZZ = [([(1, 1)], 32, 8, "randn"), ([(128, 128)], 8, 2, "randn"), ([(129, 129), (31, 31), (64, 64), (1, 1)], 8, 2, "randn"),
        ([(0, 0), (33, 33), (0, 0), (257, 257), (0, 0)], 4, 1, "randn"), ([(5, 0), (40, 7), (3, 130), (200, 128)], 4, 2, "randn"),
        ([(1, 700), (17, 500), (70, 900)], 8, 1, "randn"), ([(150, 150), (43, 300)], 3, 1, "randn"), ([(90, 90)], 10, 2, "large"),
        ([(300, 300)], 1, 1, "randn"), ([(20, 20), (45, 400)], 16, 1, "large"), ([(130, 260)], 7, 7, "tiny"),
        ([(60, 60)] * 9, 4, 4, "randn"), ([(37, 37 + 64 * i) for i in range(6)], 12, 1, "randn")]


def make_inputs(seqs, hq, hkv, seed=0, dist="randn", pad_q=0, pad_k=0, fill=0.0):
    """Seeded inputs for sequences of (queries, keys); pad_q rows of queries and pad_k keys (holding `fill`) behind the
    last sequence.  "large" multiplies q and k by 4, "tiny" scales everything down."""
    rng = np.random.default_rng(seed)
    tq, tk = sum(n for n, _ in seqs), sum(m for _, m in seqs)
    q = rng.standard_normal((tq + pad_q, hq, D), dtype=np.float32)
    k = rng.standard_normal((tk + pad_k, hkv, D), dtype=np.float32)
    v = rng.standard_normal((tk + pad_k, hkv, D), dtype=np.float32)
    if dist == "large":
        q, k = q * 4.0, k * 4.0
    elif dist == "tiny":
        q, k, v = q * 1e-3, k * 1e-3, v * 1e-2
    elif dist != "randn":
        raise ValueError(f"unknown dist {dist!r}")
    k[tk:], v[tk:] = fill, fill
    cu = lambda c: np.concatenate([[0], np.cumsum([s[c] for s in seqs])]).astype(np.int32)
    return dict(q=q.astype(np.float16), k=k.astype(np.float16), v=v.astype(np.float16), cu_q=cu(0), cu_k=cu(1))


def to_pages(k, v, nk, page_size, seed=0, spare=3, fill=np.nan):
    """Scatters packed keys (nk[s] of each sequence) into a shuffled page pool: (k_pages, v_pages
    (pages,Hkv,page_size,D), page_table (S,T) int32, -1 where a sequence has no page)."""
    hkv, d = k.shape[1], k.shape[2]
    need = [-(-int(n) // page_size) for n in nk]
    pages = sum(need) + spare
    ids = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    kp = np.full((pages, hkv, page_size, d), fill, dtype=k.dtype)
    vp = np.full((pages, hkv, page_size, d), fill, dtype=v.dtype)
    table = np.full((len(nk), max(1, max(need, default=1))), -1, dtype=np.int32)
    at = used = 0
    for s, n in enumerate(nk):
        for i in range(need[s]):
            pg, c = ids[used], min(page_size, int(n) - i * page_size)
            used += 1
            table[s, i] = pg
            kp[pg, :, :c] = k[at + i * page_size:at + i * page_size + c].swapaxes(0, 1)
            vp[pg, :, :c] = v[at + i * page_size:at + i * page_size + c].swapaxes(0, 1)
        at += int(n)
    return kp, vp, table


def flops(seqs, hq):
    """Floating-point operations of the two products over the visible pairs."""
    return 4.0 * D * hq * sum(sum(min(m, max(0, m - n + i + 1)) for i in range(n)) for n, m in seqs)
