"""The serving operators around the paged cache and the decode kernels, and what is measured of them:

    prompt   attention of whole prompts, or of chunks of prompts over a cache: packed sequences of different lengths,
             causal, grouped heads, contiguous keys or a paged cache
    accept   which drafts of a speculative tree stand, and the token after them, from given random numbers
    pages    the cache's pages: reserving, filling, copying, forking, compacting after a verification, freeing

`own` False computes the plain forms in torch, True calls the package."""
import math

import numpy as np
import torch

own = False

D = 128
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one short prompt: nothing but latency
        dict(name="prompt one short", op="prompt", seqs=1, new=128, context=0, ragged=False, heads=32, kv_heads=8, type="fp16", paged=0),
        # a batch of prompts of very different lengths, as admitted together
        dict(name="prompt ragged batch", op="prompt", seqs=24, new=1999, context=0, ragged=True, heads=32, kv_heads=8, type="bf16", paged=0),
        # one long document: bound by the tensor cores
        dict(name="prompt long", op="prompt", seqs=1, new=32768, context=0, ragged=False, heads=32, kv_heads=8, type="bf16", paged=0),
        # chunked prefill: each request adds a chunk to what its pages hold already
        dict(name="prompt chunks paged", op="prompt", seqs=8, new=512, context=16000, ragged=True, heads=64, kv_heads=8, type="fp16", paged=64),
        # a short turn on a long conversation: few rows, many keys
        dict(name="prompt short turn", op="prompt", seqs=1, new=17, context=60001, ragged=False, heads=32, kv_heads=8, type="bf16", paged=256),
        # one request's chain of drafts: nothing but latency
        dict(name="accept chain", op="accept", batch=1, drafts=8, depth=0, vocab=32768, type="fp32", draft_probs=True),
        # a batch of draft trees over a large vocabulary
        dict(name="accept trees", op="accept", batch=32, drafts=64, depth=8, vocab=131072, type="fp32", draft_probs=True),
        # drafts looked up in the text instead of drawn from a model; odd rows of 16-bit probabilities
        dict(name="accept lookup drafts", op="accept", batch=128, drafts=8, depth=0, vocab=100003, type="bf16", draft_probs=False),
        # pages moved inside the pools of all layers
        dict(name="pages copy", op="copy", pages=600, moved=256, layers=8, kv_heads=8, page=64, type="fp16"),
        # finished requests leave, prompts of different lengths enter
        dict(name="pages admit", op="admit", rows=48, longest=1500, kv_heads=8, page=64, type="bf16"),
        # every request goes on in several samples: tables shared, the last page copied
        dict(name="pages fork", op="fork", rows=32, children=4, longest=4000, layers=8, kv_heads=8, page=64, type="fp16"),
        # after a verification: the accepted drafts close up in the cache, the rest of the tail is given back
        dict(name="pages compact", op="compact", rows=64, drafts=32, longest=2000, kv_heads=8, page=64, type="fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "accept", "accept", "copy", "admit", "fork", "compact"])
    two = rng.choice(["fp16", "bf16"])
    page = rng.choice([64, 128, 256])
    if op == "prompt":
        heads, kv_heads = rng.choice([(32, 8), (32, 4), (8, 8), (16, 1), (40, 8), (24, 8), (64, 8), (7, 1), (28, 4)])
        seqs = _log(rng, 1, 64)
        paged = rng.choice([0, 0, page])
        new = _log(rng, 1, 16384 if not paged else 4096)
        context = rng.choice([0, _log(rng, 1, 60000)]) if paged else 0
        while seqs * (new + context) > 200000:
            seqs = (seqs + 1) // 2 if seqs > 1 else 1
            new, context = max(1, new // 2), context // 2
        while 4.0 * D * heads * seqs * new * (new / 2 + context) > 8e12:
            new = max(1, new // 2)
        return dict(op=op, seqs=seqs, new=new, context=context, ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads, type=two, paged=paged)
    if op == "accept":
        vocab = _log(rng, 999, 131072)
        drafts = rng.choice([1, 2, 5, 8, 16, 31, 48, 64])
        batch = _log(rng, 1, 128)
        while batch * drafts * vocab > 32 * 64 * 131072:
            batch = (batch + 1) // 2
        return dict(op=op, batch=batch, drafts=drafts, depth=rng.choice([0, 0, 4, 8]), vocab=vocab, type=rng.choice(["fp32", "fp32", "bf16", "fp16"]), draft_probs=rng.random() < 0.6)
    layers, kv_heads = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 5, 8])
    if op == "copy":
        moved = _log(rng, 1, 256)
        return dict(op=op, pages=2 * moved + rng.randrange(100), moved=moved, layers=layers, kv_heads=kv_heads, page=page, type=two)
    rows = _log(rng, 1, 64)
    if op == "admit":
        return dict(op=op, rows=rows, longest=_log(rng, 1, 1500), kv_heads=kv_heads, page=page, type=two)
    if op == "fork":
        return dict(op=op, rows=max(1, rows // 2), children=rng.randrange(1, 6), longest=_log(rng, 1, 4000), layers=layers, kv_heads=kv_heads, page=page, type=two)
    return dict(op=op, rows=rows, drafts=rng.choice([1, 3, 8, 16, 32, 60]), longest=_log(rng, 1, 2000), kv_heads=kv_heads, page=page, type=two)


def _lengths(case):
    """Each sequence's new tokens and its keys: a function of the case alone, so that work() knows them."""
    rng = np.random.default_rng([case["seqs"], case["new"], case["context"]])
    s = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * s, [case["new"] + case["context"]] * s
    new = rng.integers(1, case["new"] + 1, s)
    new[0] = case["new"]
    return new.tolist(), (new + (rng.integers(0, case["context"] + 1, s) if case["context"] else 0)).tolist()


def _row_lengths(case):
    """The lengths of the cache's rows, as _lengths."""
    n = np.random.default_rng([case["rows"], case["longest"]]).integers(1, case["longest"] + 1, case["rows"])
    n[0] = case["longest"]
    return n.tolist()


def _counts(case):
    """How many drafts each row accepts (the root among them)."""
    return np.random.default_rng([case["rows"], case["drafts"], 5]).integers(1, min(case["drafts"], 8) + 1, case["rows"]).tolist()


def work(case):
    op = case["op"]
    if op == "prompt":
        new, keys = _lengths(case)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
        return {"bytes": 2 * D * (2 * sum(new) * case["heads"] + 2 * sum(keys) * case["kv_heads"]), "flops": 4.0 * D * case["heads"] * pairs}
    if op == "accept":
        size, rows = (4 if case["type"] == "fp32" else 2), 2 if case["draft_probs"] else 1
        return {"bytes": case["batch"] * (rows * size * (case["vocab"] + case["drafts"]) + 20 * case["drafts"] + 8),
                "flops": 4.0 * case["batch"] * case["vocab"]}
    row = 2 * 2 * case["kv_heads"] * D * case.get("layers", 1)          # K and V of one position
    if op == "copy":
        return {"bytes": 2 * row * case["page"] * case["moved"], "flops": 0}
    lens = _row_lengths(case)
    if op == "admit":
        return {"bytes": 2 * row * sum(lens) + 8 * sum(-(-n // case["page"]) for n in lens), "flops": 0}
    if op == "fork":
        return {"bytes": 2 * row * case["children"] * sum(n % case["page"] for n in lens)
                + 16 * case["children"] * sum(-(-n // case["page"]) for n in lens), "flops": 0}
    return {"bytes": 2 * row * (case["drafts"] * case["rows"] + sum(_counts(case))), "flops": 0}


# ------------------------------------------------------------------------------------------------ their inputs
def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return [0] + np.cumsum(lengths).tolist()


def _table(lens, page, width, pages, seed):
    """A page table of scattered pages for rows of these lengths, -1 where there is none."""
    table = np.full((len(lens), width), -1, dtype=np.int32)
    ids, at = np.random.default_rng(seed).permutation(pages).astype(np.int32), 0
    for r, n in enumerate(lens):
        c = -(-n // page)
        table[r, :c] = ids[at:at + c]
        at += c
    return table


def _tree(rng, drafts, depth):
    """Parents (-1 for the root) and each node's ancestors-or-itself as words of 32 bits; depth 0 is a chain."""
    parents, level, masks = [-1], [0], [1]
    for i in range(1, drafts):
        ok = [j for j in range(i) if level[j] < depth - 1]
        p = i - 1 if depth == 0 else ok[int(rng.integers(max(0, len(ok) - 12), len(ok)))]
        parents.append(p)
        level.append(level[p] + 1)
        masks.append(masks[p] | 1 << i)
    words = (drafts + 31) // 32
    bits = np.array([[m >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in masks], dtype=np.uint32).view(np.int32)
    return parents, bits[:, 0] if words == 1 else bits


def _prepare_prompt(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, h, hk, page = TYPES[case["type"]], case["heads"], case["kv_heads"], case["paged"]
    new, keys = _lengths(case)
    s = dict(op="prompt", new=new, keys=keys, page=page, q=_randn(g, (sum(new), h, D), t), cu_q=_ints(_starts(new)))
    if not page:
        s.update(k=_randn(g, (sum(keys), hk, D), t), v=_randn(g, (sum(keys), hk, D), t))
        return s
    width = max(-(-n // page) for n in keys)
    pages = sum(-(-n // page) for n in keys) + 3
    table = _table(keys, page, width, pages, seed)
    s.update(k=_randn(g, (pages, hk, page, D), t), v=_randn(g, (pages, hk, page, D), t), table=_ints(table.tolist()), lens=_ints(keys))
    return s


def _prepare_accept(case, seed):
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    b, n, v, t = case["batch"], case["drafts"], case["vocab"], TYPES[case["type"]]
    trees = [_tree(rng, n, case["depth"]) for _ in range(b)]
    parents = torch.tensor([p for p, _ in trees], device="cuda").clamp(min=0)
    at = torch.arange(b, device="cuda")[:, None]
    target = torch.empty(b, n, v, dtype=t, device="cuda")
    draft = torch.empty(b, n, v, dtype=t, device="cuda") if case["draft_probs"] else None
    tokens = torch.empty(b, n, dtype=torch.int64, device="cuda")
    for i in range(b):                       # a draft model that is near the target, tokens drawn from it
        z = torch.randn(n, v, generator=g, device="cuda") * 2.5
        target[i] = torch.softmax(z, -1).to(t)
        near = torch.softmax(z + torch.randn(n, v, generator=g, device="cuda") * 0.7, -1).to(t)
        if draft is not None:
            draft[i] = near
        c = near.double().cumsum(-1)[parents[i]]
        u = torch.rand(n, 1, generator=g, device="cuda", dtype=torch.float64) * c[:, -1:]
        tokens[i] = torch.searchsorted(c, u, right=True)[:, 0].clamp(max=v - 1)
    if draft is None:                        # looked-up drafts: every other one is what the target would most likely say
        likely = target.float().argmax(-1)[at, parents]
        tokens = torch.where(torch.rand(b, n, generator=g, device="cuda") < 0.7, likely, tokens)
    u = torch.rand(b, n, generator=g, device="cuda")
    return dict(op="accept", target=target, draft=draft, tokens=tokens.int(), bits=torch.from_numpy(np.stack([w for _, w in trees])).cuda(), u=u)


def _prepare_pages(case, seed):
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    t, hk, page, op = TYPES[case["type"]], case["kv_heads"], case["page"], case["op"]
    if op == "copy":
        shape = (case["layers"], case["pages"], hk, page, D)
        ids = rng.permutation(case["pages"])[:2 * case["moved"]].tolist()
        return dict(op=op, pools=[_randn(g, shape, t), _randn(g, shape, t)], src=_ints(ids[::2]), dst=_ints(ids[1::2]))
    lens = _row_lengths(case)
    used = [-(-n // page) for n in lens]
    if op == "fork":
        c, r = case["children"], case["rows"]
        pages = sum(used) + r * c + 7
        table = np.full((r * (1 + c), max(used)), -1, dtype=np.int32)
        table[:r] = _table(lens, page, max(used), pages, seed)
        order = rng.permutation(r * c)
        refs = np.zeros(pages, dtype=np.int64)
        np.add.at(refs, table[table >= 0], 1)
        shape = (case["layers"], pages, hk, page, D)
        return dict(op=op, pools=[_randn(g, shape, t), _randn(g, shape, t)], table=_ints(table.tolist()), lens=_ints(lens + [0] * (r * c)), refs=_ints(refs.tolist()),
                    parents=_ints((order // c).tolist()), children=_ints((r + order).tolist()), keep=_ints(lens + [0] * (r * c)), page=page)
    extra = [case["drafts"]] * case["rows"] if op == "compact" else lens
    base = lens if op == "compact" else [0] * case["rows"]
    width = max(-(-(b + e) // page) for b, e in zip(base, extra))
    pages = sum(-(-(b + e) // page) for b, e in zip(base, extra)) + 7
    table = _table(base, page, width, pages, seed)
    refs = np.zeros(pages, dtype=np.int64)
    np.add.at(refs, table[table >= 0], 1)
    s = dict(op=op, pools=[_randn(g, (pages, hk, page, D), t), _randn(g, (pages, hk, page, D), t)], table=_ints(table.tolist()), lens=_ints(base), refs=_ints(refs.tolist()),
             keep=_ints(base), extra=_ints(extra), page=page, k=_randn(g, (sum(extra), hk, D), t), v=_randn(g, (sum(extra), hk, D), t), cu=_ints(_starts(extra)))
    if op == "compact":
        path = np.full((case["rows"], case["drafts"]), -1, dtype=np.int64)
        for r, n in enumerate(_counts(case)):
            path[r, 1:n] = 1 + np.sort(rng.permutation(case["drafts"] - 1)[:n - 1])
            path[r, 0] = 0
        s.update(path=_ints(path.tolist()), count=_ints(_counts(case)))
    return s


def prepare(case, seed):
    return {"prompt": _prepare_prompt, "accept": _prepare_accept}.get(case["op"], _prepare_pages)(case, seed)


# ------------------------------------------------------------------------------------------------ plain forms
def _attend(q, k, v, first):
    """q (n,H,G,D), k and v (keys,H,D): row i sees keys up to first + i."""
    n, h, grp, _ = q.shape
    kt, vt = k.float().permute(1, 2, 0), v.float().permute(1, 0, 2)
    out = torch.empty(n, h, grp, D, dtype=q.dtype, device=q.device)
    step = max(1, int(2.5e8 / (h * grp * k.shape[0])))          # rows at a time, so that the scores stay near 1 GB
    for a in range(0, n, step):
        z = min(n, a + step)
        seen = min(k.shape[0], first + z)
        s = torch.matmul(q[a:z].float().permute(1, 0, 2, 3).reshape(h, -1, D), kt[:, :, :seen]) * (1 / math.sqrt(D))
        hidden = torch.arange(seen, device=q.device) > first + torch.arange(a, z, device=q.device).repeat_interleave(grp)[:, None]
        s.masked_fill_(hidden, float("-inf"))
        p = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
        o = torch.matmul(p, vt[:, :seen]) / p.sum(-1, keepdim=True)
        out[a:z] = o.reshape(h, z - a, grp, D).permute(1, 0, 2, 3).to(q.dtype)
    return out.reshape(n, h * grp, D)


def _plain_prompt(s):
    q, hk = s["q"], s["k"].shape[1]
    cq, ck = _starts(s["new"]), _starts(s["keys"])
    outs = []
    for i, (n, keys) in enumerate(zip(s["new"], s["keys"])):
        if s["page"]:
            ids = s["table"][i, :-(-keys // s["page"])].long()
            k, v = (x[ids].transpose(1, 2).reshape(-1, hk, D)[:keys] for x in (s["k"], s["v"]))
        else:
            k, v = s["k"][ck[i]:ck[i + 1]], s["v"][ck[i]:ck[i + 1]]
        outs.append(_attend(q[cq[i]:cq[i + 1]].reshape(n, hk, -1, D), k, v, keys - n))
    return torch.cat(outs)


def _plain_accept(s):
    target, draft, u = s["target"], s["draft"], s["u"].double()
    b, n, v = target.shape
    dev = target.device
    at = torch.arange(b, device=dev)
    node = torch.arange(n, device=dev)
    words = s["bits"].reshape(b, n, -1)
    seen = (words[:, :, node // 32] >> (node % 32)) & 1                       # (b, node, ancestor or itself)
    parent = (seen * (node < node[:, None]) * (node + 1)).amax(-1) - 1        # -1: no ancestor
    cur = torch.zeros(b, dtype=torch.int64, device=dev)
    path = torch.full((b, n), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    count = torch.ones(b, dtype=torch.int64, device=dev)
    taken = torch.zeros(b, dtype=torch.float64, device=dev)                   # S: how often q has been taken off
    mass = torch.ones(b, dtype=torch.float64, device=dev)                     # M: what is left
    gone = torch.zeros(b, v, dtype=torch.bool, device=dev)                    # without q: the tokens refused so far
    for i in range(1, n):
        here = parent[:, i] == cur
        x = s["tokens"][:, i].long()
        p = target[at, cur, x].double()
        if draft is not None:
            q = draft[at, cur, x].double()
            r = (p - taken * q).clamp(min=0)
            yes = here & (r > 0) & (u[:, i] * mass * q < r)
        else:
            r = torch.where(gone[at, x], 0.0, p)
            yes = here & (r > 0) & (u[:, i] * mass < r)
        no = here & ~yes
        if draft is not None:
            taken = torch.where(no, taken + mass, taken)
            left = (target[at, cur].double() - taken[:, None] * draft[at, cur].double()).clamp_(min=0).sum(-1)
            mass = torch.where(no, left, mass)
        else:
            mass = torch.where(no, (mass - r).clamp(min=0), mass)
            gone[at, x] |= no
        path[at, count.clamp(max=n - 1)] = torch.where(yes, i, path[at, count.clamp(max=n - 1)]).int()
        count += yes
        cur = torch.where(yes, i, cur)
        taken, mass = torch.where(yes, 0.0, taken), torch.where(yes, 1.0, mass)
        gone &= ~yes[:, None]
    w = target[at, cur].double()
    rest = (w - taken[:, None] * draft[at, cur].double()).clamp(min=0) if draft is not None else torch.where(gone, 0.0, w)
    w = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    c = w.cumsum(-1)
    token = ((c > u[:, :1] * c[:, -1:]) & (w > 0)).int().argmax(-1)
    return path, count.int(), torch.where(c[:, -1] > 0, token, -1).int()


def _grant(refs, need):
    """The lowest free pages for those who need them, in their order: (where each one's begin, the free pages' ids, who is served)."""
    free = torch.argsort((refs != 0).int(), stable=True)
    end = need.cumsum(0)
    return end - need, free, (need == 0) | (end <= (refs == 0).sum())


def _plain_free(s, keep):
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
    slot = torch.arange(table.shape[1], device=table.device)
    kept = torch.minimum(lens, keep)
    out = (slot >= ((kept + page - 1) // page)[:, None]) & (slot < ((lens + page - 1) // page)[:, None])
    refs.index_add_(0, table.clamp(min=0).reshape(-1), -out.int().reshape(-1))
    table.masked_fill_(out, -1)
    lens.copy_(kept)


def _plain_reserve(s, extra):
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
    have, want = (lens + page - 1) // page, (lens + extra + page - 1) // page
    start, free, ok = _grant(refs, want - have)
    slot = torch.arange(table.shape[1], device=table.device)
    new = (slot >= have[:, None]) & (slot < want[:, None]) & ok[:, None]
    ids = free[(start[:, None] + slot - have[:, None]).clamp(0, refs.numel() - 1)]
    table.copy_(torch.where(new, ids, table))
    refs.index_add_(0, ids.reshape(-1), new.int().reshape(-1))
    lens.copy_(torch.where(ok, lens + extra, lens))


def _plain_append(s):
    table, lens, cu, page = s["table"], s["lens"].long(), s["cu"].long(), s["page"]
    t = torch.arange(s["k"].shape[0], device=table.device)
    row = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[row] - (cu[row + 1] - t)
    where = table[row, pos // page].long()
    s["pools"][0][where, :, pos % page] = s["k"]
    s["pools"][1][where, :, pos % page] = s["v"]


def _plain_fork(s):
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
    par, child = s["parents"].long(), s["children"].long()
    n = lens[par]
    full, rest = n // page, n % page
    start, free, ok = _grant(refs, (rest > 0).int())
    new = free[start.clamp(max=refs.numel() - 1)]
    slot = torch.arange(table.shape[1], device=table.device)
    old = table[par]
    shared = (slot < full[:, None]) & ok[:, None]
    own_page = (slot == full[:, None]) & (rest > 0)[:, None] & ok[:, None]
    table[child] = torch.where(shared, old, torch.where(own_page, new[:, None].int(), -1))
    refs.index_add_(0, old.clamp(min=0).reshape(-1), shared.int().reshape(-1))
    refs.index_add_(0, new, (ok & (rest > 0)).int())
    lens[child] = torch.where(ok, n, 0)
    last = old.gather(1, full.clamp(max=table.shape[1] - 1).long()[:, None])[:, 0].clamp(min=0).long()
    copied = ok[:, None] & (torch.arange(page, device=table.device) < rest[:, None])
    f, i = copied.nonzero(as_tuple=True)
    for pool in s["pools"]:
        pool[:, new[f], :, i] = pool[:, last[f], :, i]


def _plain_compact(s):
    table, page = s["table"], s["page"]
    base = s["lens"] - s["path"].shape[1]
    r, j = (torch.arange(s["path"].shape[1], device=table.device) < s["count"][:, None]).nonzero(as_tuple=True)
    src, dst = (base[r] + s["path"][r, j]).long(), (base[r] + j).long()
    from_page, to_page = table[r, src // page].long(), table[r, dst // page].long()
    for pool in s["pools"]:
        pool[to_page, :, dst % page] = pool[from_page, :, src % page]
    _plain_free(s, base + s["count"])


def _plain_pages(s):
    op = s["op"]
    if op == "copy":
        for pool in s["pools"]:
            pool[:, s["dst"].long()] = pool[:, s["src"].long()]
        return s["pools"]
    _plain_free(s, s["keep"])
    if op == "fork":
        _plain_fork(s)
    else:
        _plain_reserve(s, s["extra"])
        _plain_append(s)
    if op == "compact":
        _plain_compact(s)
    return s["pools"], s["table"], s["lens"], s["refs"]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if not own:
        return {"prompt": _plain_prompt, "accept": _plain_accept}.get(s["op"], _plain_pages)(s)
    from verified_metal_kernels_b200.kernels import accept_b200, pages_b200, prompt_b200
    op = s["op"]
    if op == "prompt":
        if s["page"]:
            return prompt_b200.kernel_paged(s["q"], s["k"], s["v"], s["table"], s["cu_q"], s["lens"])
        return prompt_b200.kernel(s["q"], s["k"], s["v"], s["cu_q"])
    if op == "accept":
        return accept_b200.kernel(s["target"], s["tokens"], s["bits"], s["u"], draft_probs=s["draft"])
    if op == "copy":
        pages_b200.copy(s["pools"], s["src"], s["dst"])
        return s["pools"]
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
    pages_b200.free(table, lens, refs, s["keep"], page)
    if op == "fork":
        pages_b200.fork(s["pools"], table, lens, refs, s["parents"], s["children"])
    else:
        pages_b200.reserve(table, lens, refs, s["extra"], page)
        pages_b200.append(s["k"], s["v"], s["pools"][0], s["pools"][1], table, s["cu"], lens)
    if op == "compact":
        pages_b200.compact(s["pools"], table, lens, refs, s["path"], s["count"])
    return s["pools"], table, lens, refs


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits. Page operators move values and compute none."""
    if case["op"] == "accept":
        return _exact_accept(_prepare_accept(case, seed))
    if case["op"] != "prompt":
        return None
    if work(case)["flops"] > 1e13:
        return None
    s = _prepare_prompt(case, seed)
    heads, hk, page = case["heads"], case["kv_heads"], case["paged"]
    q = s["q"].double()
    out = torch.empty_like(q)
    at_q = at_k = 0
    for i in range(case["seqs"]):
        n, keys = s["new"][i], s["keys"][i]
        for h in range(hk):
            if page:
                ids = [int(x) for x in s["table"][i].tolist() if x >= 0]
                k = torch.cat([s["k"][x, h] for x in ids])[:keys].double()
                v = torch.cat([s["v"][x, h] for x in ids])[:keys].double()
            else:
                k, v = s["k"][at_k:at_k + keys, h].double(), s["v"][at_k:at_k + keys, h].double()
            for a in range(0, n, 2048):
                z = min(n, a + 2048)
                for g in range(h * (heads // hk), (h + 1) * (heads // hk)):
                    score = q[at_q + a:at_q + z, g] @ k.T / math.sqrt(D)
                    score += torch.full_like(score, float("-inf")).triu(keys - n + a + 1)
                    out[at_q + a:at_q + z, g] = torch.softmax(score, -1) @ v
        at_q, at_k = at_q + n, at_k + keys
    return out


def _exact_accept(s):
    """Request by request, with the residual kept as a vector that each refused draft is taken off and that is normalised again."""
    target, tokens, u = s["target"], s["tokens"].tolist(), s["u"].double().tolist()
    b, n, v = target.shape
    words = s["bits"].reshape(b, n, -1).cpu().numpy().view(np.uint32)
    paths, counts, nexts = [], [], []
    for i in range(b):
        masks = [sum(int(w) << 32 * j for j, w in enumerate(words[i, k])) for k in range(n)]
        parent = [(masks[k] & ((1 << k) - 1)).bit_length() - 1 for k in range(n)]
        path = [0]
        while True:
            rest = target[i, path[-1]].cpu().numpy().astype(np.float64) if target.dtype != torch.bfloat16 else target[i, path[-1]].double().cpu().numpy()
            whole, q, found = rest, None, False
            scale = 1.0                                  # the residual is rest / scale
            if s["draft"] is not None:
                q = s["draft"][i, path[-1]].double().cpu().numpy()
            for k in [k for k in range(1, n) if parent[k] == path[-1]]:
                x = tokens[i][k]
                if rest[x] > 0 and u[i][k] * (1.0 if q is None else q[x]) < rest[x] / scale:
                    path.append(k)
                    found = True
                    break
                if q is None:
                    scale = max(scale - rest[x], 0.0) or 1e-300
                    rest = rest.copy()
                    rest[x] = 0.0
                else:
                    rest = np.maximum(rest - scale * q, 0.0)
                    scale = float(rest.sum()) or 1e-300
            if found:
                continue
            w = rest if rest.sum() > 0 else whole
            c = np.cumsum(w)
            nexts.append(int(np.nonzero((c > u[i][0] * c[-1]) & (w > 0))[0][0]) if c[-1] > 0 else -1)
            break
        paths.append(path + [-1] * (n - len(path)))
        counts.append(len(path))
    return torch.tensor(paths, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32), torch.tensor(nexts, dtype=torch.int32)
