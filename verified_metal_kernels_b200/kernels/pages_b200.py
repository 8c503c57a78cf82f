"""Kernel module for the pages of a paged cache on B200: what keeps the tables that every kernel_paged(...) reads.

The reference names the paged cache as the variant it left out (README.md:141-142).  State, int32 tensors on the device
that the calls change in place:

    page_table (R,T)   slot i of row r: the page of its positions [i * page_size, (i+1) * page_size), -1 behind them
    lens (R,)          positions of each row
    refs (pages,)      how many slots name a page; 0: the page is free

Pages are given lowest first, to rows in their order.  A pool is a contiguous tensor (pages, heads, page_size, width),
(layers, pages, heads, page_size, width) or, as dsa's, (pages, page_size, width), of any type whose rows are multiples of
16 bytes.  Calls on one state belong on one stream; they neither allocate on the host nor synchronise (check=True
does, and raises on what the device refused: no free page left, an index outside its tensor)."""
import struct

import torch

from .. import _lib
from ._common import calls, elsewhere, handles, need, need_on, scratch


def _state(page_table, lens, refs):
    need(page_table, "page_table", torch.int32, dims=2)
    R, T = page_table.shape
    dev = page_table.device
    need_on(lens, "lens", torch.int32, (R,), dev)
    if refs is not None:
        need(refs, "refs", torch.int32, dims=1)
        _on(refs, "refs", dev)
    return R, T, dev


def _on(t, name, dev):
    if t.device != dev:
        raise ValueError(f"{name}: expected a tensor on {dev}, got {t.device}")


def _pools(pools, dev):
    """The pools' descriptions (four int64 each), their pages and page size."""
    if isinstance(pools, torch.Tensor) or not 1 <= len(pools) <= 8:
        raise ValueError("pools: expected a list of 1 to 8 tensors")
    d, pages, page_size = [], None, None
    for i, t in enumerate(pools):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"pools[{i}]: expected a torch tensor, got {type(t).__name__}")
        if not t.is_cuda or not t.is_contiguous():
            need(t, f"pools[{i}]", t.dtype)
        shape = t.shape
        dims = len(shape)
        if dims not in (3, 4, 5) or 0 in shape:
            raise ValueError(f"pools[{i}]: expected (pages,[heads,]page_size,width) or (layers,pages,heads,page_size,width), got {tuple(shape)}")
        if t.device != dev:
            _on(t, f"pools[{i}]", dev)
        layers = shape[0] if dims == 5 else 1
        n, positions, row = shape[1 if dims == 5 else 0], shape[-2], shape[-1] * t.element_size()
        if pages is None:
            pages, page_size = n, positions
        if n != pages or positions != page_size:
            raise ValueError(f"pools[{i}]: expected {pages} pages of {page_size} positions, got {n} of {positions}")
        if row % 16:
            raise ValueError(f"pools[{i}]: a position's row must be a multiple of 16 bytes")
        d += (t.data_ptr(), layers, shape[-3] if dims > 3 else 1, row)
    return struct.pack(f"{len(d)}q", *d), pages, page_size


def _need_refs(refs, pages):
    if refs.shape[0] != pages:
        raise ValueError(f"refs: expected {pages} entries, one a page, got {refs.shape[0]}")


def _done(rc, what, check, dev):
    _lib.check(rc, what)
    if check:
        _lib.raise_on_status(dev, what)


def reserve(page_table, lens, refs, extra, page_size, check=False):
    """Row r grows by extra[r] (>= 0) positions: it gets the pages that it lacks, and lens[r] += extra[r].  A row gets all its
    pages or, where what it and the rows before it need exceeds the free pages (or its table is too short), none, and
    stays as it is.  So does a row whose last page is partly used and shared (it was cut there by free, or another row was):
    its next positions belong to the others too.  fork it into an empty row, which gets a page of its own, and free it: that
    is how a request goes on from a prefix of another one.  Returns granted (R,) int32, 1 or 0."""
    if not check:
        granted = calls().reserve(page_table, lens, refs, extra, page_size)
        if granted is not None:
            return granted
    R, T, dev = _state(page_table, lens, refs)
    need_on(extra, "extra", torch.int32, (R,), dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return reserve(page_table, lens, refs, extra, page_size, check)
    stream, status = handles(dev)
    granted = torch.empty_like(lens)
    ws = scratch(lib.vmk_pages_workspace_bytes(R, 0, refs.shape[0]), dev, stream)
    rc = lib.vmk_pages_reserve(page_table.data_ptr(), R, T, lens.data_ptr(), refs.data_ptr(), refs.shape[0], page_size, extra.data_ptr(),
                               granted.data_ptr(), *ws, status, stream)
    _done(rc, "vmk_pages_reserve", check, dev)
    return granted


def append(k, v, k_pages, v_pages, page_table, cu, lens, check=False, granted=None, refs=None):
    """Writes packed tokens into their pages: k, v (tokens,heads,width) -- views are fine, the innermost axis contiguous --
    and tokens [cu[s], cu[s+1]) of row s become its last positions: lens[s] counts them already (reserve before append).
    k_pages, v_pages (pages,heads,page_size,width), or (pages,page_size,width) for one head; k and v may differ in
    heads and width (dsa: latent rows and index keys).  Tokens outside [cu[0], cu[-1]) are not written.

    granted (R,) int32, as reserve returns it: the tokens of a row with 0 are not written.  A step that does not wait for
    the outcome of reserve passes it on here and to compact: lens of a refused row does not count its tokens, which would
    take the place of the row's last ones.  refs (pages,) int32: a token whose page other rows share is not written (and
    reported); after reserve there is none, unless a row was forked between the two calls."""
    if not check and calls().append(k, v, k_pages, v_pages, page_table, cu, lens, granted, refs):
        return
    R, T, dev = _state(page_table, lens, None)
    if granted is not None:
        need_on(granted, "granted", torch.int32, (R,), dev)
    need(cu, "cu", torch.int32, dims=1)
    S = cu.shape[0] - 1
    if S < 0 or S > R:
        raise ValueError(f"cu: expected 1 to {R + 1} entries, got {cu.shape[0]}")
    pools, pages, page_size = _pools([k_pages, v_pages], dev)
    if refs is not None:
        need_on(refs, "refs", torch.int32, (pages,), dev)
    if k_pages.dim() == 5 or v_pages.dim() == 5:
        raise ValueError("k_pages, v_pages: expected the pools of one layer")
    tokens, src = len(k) if isinstance(k, torch.Tensor) and k.dim() else 0, []
    for name, t, pool in (("k", k, k_pages), ("v", v, v_pages)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
        want = (tokens, pool.shape[1] if pool.dim() == 4 else 1, pool.shape[-1])
        if t.dtype != pool.dtype:
            raise TypeError(f"{name}: expected dtype {pool.dtype}, got {t.dtype}")
        if t.shape != want:
            raise ValueError(f"{name}: expected shape {want}, got {tuple(t.shape)}")
        if t.device != dev:
            _on(t, name, dev)
        e, (by_token, by_head, by_width), at = t.element_size(), t.stride(), t.data_ptr()
        by_token, by_head = (by_token * e if want[0] > 1 else 0), (by_head * e if want[1] > 1 else 0)
        if tokens and (by_width != 1 or at % 16 or by_token < 0 or by_head < 0 or by_token % 16 or by_head % 16):
            raise ValueError(f"{name}: expected a 16-byte aligned tensor, its innermost axis contiguous, its strides multiples of 16 bytes")
        src += (at, by_token, by_head)
    _on(cu, "cu", dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return append(k, v, k_pages, v_pages, page_table, cu, lens, check, granted, refs)
    stream, status = handles(dev)
    rc = lib.vmk_pages_append_granted(pools, struct.pack("6q", *src), pages, page_size, page_table.data_ptr(), T, cu.data_ptr(),
                                      lens.data_ptr(), _lib.ptr(refs), _lib.ptr(granted), S, tokens, status,
                                      stream)
    _done(rc, "vmk_pages_append_granted", check, dev)


def fork(pools, page_table, lens, refs, parents, children, check=False):
    """Row children[f] (of length 0) becomes a copy of row parents[f], for every entry f of the two (F,) int32 tensors: full
    pages are shared, the used rows of a last page that is not full are copied into a page of its own, in every pool.
    parents[f] < 0: an entry that does nothing.  Refused (and reported): a child that is not empty, out of range, or
    named a second time; entries for which no free page is left."""
    if not check and calls().fork(pools, page_table, lens, refs, parents, children):
        return
    R, T, dev = _state(page_table, lens, refs)
    desc, pages, page_size = _pools(pools, dev)
    _need_refs(refs, pages)
    need(parents, "parents", torch.int32, dims=1)
    F = parents.shape[0]
    need_on(children, "children", torch.int32, (F,), dev)
    _on(parents, "parents", dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return fork(pools, page_table, lens, refs, parents, children, check)
    stream, status = handles(dev)
    ws = scratch(lib.vmk_pages_workspace_bytes(R, F, 0), dev, stream)
    rc = lib.vmk_pages_fork(desc, len(pools), page_table.data_ptr(), R, T, lens.data_ptr(), refs.data_ptr(), pages, page_size, parents.data_ptr(),
                            children.data_ptr(), F, *ws, status, stream)
    _done(rc, "vmk_pages_fork", check, dev)


def compact(pools, page_table, lens, refs, path, count, check=False, granted=None):
    """After kd drafts at the end of each row were verified: the accepted ones, path (R,kd) int32 and count (R,) int32 as
    accept_b200.kernel gives them, close up behind the positions before the drafts, lens[r] becomes lens[r] - kd +
    count[r], and pages behind that are given back.  count[r] < 0: the row stays as it is, and so does a row with 0 in
    granted (R,) int32 (see append): it got no place for its drafts.

    A row moves as a whole or not at all: where an entry would move into a page that other rows share, or its path does not
    ascend, the row keeps its length and its pages (and the call reports it)."""
    if not check and calls().compact(pools, page_table, lens, refs, path, count, granted):
        return
    R, T, dev = _state(page_table, lens, refs)
    desc, pages, page_size = _pools(pools, dev)
    _need_refs(refs, pages)
    need(path, "path", torch.int32, dims=2)
    kd = path.shape[1]
    need_on(path, "path", torch.int32, (R, kd), dev)
    need_on(count, "count", torch.int32, (R,), dev)
    if granted is not None:
        need_on(granted, "granted", torch.int32, (R,), dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return compact(pools, page_table, lens, refs, path, count, check, granted)
    stream, status = handles(dev)
    rc = lib.vmk_pages_compact_granted(desc, len(pools), page_table.data_ptr(), R, T, lens.data_ptr(), refs.data_ptr(), pages, page_size,
                                       path.data_ptr(), count.data_ptr(), _lib.ptr(granted), kd, status, stream)
    _done(rc, "vmk_pages_compact_granted", check, dev)


def free(page_table, lens, refs, keep, page_size, check=False):
    """Row r keeps its first keep[r] (>= 0) positions; the pages behind them are given back (a page that other rows share
    stays theirs), and their slots become -1.  keep[r] = 0 frees the row, keep[r] >= lens[r] leaves it as it is."""
    if not check and calls().free(page_table, lens, refs, keep, page_size):
        return
    R, T, dev = _state(page_table, lens, refs)
    need_on(keep, "keep", torch.int32, (R,), dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return free(page_table, lens, refs, keep, page_size, check)
    stream, status = handles(dev)
    rc = lib.vmk_pages_free(page_table.data_ptr(), R, T, lens.data_ptr(), refs.data_ptr(), refs.shape[0], page_size, keep.data_ptr(),
                            status, stream)
    _done(rc, "vmk_pages_free", check, dev)


def copy(pools, src, dst, check=False):
    """Page src[i] -> page dst[i] in every pool and layer; src, dst (n,) int32.  No page may be both in src and in dst, or
    twice in dst."""
    if not check and calls().copy(pools, src, dst):
        return
    if isinstance(pools, torch.Tensor) or not pools or not isinstance(pools[0], torch.Tensor):
        raise ValueError("pools: expected a list of 1 to 8 tensors")
    dev = pools[0].device
    desc, pages, page_size = _pools(pools, dev)
    need(src, "src", torch.int32, dims=1)
    need_on(dst, "dst", torch.int32, tuple(src.shape), dev)
    _on(src, "src", dev)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return copy(pools, src, dst, check)
    stream, status = handles(dev)
    rc = lib.vmk_pages_copy(desc, len(pools), pages, page_size, src.data_ptr(), dst.data_ptr(), src.shape[0], status,
                            stream)
    _done(rc, "vmk_pages_copy", check, dev)
