"""The page operators restated one row after another in NumPy, as the tests' truth."""
import numpy as np


class Model:
    def __init__(self, table, lens, refs, page_size, pools=()):
        """pools: arrays (layers, pages, heads, page_size, width)."""
        self.table, self.lens, self.refs, self.ps = table.copy(), lens.copy(), refs.copy(), page_size
        self.pools = [p.copy() for p in pools]
        self.status = 0

    def _pages(self, n):
        return -(-int(n) // self.ps)

    def reserve(self, extra):
        free = [int(i) for i in np.nonzero(self.refs == 0)[0]]
        asked, granted, refs = 0, [], self.refs.copy()
        for r, more in enumerate(int(x) for x in extra):
            have, want = self._pages(self.lens[r]), self._pages(self.lens[r] + max(more, 0))
            if more < 0 or want > self.table.shape[1]:
                self.status |= 2 if more < 0 else 4
                granted.append(0)
                continue
            if more > 0 and self.lens[r] % self.ps and refs[self.table[r, have - 1]] > 1:
                self.status |= 4                # the positions behind it are another row's
                granted.append(0)
                continue
            start, asked = asked, asked + want - have
            if want > have and asked > len(free):
                self.status |= 4
                granted.append(0)
                continue
            for i in range(want - have):
                self.table[r, have + i] = free[start + i]
                self.refs[free[start + i]] = 1
            self.lens[r] += more
            granted.append(1)
        return np.array(granted, dtype=np.int32)

    def free(self, keep):
        for r, k in enumerate(int(x) for x in keep):
            if k < 0:
                self.status |= 2
                continue
            k = min(k, int(self.lens[r]))
            for i in range(self._pages(k), self._pages(self.lens[r])):
                self.refs[self.table[r, i]] -= 1
                self.table[r, i] = -1
            self.lens[r] = k

    def append(self, sources, cu):
        """sources: one (tokens, heads, width) array per pool; the pools have one layer."""
        for s in range(len(cu) - 1):
            for t in range(cu[s], cu[s + 1]):
                pos = int(self.lens[s]) - (cu[s + 1] - t)
                for pool, src in zip(self.pools, sources):
                    pool[0, self.table[s, pos // self.ps], :, pos % self.ps] = src[t]

    def fork(self, parents, children):
        free = [int(i) for i in np.nonzero(self.refs == 0)[0]]
        lens, seen, asked = self.lens.copy(), set(), 0
        for par, c in zip((int(x) for x in parents), (int(x) for x in children)):
            if par < 0:
                continue
            R = len(lens)
            if par >= R or not 0 <= c < R or c in seen or lens[c] != 0:
                self.status |= 2
                seen.add(c)
                continue
            seen.add(c)
            n = int(lens[par])
            full, rest = divmod(n, self.ps)
            if rest:
                asked += 1
                if asked > len(free):
                    self.status |= 4
                    continue
            for i in range(full):
                self.table[c, i] = self.table[par, i]
                self.refs[self.table[par, i]] += 1
            if rest:
                new = free[asked - 1]
                for pool in self.pools:
                    pool[:, new, :, :rest] = pool[:, self.table[par, full], :, :rest]
                self.table[c, full] = new
                self.refs[new] = 1
            self.lens[c] = n

    def compact(self, path, count):
        kd = path.shape[1]
        keep = self.lens.copy()
        for r, n in enumerate(int(x) for x in count):
            if n < 0:
                continue
            base = int(self.lens[r]) - kd
            for j in range(n):
                a, b = base + int(path[r, j]), base + j
                for pool in self.pools:
                    pool[:, self.table[r, b // self.ps], :, b % self.ps] = pool[:, self.table[r, a // self.ps], :, a % self.ps]
            keep[r] = base + n
        self.free(keep)

    def copy(self, src, dst):
        for s, d in zip(src, dst):
            for pool in self.pools:
                pool[:, d] = pool[:, s]
