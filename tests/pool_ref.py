"""A pool of pages in plain Python, one request and one page at a time (the semantics of ``pages``)."""
import copy

import numpy as np


def held(rows, block):
    return -(-rows // block)


class Pool:
    def __init__(self, tables, lengths, refs, block):
        self.tables, self.lengths, self.refs, self.block = [list(t) for t in tables], list(lengths), list(refs), block

    @classmethod
    def empty(cls, pages, block, requests, cols, reserved=0):
        return cls([[-1] * cols for _ in range(requests)], [0] * requests, [int(p < reserved) for p in range(pages)], block)

    @classmethod
    def random(cls, rng, lengths, block, cols, pages, share=0.0, reserved=0):
        """Requests with pages in random order; some begin with the whole pages (or all) of an earlier one."""
        pool = cls.empty(pages, block, len(lengths), cols, reserved)
        ids = [p for p in rng.permutation(pages).tolist() if p >= reserved]
        for r, n in enumerate(lengths):
            own = held(n, block)
            if r and rng.random() < share:
                parent = int(rng.integers(r))
                common = min(held(pool.lengths[parent], block), own)
                if rng.random() < 0.5:      # nothing beyond the parent: a shared last page with rows in it
                    n = pool.lengths[r] = min(n, pool.lengths[parent])
                    common = own = held(n, block)
                elif common and n != pool.lengths[parent]:
                    common = min(common, min(n, pool.lengths[parent]) // block)
                for c in range(common):
                    pool.tables[r][c] = pool.tables[parent][c]
            else:
                common = 0
            pool.lengths[r] = n
            for c in range(own):
                if c >= common:
                    pool.tables[r][c] = ids.pop()
                pool.refs[pool.tables[r][c]] += 1
        return pool

    def copy(self):
        return copy.deepcopy(self)

    def free(self):
        return [p for p, n in enumerate(self.refs) if n == 0]

    def words(self):
        out = np.zeros(-(-len(self.refs) // 32), np.uint32)
        for p in self.free():
            out[p // 32] |= np.uint32(1) << np.uint32(p % 32)
        return out.view(np.int32)

    def check(self, extra=0):
        """Tables, lengths and counts agree."""
        seen = [0] * len(self.refs)
        for t, n in zip(self.tables, self.lengths):
            own = held(n, self.block)
            assert all(p >= 0 for p in t[:own]) and all(p == -1 for p in t[own:])
            for p in t[:own]:
                seen[p] += 1
        assert [a - b for a, b in zip(self.refs, seen)] == [int(p < extra) for p in range(len(seen))]

    def release(self, requests, lengths=None):
        for i, r in enumerate(requests):
            if 0 <= r < len(self.lengths):
                new = max(0, lengths[i]) if lengths is not None else 0
                for c in range(held(new, self.block), held(self.lengths[r], self.block)):
                    self.refs[self.tables[r][c]] -= 1
                    self.tables[r][c] = -1
                self.lengths[r] = min(self.lengths[r], new)

    def fork(self, parents, children):
        R, ok = len(self.lengths), []
        before, tables = list(self.lengths), [list(t) for t in self.tables]
        for i, (p, c) in enumerate(zip(parents, children)):
            good = 0 <= p < R and 0 <= c < R and before[c] == 0 and c not in children[:i] and p not in children
            ok.append(good)
            if good:
                self.lengths[c] = before[p]
                for k in range(held(before[p], self.block)):
                    self.tables[c][k] = tables[p][k]
                    self.refs[tables[p][k]] += 1
        return ok

    def extend(self, lengths, write_from=None):
        """``(ok, pairs)`` with ``pairs[r]`` a dict column -> (source, target)."""
        free, b, cols = self.free(), self.block, len(self.tables[0]) if self.tables else 0
        refs, asked, at, ok, pairs, dropped = list(self.refs), 0, 0, [], [], []
        for r, n in enumerate(self.lengths):
            want = max(n, lengths[r])
            start = n if write_from is None else min(max(write_from[r], 0), n)
            pairs.append({})
            if want > cols * b:
                ok.append(False)
                continue
            takes = [] if want <= start else [c for c in range(start // b, held(want, b))
                                              if c >= held(n, b) or refs[self.tables[r][c]] > 1]
            asked += len(takes)
            ok.append(not takes or asked <= len(free))
            if not ok[-1]:
                continue
            for c in takes:
                page = free[at]
                at += 1
                if c < held(n, b):
                    pairs[r][c] = (self.tables[r][c], page)
                    dropped.append(self.tables[r][c])
                self.tables[r][c] = page
                self.refs[page] = 1
            self.lengths[r] = want
        for page in dropped:
            self.refs[page] -= 1
        return ok, pairs

    def compact(self):
        used = sum(n > 0 for n in self.refs)
        movers = [p for p in range(used, len(self.refs)) if self.refs[p]]
        holes = [p for p in range(used) if not self.refs[p]]
        place = dict(zip(movers, holes))
        for t, n in zip(self.tables, self.lengths):
            for c in range(held(n, self.block)):
                t[c] = place.get(t[c], t[c])
        for a, b in place.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        return movers, holes
