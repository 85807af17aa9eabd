"""The pages of a paged cache, stated with Python lists (oracle; test infrastructure only).

`Pool` holds what muse_spark_open_b200/pages.py keeps on the device; every method does what the function of its name does,
entry by entry, and returns the kinds of problems it met ("bounds", "capacity").  Caches are CPU tensors [num_pages,
page_size, ...] changed in place.
"""
from __future__ import annotations


class Pool:
    def __init__(self, num_pages, page_size, rows, max_pages):
        self.size, self.max_pages = page_size, max_pages
        self.table = [[-1] * max_pages for _ in range(rows)]
        self.seq, self.refs = [0] * rows, [0] * num_pages

    def _free_list(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def _drop(self, row, lp):
        if self.table[row][lp] >= 0:
            self.refs[self.table[row][lp]] -= 1
            self.table[row][lp] = -1

    def _first_of(self, rows):
        """For each entry: whether it names a row, and is the first that names it."""
        seen, ok = set(), []
        for r in rows:
            ok.append(0 <= r < len(self.table) and r not in seen)
            seen.add(r)
        return ok

    def extend(self, rows, counts):
        """(flat cache rows of the new tokens, problems)"""
        free, bad, loc = self._free_list(), set(), []
        for r, n, ok in zip(rows, counts, self._first_of(rows)):
            if not ok:
                bad.add("bounds")
                loc += [-1] * n
                continue
            span = {pos // self.size for pos in range(self.seq[r], self.seq[r] + n)}
            if any(self.refs[self.table[r][lp]] > 1 for lp in span if lp < self.max_pages and self.table[r][lp] >= 0):
                bad.add("bounds")  # a page that other rows share
                loc += [-1] * n
                continue
            for pos in range(self.seq[r], self.seq[r] + n):
                lp = pos // self.size
                if lp >= self.max_pages:
                    bad.add("capacity")
                    loc.append(-1)
                    continue
                if self.table[r][lp] < 0:
                    if free:
                        self.table[r][lp] = free.pop(0)
                        self.refs[self.table[r][lp]] = 1
                    else:
                        bad.add("capacity")
                loc.append(self.table[r][lp] * self.size + pos % self.size if self.table[r][lp] >= 0 else -1)
        return loc, bad

    def fork(self, parents, children, caches):
        free, bad, todo = self._free_list(), set(), []
        good = self._first_of(children)
        for p, c, ok in zip(parents, children, good):
            if not ok or not 0 <= p < len(self.table) or c in parents:
                bad.add("bounds")
                continue
            full, part = divmod(self.seq[p], self.size)
            row = self.table[p][:full] + [-1] * (self.max_pages - full)
            copy = None
            seq = self.seq[p]
            if part and self.table[p][full] >= 0:
                if free:
                    row[full] = free.pop(0)
                    copy = (self.table[p][full], row[full], part)
                else:
                    bad.add("capacity")
                    row, seq = [-1] * self.max_pages, 0
            todo.append((c, row, seq, copy))
        for c, row, seq, copy in todo:
            for x in row:
                if x >= 0:
                    self.refs[x] += 1
        for c, row, seq, copy in todo:
            for lp in range(self.max_pages):
                self._drop(c, lp)
            self.table[c], self.seq[c] = list(row), seq
            if copy:
                for cache in caches:
                    cache[copy[1], :copy[2]] = cache[copy[0], :copy[2]]
        return bad

    def free(self, rows):
        bad = set()
        for r in rows:
            if not 0 <= r < len(self.table):
                bad.add("bounds")
                continue
            for lp in range(self.max_pages):
                self._drop(r, lp)
            self.seq[r] = 0
        return bad

    def trim(self, rows, window, sinks):
        bad = set()
        for r in rows:
            if not 0 <= r < len(self.table):
                bad.add("bounds")
                continue
            for lp in range(self.max_pages):
                first, last = lp * self.size, (lp + 1) * self.size - 1
                if window and last <= self.seq[r] - window and first >= sinks:  # the next token sees s > seq - window
                    self._drop(r, lp)
        return bad

    def compact(self, caches):
        """(pages in use, pages moved)"""
        n = sum(1 for r in self.refs if r > 0)
        src = [i for i in range(n, len(self.refs)) if self.refs[i] > 0]
        dst = [i for i in range(n) if self.refs[i] == 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            for cache in caches:
                cache[b] = cache[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(x, x) for x in row] for row in self.table]
        return n, len(src)

    def consistent(self):
        """refs count the table's entries, and nothing else."""
        count = [0] * len(self.refs)
        for row in self.table:
            for x in row:
                if x >= 0:
                    count[x] += 1
        return count == self.refs
