"""A plain page pool for the tests of ``sgl_amd_mono.moe.pages``: lists of pages, counts of holders, and the
bytes of the caches as one number a page row."""


class Pool:
    def __init__(self, pages, page_size, caches=()):
        self.pages, self.ps = pages, page_size
        self.refs = [0] * pages
        self.caches = [c.clone() for c in caches]  # [pages, ...] each
        self.errors = []  # (code, sequence)

    def need(self, n):
        return -(-n // self.ps)

    def free(self):
        return [p for p in range(self.pages) if self.refs[p] == 0]

    def adopt(self, table, lens):
        self.refs = [0] * self.pages
        for row, n in zip(table, lens):
            for p in row[: self.need(n)]:
                self.refs[p] += 1
        for b, (row, n) in enumerate(zip(table, lens)):
            if n % self.ps and self.refs[row[n // self.ps]] > 1:
                self.errors.append((5, b))

    def copy(self, src, dst):
        for c in self.caches:
            c[dst] = c[src].clone()

    def grow(self, table, lens, add, tokens):
        """-> slots, positions, starts; table (lists of full width) and lens in place."""
        free, needed, at = self.free(), 0, 0
        slots, positions, starts = [-1] * tokens, [0] * tokens, []
        taken = []
        for b, a in enumerate(add):
            starts.append(min(at, tokens))
            if a < 0:
                self.errors.append((1, b))
                a = 0
            n = lens[b]
            first, at = at, at + a
            if n + a > len(table[b]) * self.ps or at > tokens:
                self.errors.append((4, b))
                continue
            k = self.need(n + a) - self.need(n)
            needed += k
            if k and needed > len(free):
                self.errors.append((3, b))
                continue
            for i, p in enumerate(free[needed - k : needed]):
                table[b][self.need(n) + i] = p
                taken.append(p)
            for i in range(a):
                positions[first + i] = n + i
                slots[first + i] = table[b][(n + i) // self.ps] * self.ps + (n + i) % self.ps
            lens[b] = n + a
        for p in taken:
            self.refs[p] = 1
        starts.append(min(at, tokens))
        return slots, positions, starts

    def trim(self, table, lens, keep):
        free, was = self.free(), list(self.refs)
        gone, taken = [], 0
        for b, k in enumerate(keep):
            n, to = lens[b], min(lens[b], max(k, 0))
            if to < n and to % self.ps and was[table[b][to // self.ps]] > 1:
                taken += 1
                if taken > len(free):
                    self.errors.append((3, b))
                    continue
                e, p = to // self.ps, free[taken - 1]
                self.copy([table[b][e]], [p])
                self.refs[p] = 1
                gone.append(table[b][e])
                table[b][e] = p
            gone += table[b][self.need(to) : self.need(n)]
            lens[b] = to
        for p in gone:
            self.refs[p] -= 1

    def fork(self, table, lens, parents):
        free, taken = self.free(), 0
        old, old_lens = [list(r) for r in table], list(lens)
        seen = set()
        for b, r in enumerate(parents):
            if not 0 <= r < len(parents):
                if r != -1:
                    self.errors.append((1, b))
                lens[b] = 0
                continue
            n = old_lens[r]
            own = None
            if n % self.ps and r in seen:
                taken += 1
                if taken > len(free):
                    self.errors.append((3, b))
                    lens[b] = 0
                    continue
                own = free[taken - 1]
                self.copy([old[r][n // self.ps]], [own])
            seen.add(r)
            table[b][: self.need(n)] = old[r][: self.need(n)]
            if own is not None:
                table[b][n // self.ps] = own
            lens[b] = n
        # (counts anew, with those of sequences that the table does not have)
        for row, n in zip(old, old_lens):
            for p in row[: self.need(n)]:
                self.refs[p] -= 1
        for row, n in zip(table, lens):
            for p in row[: self.need(n)]:
                self.refs[p] += 1

    def compact(self, table, lens):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, self.pages) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        if src:
            self.copy(src, dst)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        for row, n in zip(table, lens):
            for i in range(self.need(n)):
                row[i] = to.get(row[i], row[i])
