"""A page pool in plain Python, to check the GPU's against: whole numbers, one right answer each."""

from __future__ import annotations


class Pool:
    def __init__(self, batch: int, columns: int, pages: int, page: int):
        self.table = [[-1] * columns for _ in range(batch)]
        self.lengths, self.refs, self.page = [0] * batch, [0] * pages, page

    @staticmethod
    def real(n: int) -> int:
        return -1 - n if n < 0 else n

    def pages_of(self, n: int) -> int:
        return -(-n // self.page)

    def extend(self, news: list[int]):
        """(slots of every sequence's new tokens, served, copies (source, target, filled) or None)."""
        free = [p for p, r in enumerate(self.refs) if r == 0]
        refs, at, slots, served, copies = list(self.refs), 0, [], [], []
        for b, n in enumerate(news):
            row, n0 = self.table[b], self.real(self.lengths[b])
            have, want = self.pages_of(n0), self.pages_of(n0 + n)
            if n > 0 and n0 + n > len(row) * self.page:
                ok, need = False, 0
            else:
                last = row[n0 // self.page] if n > 0 and n0 % self.page else -1
                copied = last >= 0 and self.refs[last] > 1
                need = (want - have + copied) if n > 0 else 0
                ok = need == 0 or at + need <= len(free)
                at += need  # (a sequence that is not served keeps those behind it from being served, too)
            copies.append(None)
            if ok and need:
                mine = free[at - need:at]
                if copied:
                    copies[b] = (last, mine[0], n0 % self.page)
                    refs[last] -= 1
                    row[have - 1] = mine[0]
                    for col, p in zip(range(have, want), mine[1:]):
                        row[col] = p
                else:
                    for col, p in zip(range(have, want), mine):
                        row[col] = p
                for p in mine:
                    refs[p] = 1
            served.append(ok)
            self.lengths[b] = n0 + n if ok else -1 - n0
            slots.append([row[j // self.page] * self.page + j % self.page if ok else -1 for j in range(n0, n0 + n)])
        self.refs = refs
        return slots, served, copies

    def truncate(self, keep: list[int]) -> None:
        for b, k in enumerate(keep):
            n = self.real(self.lengths[b])
            now = min(n, max(k, 0))
            for col in range(self.pages_of(now), self.pages_of(n)):
                self.refs[self.table[b][col]] -= 1
                self.table[b][col] = -1
            self.lengths[b] = now

    def reorder(self, parents: list[list[int]]) -> None:
        rows = [g * len(group) + k for g, group in enumerate(parents) for k in group]
        old, lens = [list(r) for r in self.table], list(self.lengths)
        for b in range(len(rows)):
            for p in old[b][:self.pages_of(self.real(lens[b]))]:
                self.refs[p] -= 1
        for b, r in enumerate(rows):
            used = self.pages_of(self.real(lens[r]))
            self.table[b] = old[r][:used] + [-1] * (len(old[r]) - used)
            self.lengths[b] = lens[r]
            for p in old[r][:used]:
                self.refs[p] += 1

    def check(self) -> None:
        held = [0] * len(self.refs)
        for b, row in enumerate(self.table):
            used = self.pages_of(self.real(self.lengths[b]))
            assert all(p >= 0 for p in row[:used]) and all(p == -1 for p in row[used:])
            for p in row[:used]:
                held[p] += 1
        assert held == self.refs
