"""A plain implementation of the page pool, one entry after another."""

from __future__ import annotations

import numpy as np


class Pool:
    def __init__(self, pages: int, page_size: int) -> None:
        self.refs = np.zeros(pages, dtype=np.int64)
        self.size = page_size

    def holds(self, page: int) -> bool:
        return 0 <= page < len(self.refs)

    def give(self, taken: set) -> int:
        for page in range(len(self.refs)):
            if self.refs[page] == 0 and page not in taken:
                return page
        return -1

    def words(self) -> np.ndarray:
        bits = np.zeros(-(-len(self.refs) // 32) * 32, dtype=np.uint32)
        bits[:len(self.refs)] = self.refs == 0
        shifted = bits.reshape(-1, 32) << np.arange(32, dtype=np.uint32)
        return np.bitwise_or.reduce(shifted, axis=1).view(np.int32)

    def reserve(self, table, lengths, counts) -> int:
        missing = 0
        for b, (length, count) in enumerate(zip(lengths, counts)):
            length, count = max(0, int(length)), max(0, int(count))
            for slot in range(-(-length // self.size), -(-(length + count) // self.size)):
                if slot < table.shape[1] and self.holds(table[b, slot]):
                    continue
                page = self.give(set()) if slot < table.shape[1] else -1
                if page < 0:
                    missing += 1
                else:
                    table[b, slot] = page
                    self.refs[page] = 1
        return missing

    def release(self, table, first=None, last=None) -> None:
        for b in range(table.shape[0]):
            begin = 0 if first is None else max(0, int(first[b]))
            end = table.shape[1] if last is None else min(table.shape[1], int(last[b]))
            for slot in range(begin, end):
                if self.holds(table[b, slot]):
                    self.refs[table[b, slot]] -= 1
                    table[b, slot] = -1

    def fork(self, table, lengths, parents):
        rows, width = len(parents), table.shape[1]
        new, new_lengths = np.full((rows, width), -1, dtype=np.int32), np.zeros(rows, dtype=np.int32)
        copies, missing, seen, taken = [], 0, set(), set()
        for r, parent in enumerate(parents):
            if not 0 <= parent < table.shape[0]:
                continue
            length = max(0, int(lengths[parent]))
            whole = length // self.size
            new_lengths[r] = length
            unfinished = length % self.size and whole < width and self.holds(table[parent, whole])
            if parent not in seen:
                seen.add(parent)
                new[r] = table[parent]
                if not unfinished or self.refs[table[parent, whole]] < 2:
                    continue
                new[r, whole] = -1
            else:
                new[r, :whole] = table[parent, :whole]
            if unfinished:
                page = self.give(taken)
                if page < 0:
                    missing += 1
                    new_lengths[r] = whole * self.size
                else:
                    taken.add(page)
                    new[r, whole] = page
                    copies.append((int(table[parent, whole]), page))
        for entries, step in ((new, 1), (table, -1)):
            for page in entries.flatten():
                if self.holds(page):
                    self.refs[page] += step
        return new, new_lengths, copies, missing

    def compact(self, table):
        held = [page for page in range(len(self.refs)) if self.refs[page] > 0]
        free = [page for page in range(len(held)) if self.refs[page] == 0]
        copies = list(zip([page for page in held if page >= len(held)], free))
        for source, target in copies:
            self.refs[target], self.refs[source] = self.refs[source], 0
            table[table == source] = target
        return copies, len(held)
