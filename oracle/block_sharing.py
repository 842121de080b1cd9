"""Block sharing, beam reordering and compaction restated on Python lists (test infrastructure only)."""
from __future__ import annotations

import numpy as np

SUCCESS, INSUFFICIENT_SPACE, FAILURE, ROW_FULL, INVALID = range(5)


class SharedPool:
    """The state of a shared block pool: free stack, rows (None: no entry) and holder counts."""

    def __init__(self, num_blocks: int, max_seqs: int, max_blocks: int, block_size: int):
        self.NB, self.BS, self.max_blocks = num_blocks, block_size, max_blocks
        self.stack = list(range(num_blocks))
        self.rows: list = [None] * max_seqs
        self.ref = [0] * num_blocks

    def allocate(self, slot: int, n: int) -> int:
        row = self.rows[slot] or []
        if len(self.stack) < n:
            return INSUFFICIENT_SPACE
        if len(row) + n > self.max_blocks:
            return ROW_FULL
        new = [self.stack.pop() for _ in range(n)]
        for b in new:
            self.ref[b] = 1
        self.rows[slot] = row + new
        return SUCCESS

    def release(self, slot: int) -> int:
        if self.rows[slot] is None:
            return FAILURE
        for b in self.rows[slot]:
            self.ref[b] -= 1
            if self.ref[b] == 0:
                self.stack.append(b)
        self.rows[slot] = None
        return SUCCESS

    def fork(self, slot: int, tokens: int, parent: int):
        """(status, (src, dst, slots) of the page copy or None)."""
        old = self.rows[parent]
        full, tail = divmod(tokens, self.BS)
        if old is None or self.rows[slot] is not None:
            return FAILURE, None
        if full + (tail > 0) > len(old):
            return ROW_FULL, None
        if tail and not self.stack:
            return INSUFFICIENT_SPACE, None
        row, copy = list(old[:full]), None
        for b in row:
            self.ref[b] += 1
        if tail:
            b = self.stack.pop()
            self.ref[b] = 1
            row.append(b)
            copy = (old[full], b, tail)
        self.rows[slot] = row
        return SUCCESS, copy

    def may_reorder(self, slots, tokens) -> bool:
        """Whether a partly filled last block, which copies and the next tokens write, belongs to its row alone."""
        full, tail = divmod(tokens, self.BS)
        return not tail or all(self.ref[self.rows[s][full]] == 1 for s in slots)

    def reorder(self, slots, parents, tokens):
        """One group: (new slots, page copies); freed blocks are returned, to be pushed in ascending order by ``push``."""
        K = len(slots)
        full, tail = divmod(tokens, self.BS)
        spare = [slots[k] for k in range(K) if k not in parents]
        out, copies, freed, seen = [], [], [], set()
        for j in range(K):
            p = parents[j]
            if p not in seen:
                seen.add(p)
                out.append(slots[p])
                continue
            child, donor = spare.pop(0), slots[p]
            out.append(child)
            for c in range(full):
                was, now = self.rows[child][c], self.rows[donor][c]
                if was != now:
                    self.rows[child][c] = now
                    self.ref[now] += 1
                    self.ref[was] -= 1
                    if self.ref[was] == 0:
                        freed.append(was)
            if tail:
                copies.append((self.rows[donor][full], self.rows[child][full], tail))
        return out, copies, freed

    def push(self, freed) -> None:
        self.stack.extend(sorted(freed))

    def compact(self, after=None):
        """(live, moves [(src, dst)])."""
        after = self.NB if after is None else after
        live = sum(r > 0 for r in self.ref)
        assert live <= after
        holes = [b for b in range(live) if self.ref[b] == 0]
        moved = [b for b in range(live, self.NB) if self.ref[b] > 0]
        to = dict(zip(moved, holes))
        for s, d in to.items():
            self.ref[d], self.ref[s] = self.ref[s], 0
        self.rows = [None if r is None else [to.get(b, b) for b in r] for r in self.rows]
        self.stack = list(range(after - 1, live - 1, -1))
        return live, list(to.items())

    def check(self) -> None:
        """Every held block is counted once per row, every other block is on the stack once."""
        ref = [0] * self.NB
        for r in self.rows:
            for b in r or []:
                ref[b] += 1
        assert ref == self.ref
        assert len(set(self.stack)) == len(self.stack) and all(ref[b] == 0 for b in self.stack)


def copy_pages(pages: np.ndarray, copies) -> None:
    """pages [block, slot, ...]: the first slots of src to dst, all sources read first."""
    got = [pages[s, :n].copy() for s, _, n in copies]
    for (_, d, n), g in zip(copies, got):
        pages[d, :n] = g
