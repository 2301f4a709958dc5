"""Which pages of a paged cache belong to which sequence: host bookkeeping.

The device side is ops.KV8Cache (the pages), ops.kv8_append and ops.gqa_kv8
(which follow a page table) and ops.kv8_copy_pages (which carries out the
copies that extend() and compact() name).  A page may belong to several
sequences, whose prefix it holds; it is written only while it belongs to one.
"""
from __future__ import annotations

from operator import index

import torch


class KVPages:
    """The pages of a pool, handed out, shared, taken back and moved together.

    Sequences are whole numbers given out by new() and fork().  Every method
    either succeeds or raises and changes nothing."""

    def __init__(self, pages: int, page: int):
        if pages < 1 or page < 1:
            raise ValueError(f"pages ({pages}) and page ({page}) must be positive")
        self.pages, self.page = pages, page
        self._free = list(range(pages - 1, -1, -1))  # the lowest number is handed out first
        self._users = [0] * pages
        self._seqs: dict[int, list] = {}             # sequence -> [its pages, its tokens]
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _of(self, seq: int) -> list:
        if seq not in self._seqs:
            raise KeyError(f"no sequence {seq}")
        return self._seqs[seq]

    def length(self, seq: int) -> int:
        return self._of(seq)[1]

    def pages_of(self, seq: int) -> tuple[int, ...]:
        return tuple(self._of(seq)[0])

    def new(self) -> int:
        """A sequence of no tokens."""
        self._next += 1
        self._seqs[self._next] = [[], 0]
        return self._next

    def fork(self, seq: int) -> int:
        """A sequence of the same tokens on the same pages."""
        pages, tokens = self._of(seq)
        child = self.new()
        self._seqs[child] = [list(pages), tokens]
        for p in pages:
            self._users[p] += 1
        return child

    def extend(self, seq: int, tokens: int) -> list[tuple[int, int]]:
        """Room for `tokens` more tokens, which length() and table() count from now on.

        Returns the page copies, (from, to), to carry out before they are
        written: of a last page that is partly filled and shared, which the sequence
        then holds alone.  MemoryError where the pool has too few pages."""
        return self.extend_all([(seq, tokens)])

    def extend_all(self, wants) -> list[tuple[int, int]]:
        """extend() for each (sequence, tokens) of a step, or for none: where the pool has too few
        pages for all of them, MemoryError, and no sequence has moved to a page whose copy is lost
        with the call.  The copies returned are one list for ops.kv8_copy_pages."""
        more: dict[int, int] = {}
        for seq, tokens in wants:
            tokens = index(tokens)
            if tokens < 0:
                raise ValueError(f"tokens ({tokens}) must not be negative")
            self._of(seq)
            more[seq] = more.get(seq, 0) + tokens
        plan, users, need = [], {}, 0
        for seq, tokens in more.items():
            pages, old = self._seqs[seq]
            if tokens == 0:
                continue
            split = False
            if old % self.page:
                last = pages[-1]
                left = users.get(last, self._users[last])  # who holds it once those before have their own
                split = left > 1
                users[last] = left - split
            fresh = -(-(old + tokens) // self.page) - len(pages)
            plan.append((self._seqs[seq], split, fresh, old + tokens))
            need += fresh + split
        if need > len(self._free):
            raise MemoryError(f"{need} pages are needed and {len(self._free)} are free")
        copies = []
        for entry, split, fresh, tokens in plan:
            pages = entry[0]
            if split:
                copies.append((pages[-1], self._take()))
                self._users[pages[-1]] -= 1
                pages[-1] = copies[-1][1]
            pages.extend(self._take() for _ in range(fresh))
            entry[1] = tokens
        return copies

    def truncate(self, seq: int, tokens: int) -> None:
        """Drops the sequence's tokens from `tokens` on (rejected ones), and the pages that only they were on.  The page
        that they shared with the tokens before them keeps the scales that they raised: extending a fork() instead
        leaves that page as it was."""
        entry = self._of(seq)
        if not 0 <= tokens <= entry[1]:
            raise ValueError(f"tokens ({tokens}) must be 0 to {entry[1]}")
        keep = -(-tokens // self.page)
        for p in reversed(entry[0][keep:]):
            self._drop(p)
        del entry[0][keep:]
        entry[1] = tokens

    def free(self, seq: int) -> None:
        """Ends the sequence; pages that no other one holds go back to the pool."""
        for p in reversed(self._of(seq)[0]):
            self._drop(p)
        del self._seqs[seq]

    def compact(self) -> list[tuple[int, int]]:
        """Moves the pages in use to the lowest numbers, and the tables with them.

        Returns the copies, (from, to), to carry out before the tables are used: no page
        is in both columns."""
        used = [p for p in range(self.pages) if self._users[p]]
        holes = [p for p in range(len(used)) if not self._users[p]]
        moves = list(zip(used[len(used) - len(holes):], holes)) if holes else []
        to = dict(moves)
        for a, b in moves:
            self._users[b], self._users[a] = self._users[a], 0
        for entry in self._seqs.values():
            entry[0] = [to.get(p, p) for p in entry[0]]
        self._free = list(range(self.pages - 1, len(used) - 1, -1))
        return moves

    def table(self, seqs, columns: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(page_table [B, columns], kv_lens [B]) of these sequences, int32 on the host; -1 where there is no page."""
        entries = [self._of(s) for s in seqs]
        most = max([1] + [len(e[0]) for e in entries])
        if columns is None:
            columns = most
        if columns < most:
            raise ValueError(f"{columns} columns are too few for {most} pages")
        rows = [e[0] + [-1] * (columns - len(e[0])) for e in entries]
        return (torch.tensor(rows, dtype=torch.int32).reshape(len(entries), columns),
                torch.tensor([e[1] for e in entries], dtype=torch.int32))

    def _take(self) -> int:
        p = self._free.pop()
        self._users[p] = 1
        return p

    def _drop(self, p: int) -> None:
        self._users[p] -= 1
        if not self._users[p]:
            self._free.append(p)


def copy_lists(copies, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """(src, dst) for ops.kv8_copy_pages of extend()'s or compact()'s copies."""
    pairs = torch.tensor(list(copies), dtype=torch.int32).reshape(-1, 2)
    return pairs[:, 0].contiguous().to(device), pairs[:, 1].contiguous().to(device)
