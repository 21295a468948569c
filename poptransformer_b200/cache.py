"""Sequence slots and cache pages for decoders whose sequences have positions of their own.

A slot is a row of the page table and the place of a sequence's recurrent state; pages hold `page_size` positions of every
attention layer's keys and values (the pools of all layers share one page numbering).  Slots and pages are handed out on demand
and returned when a sequence ends.  Sequences that forked share the pages that both have filled; a page is handed back when its last
owner returns it, and nobody writes to a page that has two.  Nothing is cleared on return: kernels read no key beyond a sequence's own position and
ignore a slot's old recurrent state at position 0.
"""
import torch

from ._lib import PtError


class SequenceSlots:
    def __init__(self, max_seqs, max_len, page_size=64, n_pages=None, device="cuda"):
        self.max_seqs, self.max_len, self.page_size, self.device = max_seqs, max_len, page_size, device
        self.max_pages = -(-max_len // page_size)
        self.n_pages = max_seqs * self.max_pages if n_pages is None else n_pages
        self._free_slots = list(range(max_seqs - 1, -1, -1))
        self._free_pages = list(range(self.n_pages - 1, -1, -1))
        self._pages = {}                       # slot -> pages in position order
        self._owners = {}                      # page -> slots that have it, where there are several
        self.length = {}                       # slot -> positions cached so far
        self.page_table = torch.zeros((max_seqs, self.max_pages), dtype=torch.int32, device=device)

    @property
    def free_slots(self):
        return len(self._free_slots)

    @property
    def free_pages(self):
        return len(self._free_pages)

    def open(self):
        """A slot for a new sequence (length 0, no pages yet)."""
        if not self._free_slots:
            raise PtError(f"all {self.max_seqs} sequence slots are in use")
        slot = self._free_slots.pop()
        self._pages[slot], self.length[slot] = [], 0
        return slot

    def extend(self, slot, n):
        """Makes room for `n` more positions and counts them as cached; returns the first of them."""
        start = self.length[slot]
        if start + n > self.max_len:
            raise PtError(f"a sequence of {start} + {n} tokens exceeds max_len={self.max_len}")
        pages = self._pages[slot]
        need = -(-(start + n) // self.page_size) - len(pages)
        if need > len(self._free_pages):
            raise PtError(f"{need} more cache pages needed, {len(self._free_pages)} of {self.n_pages} are free")
        if need > 0:
            first = len(pages)
            pages.extend(self._free_pages.pop() for _ in range(need))
            self.page_table[slot, first:len(pages)] = torch.tensor(pages[first:], dtype=torch.int32).to(self.device)
        self.length[slot] = start + n
        return start

    def _set_table(self, slot, first, pages):
        if pages:
            self.page_table[slot, first:first + len(pages)] = torch.tensor(pages, dtype=torch.int32).to(self.device)

    def _release(self, pages):
        for page in pages:
            if page in self._owners:
                self._owners[page] -= 1
                if self._owners[page] == 1:
                    del self._owners[page]
            else:
                self._free_pages.append(page)

    def fork(self, slot, n=None):
        """A new sequence that begins with the first `n` positions of another (default: all of them).  Full pages are shared.  Returns the
        new slot and the (source, destination) pages that have to be copied in every layer (PagePools.copy) before either sequence goes on: the
        one that is not full, if there is one."""
        length = self.length[slot]
        n = length if n is None else int(n)
        if not 0 <= n <= length:
            raise PtError(f"fork: {n} of {length} positions")
        full, rest = divmod(n, self.page_size)
        if not self._free_slots:
            raise PtError(f"all {self.max_seqs} sequence slots are in use")
        if rest and not self._free_pages:
            raise PtError(f"1 more cache page needed, 0 of {self.n_pages} are free")
        new = self._free_slots.pop()
        pages, copies = self._pages[slot][:full], []
        for page in pages:
            self._owners[page] = self._owners.get(page, 1) + 1
        if rest:
            copies.append((self._pages[slot][full], self._free_pages.pop()))
            pages = pages + [copies[0][1]]
        self._pages[new], self.length[new] = pages, n
        self._set_table(new, 0, pages)
        return new, copies

    def truncate(self, slot, n):
        """Keeps the first `n` positions of a sequence (drafted tokens that were refused go this way) and hands the pages behind them back.  Returns the
        (source, destination) pages that have to be copied before any sequence goes on: its last one, where that is shared and not full (the other owner may then write to it)."""
        length, n = self.length[slot], int(n)
        if not 0 <= n <= length:
            raise PtError(f"truncate: {n} of {length} positions")
        pages, keep, copies = self._pages[slot], -(-n // self.page_size), []
        if n % self.page_size and pages[keep - 1] in self._owners:
            gone = pages[keep:]
            if not self._free_pages and all(p in self._owners for p in gone):
                raise PtError(f"1 more cache page needed, 0 of {self.n_pages} are free")
        self._release(reversed(pages[keep:]))
        del pages[keep:]
        if n % self.page_size and pages[-1] in self._owners:
            copies.append((pages[-1], self._free_pages.pop()))
            self._release([pages[-1]])
            pages[-1] = copies[0][1]
            self._set_table(slot, keep - 1, pages[-1:])
        self.length[slot] = n
        return copies

    def compact(self):
        """Moves the pages in use to the lowest numbers.  Returns the (source, destination) pages that have to be copied in every layer before
        any sequence goes on; from the number of pages in use on, the pool is then free."""
        used = sorted({p for pages in self._pages.values() for p in pages})
        holes = sorted(set(range(len(used))) - set(used))
        moves = dict(zip((p for p in used if p >= len(used)), holes))
        for slot, pages in self._pages.items():
            if any(p in moves for p in pages):
                pages[:] = [moves.get(p, p) for p in pages]
                self._set_table(slot, 0, pages)
        self._owners = {moves.get(p, p): n for p, n in self._owners.items()}
        self._free_pages = list(range(self.n_pages - 1, len(used) - 1, -1))
        return list(moves.items())

    def close(self, slot):
        """Ends a sequence: its slot and pages can be used by the next one."""
        self._release(reversed(self._pages.pop(slot)))
        del self.length[slot]
        self._free_slots.append(slot)

    def close_all(self):
        for slot in list(self._pages):
            self.close(slot)
        self._free_slots.sort(reverse=True)    # the next open() calls return 0, 1, 2, ...
