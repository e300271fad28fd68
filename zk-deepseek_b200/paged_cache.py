"""The cache of a model whose sequences share one pool of pages: what `SequenceCache` keeps per slot, kept in pages of a fixed
number of positions, so that a sequence takes only what it has grown to, and sequences that begin alike hold those
pages once.

A slot is a row of the page table and a block of recurrent state.  Every page has a count of the slots that hold it.  `fork`
hands a second slot the same pages; a step that writes into a page which others hold as well gets a copy of the part
that is filled.  `compact` moves the pages in use to the front of the pool.  Page numbers are kept on the host; a step takes the
rows of its slots with it.
"""
import heapq

import torch

try:
    from .sequence_cache import CacheFull
except ImportError:  # pragma: no cover - this directory first on sys.path
    from sequence_cache import CacheFull


def _copy_pages(buffers, source, target, positions=None):
    try:
        from . import float_kernel as K
    except ImportError:  # pragma: no cover
        import float_kernel as K
    K.copy_pages(buffers, source, target, positions=positions)


def check_pages(page, pages=None):
    if page not in (8, 16, 32, 64, 128, 256, 512, 1024):
        raise ValueError("pages of %r positions: a power of two from 8 to 1024" % (page,))
    if pages is not None and pages < 1:
        raise ValueError("a pool of %d pages" % pages)


class PagedCache:
    def __init__(self, pitches, owners, slots, capacity, dtype, device, states=(), page=64, pages=None, copy=_copy_pages):
        """pitches, owners, slots, states: as for `SequenceCache`; capacity: most positions of a sequence; page: positions of a
        page; pages: of the pool (default: enough for all slots at their capacity); copy: what copies pages"""
        check_pages(page, pages)
        self.slots, self.capacity, self.page, self.copy = slots, capacity, page, copy
        self.columns = -(-capacity // page)
        self.pages = slots * self.columns if pages is None else pages
        check_pages(page, self.pages)
        self.owners = list(owners)
        self.buffers = [None if p is None else torch.zeros(self.pages, page, p, dtype=dtype, device=device) for p in pitches]
        for i, o in enumerate(self.owners):
            if o is not None and self.buffers[o] is None:
                raise ValueError("layer %d reads the entries of layer %d, which stores none" % (i, o))
        self.states = [{n: torch.zeros((slots,) + tuple(shape), dtype=dt, device=device) for n, (shape, dt) in s.items()} for s in states]
        self._free, self._taken = list(range(slots - 1, -1, -1)), [False] * slots
        self.lengths = [0] * slots
        self.held = [[] for _ in range(slots)]         # page numbers of every slot
        self.counts = [0] * self.pages
        self._spare = list(range(self.pages))          # a heap: the lowest page first
        self.version = 0                               # counts the changes of any table row

    def buffer(self, layer):
        return self.buffers[self.owners[layer]]

    def state(self, layer, name):
        return self.states[layer][name]

    def free_slots(self):
        return len(self._free)

    def free_pages(self):
        return len(self._spare)

    def bytes(self):
        return sum(t.numel() * t.element_size() for t in [b for b in self.buffers if b is not None] + [t for s in self.states for t in s.values()])

    def table(self, slots):
        """int32 [len(slots), columns]: the page numbers of these slots, -1 where they hold none"""
        t = torch.full((len(slots), self.columns), -1, dtype=torch.int32)
        for row, s in zip(t, slots):
            row[:len(self.held[s])] = torch.tensor(self.held[s], dtype=torch.int32)
        return t

    # -- slots and pages -------------------------------------------------------------------------------------------
    def _used(self, slot):
        if not 0 <= slot < self.slots or not self._taken[slot]:
            raise ValueError("slot %d is not in use" % slot)

    def _take(self):
        page = heapq.heappop(self._spare)
        self.counts[page] = 1
        return page

    def _give(self, pages):
        for p in pages:
            self.counts[p] -= 1
            if not self.counts[p]:
                heapq.heappush(self._spare, p)

    def acquire(self):
        if not self._free:
            raise CacheFull("all %d cache slots are in use" % self.slots)
        slot = self._free.pop()
        self.lengths[slot], self._taken[slot] = 0, True
        return slot

    def release(self, slot):
        self._used(slot)
        self._give(self.held[slot])
        self.held[slot], self.lengths[slot], self._taken[slot] = [], 0, False
        self._free.append(slot)
        self.version += 1

    def extend(self, slot, start, n):
        self.extend_all([slot], start, n)

    def extend_all(self, slots, start, n):
        """the step about to run writes positions start .. start + n - 1 of these slots; nothing changes where it does not fit or a copy
        fails"""
        if len(set(slots)) != len(slots):
            raise ValueError("a slot twice in one step")
        for s in slots:
            self._used(s)
            if start != self.lengths[s]:
                raise ValueError("slot %d holds %d positions, the step starts at %d" % (s, self.lengths[s], start))
        if start + n > self.capacity:
            raise CacheFull("%d positions do not fit a sequence of %d" % (start + n, self.capacity))
        if n == 0:
            return
        last, inside = start // self.page, start % self.page
        # the page that the step writes on in: of those who hold it, all but one get a copy
        copies, seen = [], {}
        if inside:
            for s in slots:
                p = self.held[s][last]
                seen[p] = seen.get(p, 0) + 1
                if seen[p] < self.counts[p]:
                    copies.append(s)
        more = -(-(start + n) // self.page) - -(-start // self.page)
        if len(copies) + more * len(slots) > len(self._spare):
            raise CacheFull("%d pages are free, the step takes %d" % (len(self._spare), len(copies) + more * len(slots)))
        source, target = [self.held[s][last] for s in copies], [self._take() for _ in copies]
        if source:
            try:
                self.copy(self._pools(), source, target, positions=inside)
            except Exception:
                self._give(target)
                raise
            for s, p in zip(copies, target):
                self.held[s][last] = p
            self._give(source)
        for s in slots:
            self.held[s].extend(self._take() for _ in range(more))
            self.lengths[s] = start + n
        if source or more:
            self.version += 1

    def truncate(self, slot, length):
        """forget the positions from `length` on; a recurrent state can only be forgotten as a whole"""
        self._used(slot)
        if not 0 <= length <= self.lengths[slot]:
            raise ValueError("slot %d holds %d positions" % (slot, self.lengths[slot]))
        if any(self.states) and length not in (0, self.lengths[slot]):
            raise ValueError("the recurrent state of slot %d stands at position %d" % (slot, self.lengths[slot]))
        keep = -(-length // self.page)
        self._give(self.held[slot][keep:])
        del self.held[slot][keep:]
        self.lengths[slot] = length
        self.version += 1

    def fork(self, slot):
        """a new slot that stands where this one does, on the same pages"""
        self._used(slot)
        new = self.acquire()
        self.held[new], self.lengths[new] = list(self.held[slot]), self.lengths[slot]
        for p in self.held[new]:
            self.counts[p] += 1
        self.version += 1
        if self.lengths[slot]:
            try:
                copy_states(self.copy, self.states, slot, new)
            except Exception:
                self.release(new)
                raise
        return new

    def compact(self):
        """moves the pages in use to the front of the pool; returns how many moved"""
        used = sum(1 for c in self.counts if c)
        target = [p for p in range(used) if not self.counts[p]]
        source = [p for p in range(used, self.pages) if self.counts[p]]
        if not source:
            return 0
        self.copy(self._pools(), source, target)
        to = dict(zip(source, target))
        for pages in self.held:
            pages[:] = [to.get(p, p) for p in pages]
        for s, t in to.items():
            self.counts[t], self.counts[s] = self.counts[s], 0
        self._spare = list(range(used, self.pages))
        self.version += 1
        return len(source)

    def _pools(self):
        return [b for b in self.buffers if b is not None]


def copy_states(copy, states, source, target):
    """the recurrent state of one slot over another's, in every layer"""
    blocks = [t.view(t.shape[0], 1, t[0].numel()) for s in states for t in s.values()]
    if blocks:
        copy(blocks, [source], [target])
