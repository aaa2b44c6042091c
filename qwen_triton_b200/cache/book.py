"""Host-side bookkeeping of the cache: which sequence holds which slot and which pages.

A *slot* belongs to one live sequence: it indexes the fixed-size per-sequence state and carries
the sequence's length and, for each cache group, the list of pages that hold its keys and values.
Pages are ``page_tokens`` positions long.  A group that keeps all keys takes pages as the sequence
grows; a group that keeps a window of them takes at most ``ring_pages`` and reuses them as a ring.
Slots and pages go back to their free lists when the sequence ends and are handed out again.

A sequence may start with the leading whole pages of another one (``alloc(prefix_of, tokens)``): such a page is held by
several slots, nobody writes to it any more (a sequence writes at its length and beyond), and it goes back to the free list when the
last of them ends.  Groups that keep a window reuse their pages and cannot be shared.

No device memory is touched here, so the invariants (no slot or page lost, held twice or freed
twice) can be checked without a GPU.  The reference keeps one length for the whole batch and grows
its tensors by reallocation (qwen_triton/modules/cache.py:21-65).
"""
from __future__ import annotations

from dataclasses import dataclass, field


class CacheError(RuntimeError):
    pass


class CacheFull(CacheError):
    """No free slot or page is left for the request."""


@dataclass(frozen=True)
class GroupGeometry:
    """One cache group as the book sees it: its page pool and, for a windowed group, its ring."""

    num_pages: int
    ring_pages: int = 0      # 0: keeps every position; else pages of the ring a sequence cycles through


@dataclass
class _Slot:
    length: int = 0
    pages: list[list[int]] = field(default_factory=list)   # per group
    shared: int = 0                                        # leading pages taken from another slot


class CacheBook:
    def __init__(self, num_slots: int, page_tokens: int, groups: list[GroupGeometry], max_seq_len: int) -> None:
        if num_slots <= 0 or page_tokens <= 0 or max_seq_len <= 0:
            raise ValueError("num_slots, page_tokens and max_seq_len must be positive")
        self.num_slots = num_slots
        self.page_tokens = page_tokens
        self.groups = list(groups)
        self.max_seq_len = max_seq_len
        self._free_slots = list(range(num_slots - 1, -1, -1))         # pop() hands out the lowest number first
        self._free_pages = [list(range(g.num_pages - 1, -1, -1)) for g in self.groups]
        self._live: dict[int, _Slot] = {}
        self._holders: list[dict[int, int]] = [{} for _ in self.groups]   # pages held by more than one slot, and by how many
        self._sharers = 0                                                 # live slots that started with another one's pages
        self._grouped: tuple[tuple[int, ...], list] | None = None         # slots of the last ``shared_groups`` and its result, until a slot comes or goes

    # ------------------------------------------------------------------ slots
    def alloc(self, prefix_of: int | None = None, tokens: int = 0) -> int:
        """A slot for a new sequence, empty, or with the first ``tokens`` (whole pages) of the sequence in ``prefix_of``."""
        source = None
        if prefix_of is not None:
            source = self._entry(prefix_of)
            if tokens <= 0 or tokens % self.page_tokens or tokens > source.length:
                raise CacheError(f"slot {prefix_of}: {tokens} of its {source.length} tokens are not whole pages of {self.page_tokens}")
            if any(g.ring_pages for g in self.groups):
                raise CacheError("pages of a windowed cache group are used again and cannot be shared")
        if not self._free_slots:
            raise CacheFull(f"all {self.num_slots} sequence slots are in use")
        slot = self._free_slots.pop()
        self._grouped = None
        entry = self._live[slot] = _Slot(0, [[] for _ in self.groups])
        if source is not None:
            entry.length, entry.shared = tokens, tokens // self.page_tokens
            self._sharers += 1
            for held, holders, pages in zip(source.pages, self._holders, entry.pages):
                pages.extend(held[:entry.shared])
                for page in pages:
                    holders[page] = holders.get(page, 1) + 1
        return slot

    def free(self, slot: int) -> None:
        entry = self._live.pop(slot, None)
        if entry is None:
            raise CacheError(f"slot {slot} is not in use (freed twice, or never allocated)")
        self._grouped = None
        self._sharers -= entry.shared > 0
        for group, pages in enumerate(entry.pages):
            holders = self._holders[group]
            if not holders:
                self._free_pages[group].extend(reversed(pages))
                continue
            for page in reversed(pages):
                count = holders.get(page, 1)
                if count == 1:
                    self._free_pages[group].append(page)
                elif count == 2:
                    del holders[page]
                else:
                    holders[page] = count - 1
        self._free_slots.append(slot)

    def is_live(self, slot: int) -> bool:
        return slot in self._live

    def live_slots(self) -> list[int]:
        return sorted(self._live)

    def length(self, slot: int) -> int:
        return self._entry(slot).length

    def _entry(self, slot: int) -> _Slot:
        try:
            return self._live[slot]
        except KeyError:
            raise CacheError(f"slot {slot} is not in use") from None

    # ------------------------------------------------------------------ pages
    def pages_needed(self, group: int, length: int) -> int:
        pages = -(-length // self.page_tokens)
        ring = self.groups[group].ring_pages
        return min(pages, ring) if ring else pages

    def can_hold(self, lengths_by_slot: dict[int, int]) -> bool:
        """Whether every slot can grow to the given length at once."""
        for group in range(len(self.groups)):
            extra = 0
            for slot, length in lengths_by_slot.items():
                extra += max(0, self.pages_needed(group, length) - len(self._entry(slot).pages[group]))
            if extra > len(self._free_pages[group]):
                return False
        return True

    def extend(self, slot: int, new_length: int) -> None:
        """Make room for positions below ``new_length`` and record the new length."""
        entry = self._entry(slot)
        if new_length < entry.length:
            raise CacheError(f"slot {slot}: a sequence cannot shrink ({entry.length} -> {new_length})")
        if new_length > self.max_seq_len:
            raise CacheFull(f"slot {slot}: {new_length} tokens exceed the longest sequence the cache holds ({self.max_seq_len})")
        wanted = [self.pages_needed(g, new_length) - len(entry.pages[g]) for g in range(len(self.groups))]
        for group, count in enumerate(wanted):
            if count > len(self._free_pages[group]):
                raise CacheFull(f"cache group {group}: {count} more pages needed, {len(self._free_pages[group])} free")
        for group, count in enumerate(wanted):
            for _ in range(max(0, count)):
                entry.pages[group].append(self._free_pages[group].pop())
        entry.length = new_length

    def pages(self, slot: int, group: int) -> list[int]:
        return self._entry(slot).pages[group]

    def shared_groups(self, slots: list[int]) -> list[tuple[list[int], int]]:
        """Which of ``slots`` share leading tokens: (places in ``slots``, tokens that all of them hold on the same pages) for every group of two and more, and
        one group of the rest with 0 tokens, if there is a rest.  Empty where none do.  Where prefixes of prefixes are shared there are several ways to group
        sequences; the one with the most tokens that members hold beside another one, sum of (members - 1) * tokens, is taken."""
        if not self._sharers or not self.groups:
            return []
        # pages that a sequence adds as it grows are its own, so that step after step of the same sequences has the same groups
        if self._grouped is None or self._grouped[0] != tuple(slots):
            self._grouped = tuple(slots), self._find_groups(slots)
        return [(list(places), tokens) for places, tokens in self._grouped[1]]

    def _find_groups(self, slots: list[int]) -> list[tuple[list[int], int]]:
        entries = [self._entry(slot) for slot in slots]
        pages = [entry.pages[0] for entry in entries]
        # A tree: a node's places agree on the pages in front of its depth and go apart there, into places by themselves and branches, which are nodes again.
        # A page that two sequences both hold at a place has the same pages in front of it in both.
        nodes: list[tuple[int, list[int], list[int], tuple[int, ...]]] = []       # (depth, places by themselves, branches, depths of the nodes above)
        work = [(-1, list(range(len(slots))))]
        while work:
            parent, places = work.pop()
            depth, above = 0, ()
            if parent >= 0:
                depth, above = self._common_pages(entries, places, nodes[parent][0] + 1), (*nodes[parent][3], nodes[parent][0])
                nodes[parent][2].append(len(nodes))
            branches: dict[int, list[int]] = {}
            alone = []
            for place in places:
                if len(pages[place]) > depth:
                    branches.setdefault(pages[place][depth], []).append(place)
                else:
                    alone.append(place)
            for branch in branches.values():
                if len(branch) == 1:
                    alone += branch
                else:
                    work.append((len(nodes), branch))
            nodes.append((depth, alone, [], above))
        # From the leaves on: what a node's places are worth where each may join a group of an upper node's depth, and whether the node has a group of its own
        # then, which reads its pages once itself.
        worth: list[dict[int, tuple[int, bool]]] = [{} for _ in nodes]
        for node in reversed(range(len(nodes))):
            depth, alone, branches, above = nodes[node]

            def joined(to: int) -> int:
                return len(alone) * to + sum(worth[branch][to][0] for branch in branches)
            own = joined(depth) - depth
            for upper in above or (0,):
                without = joined(upper)
                worth[node][upper] = (max(own, without), own > without)
        members: dict[int, list[int]] = {}
        work = [(0, -1)]                                          # a node, and the node whose group its places join (-1: none)
        while work:
            node, group = work.pop()
            depth, alone, branches, above = nodes[node]
            if worth[node][nodes[group][0] if group >= 0 else 0][1]:
                group = node
            members.setdefault(group, []).extend(alone)
            work += [(branch, group) for branch in branches]
        groups = sorted((sorted(places), nodes[node][0] * self.page_tokens) for node, places in members.items() if node >= 0)
        if not groups:
            return []
        rest = sorted(members.get(-1, ()))
        return groups + [(rest, 0)] if rest else groups

    @staticmethod
    def _common_pages(entries: list[_Slot], places: list[int], low: int) -> int:
        """Leading pages that the sequences at ``places`` all hold, of which the first ``low`` are known to be."""
        lists = [entries[place].pages[0] for place in places]
        first, high = lists[0], min(len(pages) for pages in lists)

        def agree(n: int) -> bool:
            page = first[n - 1]
            return all(pages[n - 1] == page for pages in lists)

        # what they took from another sequence is common to them all as a rule, and no more
        guess = min(high, max(low, min((entries[place].shared for place in places if entries[place].shared), default=low)))
        if not agree(guess):
            high = guess - 1
        elif guess == high or not agree(guess + 1):
            return guess
        else:
            low = guess + 1
        while low < high:
            middle = (low + high + 1) // 2
            if agree(middle):
                low = middle
            else:
                high = middle - 1
        return low

    def free_pages(self, group: int) -> int:
        return len(self._free_pages[group])

    def free_slot_count(self) -> int:
        return len(self._free_slots)

    # ------------------------------------------------------------------ checks
    def check(self) -> None:
        """Raise if a slot or page is lost or held twice."""
        slots = self._free_slots + list(self._live)
        if sorted(slots) != list(range(self.num_slots)):
            raise CacheError(f"slot accounting is broken: {sorted(slots)}")
        for group, geometry in enumerate(self.groups):
            held: dict[int, int] = {}
            for entry in self._live.values():
                for page in entry.pages[group]:
                    held[page] = held.get(page, 0) + 1
            if {page: n for page, n in held.items() if n > 1} != self._holders[group]:
                raise CacheError(f"page accounting of group {group} is broken: pages held more than once")
            everything = self._free_pages[group] + list(held)
            if sorted(everything) != list(range(geometry.num_pages)):
                raise CacheError(f"page accounting of group {group} is broken")
