"""Pages held by several sequences: the book's accounting, which sequences share, and the generation loop's use of it (no GPU)."""
import random

import numpy as np
import pytest

from qwen_triton_b200.cache import CacheBook, CacheError, CacheFull, GroupGeometry, SequenceCache
from qwen_triton_b200.engine.generate import common_prefix, generate, plan_batches
from qwen_triton_b200.engine.step import shared_shape
from qwen_triton_b200.parts.base import KVRequest, StateRequest
from qwen_triton_b200.sampling import SamplingParams, uniform_for
from qwen_triton_b200.sampling.sampler import uniforms_for
from test_generate_loop import ArgmaxSampler, ScriptedEngine


def make_book(slots=8, pages=20, groups=1):
    return CacheBook(slots, 64, [GroupGeometry(pages) for _ in range(groups)], 4096)


def test_a_sequence_starts_with_another_ones_pages():
    book = make_book(groups=2)
    a = book.alloc()
    book.extend(a, 200)
    b = book.alloc(a, 128)
    assert book.length(b) == 128
    for group in range(2):
        assert book.pages(b, group) == book.pages(a, group)[:2] and book.free_pages(group) == 16
    book.extend(b, 130)                                    # its own page behind the shared ones
    assert book.pages(b, 0)[2] != book.pages(a, 0)[2]
    book.check()
    book.free(a)                                           # the shared pages stay with b
    assert book.free_pages(0) == 17
    book.check()
    book.free(b)
    assert book.free_pages(0) == book.free_pages(1) == 20
    book.check()


def test_what_cannot_be_shared():
    book = make_book(slots=2)
    a = book.alloc()
    book.extend(a, 100)
    for tokens in (0, -64, 63, 100, 128):
        with pytest.raises(CacheError, match="whole pages"):
            book.alloc(a, tokens)
    with pytest.raises(CacheError, match="not in use"):
        book.alloc(1, 64)
    book.alloc(a, 64)
    with pytest.raises(CacheFull):
        book.alloc(a, 64)
    windowed = CacheBook(4, 64, [GroupGeometry(8), GroupGeometry(8, 2)], 4096)
    slot = windowed.alloc()
    windowed.extend(slot, 64)
    with pytest.raises(CacheError, match="windowed"):
        windowed.alloc(slot, 64)
    windowed.check()
    common = dict(max_tokens=512, max_seq_len=512, dtype=None, device=None, allocate=False)
    import torch
    common["dtype"] = torch.float32
    assert SequenceCache([KVRequest(2, 16)], [None], **common).can_share
    assert not SequenceCache([KVRequest(2, 16, 64)], [None], **common).can_share


def test_random_lives_of_sharing_sequences():
    rng = random.Random(5)
    book = make_book(slots=12, pages=60, groups=2)
    for _ in range(2000):
        live = book.live_slots()
        what = rng.random()
        try:
            if what < 0.25 or not live:
                book.alloc()
            elif what < 0.5:
                source = rng.choice(live)
                whole = book.length(source) // 64
                if whole:
                    book.alloc(source, 64 * rng.randint(1, whole))
            elif what < 0.8:
                slot = rng.choice(live)
                book.extend(slot, book.length(slot) + rng.randint(0, 150))
            else:
                book.free(rng.choice(live))
        except CacheFull:
            book.free(rng.choice(book.live_slots()))
        book.check()
        live = book.live_slots()
        rng.shuffle(live)
        groups = book.shared_groups(live)
        if groups:
            assert sorted(place for places, _ in groups for place in places) == list(range(len(live)))
        for places, tokens in groups:
            pages = [tuple(book.pages(live[p], 0)[:tokens // 64]) for p in places]
            assert len(set(pages)) == 1 if tokens else True
            assert tokens == 0 or (len(places) > 1 and all(book.length(live[p]) >= tokens for p in places))
    for slot in book.live_slots():
        book.free(slot)
    assert book.shared_groups([]) == [] and book.free_pages(0) == 60
    book.check()


def test_groups_of_sequences_that_share():
    book = make_book()
    a, other = book.alloc(), book.alloc()
    book.extend(a, 200)
    book.extend(other, 70)
    assert book.shared_groups([a, other]) == []
    b, c = book.alloc(a, 192), book.alloc(a, 64)
    assert book.shared_groups([b, other, a]) == [([0, 2], 192), ([1], 0)]
    assert book.shared_groups([c, b]) == [([0, 1], 64)]
    assert book.shared_groups([b, other]) == []             # alone, each of them
    book.free(a)
    assert book.shared_groups([c, b]) == [([0, 1], 64)]


def test_shapes_are_rounded_up():
    assert shared_shape([([0, 2, 3], 192), ([1], 0)], [200, 90, 260, 193]) == (2, 4, 256, 128)
    assert shared_shape([([0, 1], 1024)], [1025, 1030]) == (1, 2, 1024, 64)
    assert shared_shape([([0, 1], 1088)], [1100, 1200]) == (1, 2, 2048, 128)


def test_the_prefix_of_all_prompts():
    long = list(range(300))
    assert common_prefix([long, long[:200] + [7], long], 64) == 192
    assert common_prefix([long[:128], long], 64) == 64       # a token of each is left over
    assert common_prefix([long[:129], long], 64) == 128
    assert common_prefix([long], 64) == 0 and common_prefix([[1] + long, long], 64) == 0


def test_batches_hold_what_is_shared_once():
    lengths = [300] * 6
    assert plan_batches(lengths, 20, page_tokens=64, total_pages=12, num_slots=8, max_seq_len=4096) == [[0, 1], [2, 3], [4, 5]]
    assert plan_batches(lengths, 20, page_tokens=64, total_pages=12, num_slots=8, max_seq_len=4096, shared_tokens=256) == [[0, 1, 2, 3, 4, 5]]
    assert plan_batches(lengths, 20, page_tokens=64, total_pages=7, num_slots=8, max_seq_len=4096, shared_tokens=256) == [[0, 1, 2], [3, 4, 5]]


class SharingEngine(ScriptedEngine):
    """Counts what each sequence holds; a shared start is taken from a sequence that holds it."""

    can_share = True

    def __init__(self, **kw):
        super().__init__(**kw)
        self.shared: list[tuple[int, int, int]] = []

    def new_sequence(self, prefix_of=None, tokens=None):
        slot = super().new_sequence()
        if prefix_of is not None:
            assert tokens % self.page_tokens == 0 and 0 < tokens <= self.lengths[prefix_of]
            self.lengths[slot] = tokens
            self.shared.append((slot, prefix_of, tokens))
        return slot

    def step(self, entries):
        if len(entries) == 1 and not entries[0].want:
            self.steps.append([(entries[0].slot, len(entries[0].tokens))])
            self.lengths[entries[0].slot] += len(entries[0].tokens)
            return None
        return super().step(entries)


def test_generation_runs_the_shared_prefix_once():
    prompts = [[1, 2, 3, 4, 5, 6, 7, 8, 9, 10 + i] for i in range(3)]
    plain = generate(ScriptedEngine(total_pages=30, vocab=90), prompts, max_new_tokens=3, sampler=ArgmaxSampler())
    engine = SharingEngine(total_pages=30, vocab=90)
    shared = generate(engine, prompts, max_new_tokens=3, sampler=ArgmaxSampler(), share_prefix=True)
    assert [r.tokens for r in shared] == [r.tokens for r in plain]
    assert engine.steps[0] == [(0, 8)] and engine.steps[1] == [(0, 2), (1, 2), (2, 2)]
    assert engine.shared == [(1, 0, 8), (2, 0, 8)] and not engine.lengths
    engine = SharingEngine(total_pages=30, vocab=90)          # not asked for, nothing shared
    generate(engine, prompts, max_new_tokens=3, sampler=ArgmaxSampler())
    assert engine.steps[0] == [(0, 10), (1, 10), (2, 10)] and not engine.shared


def test_parameters_of_each_request():
    class Sampler:
        def __init__(self):
            self.seen = []

        def sample(self, logits, params, requests, steps):
            self.seen.append((params, list(requests)))
            return logits.argmax(dim=-1).tolist()

    params = [SamplingParams(temperature=0.5, seed=i, min_p=0.1) for i in range(3)]
    sampler = Sampler()
    generate(ScriptedEngine(), [[46], [10], [20]], max_new_tokens=4, sampling=params, sampler=sampler)
    assert sampler.seen[0] == (params, [0, 1, 2]) and sampler.seen[-1] == (params[1:], [1, 2])      # the first ends early
    with pytest.raises(ValueError, match="sampling parameters"):
        generate(ScriptedEngine(), [[1], [2]], sampling=params, sampler=sampler)
    with pytest.raises(ValueError, match="min_p"):
        SamplingParams(min_p=1.5)


def test_uniform_numbers_of_many_rows():
    rng = random.Random(1)
    rows = [(rng.getrandbits(64), rng.randrange(1 << 20), rng.randrange(1 << 16)) for _ in range(200)] + [(0, 0, 0), ((1 << 64) - 1, 5, 7)]
    got = uniforms_for(np.array([r[0] for r in rows], dtype=np.uint64), np.array([r[1] for r in rows]), np.array([r[2] for r in rows]))
    assert got.dtype == np.float32 and got.tolist() == [uniform_for(*r) for r in rows]


def worth_of(groups):
    return sum((len(places) - 1) * tokens for places, tokens in groups if tokens)


def test_prefixes_of_prefixes():
    """A short start that all hold beside long ones that some hold: each sequence is grouped where more is shared."""
    book = make_book(slots=24, pages=400)
    deep = book.alloc()
    book.extend(deep, 3000)
    drafts = [book.alloc(deep, 2560) for _ in range(4)]
    assert book.shared_groups([deep, *drafts]) == [([0, 1, 2, 3, 4], 2560)]
    shallow = book.alloc(deep, 64)                          # one more, that took a page only: the others stay together
    assert book.shared_groups([deep, shallow, *drafts]) == [([0, 2, 3, 4, 5], 2560), ([1], 0)]
    also = book.alloc(deep, 64)
    assert book.shared_groups([also, deep, shallow, *drafts]) == [([0, 2], 64), ([1, 3, 4, 5, 6], 2560)]
    assert book.shared_groups([deep, shallow]) == [([0, 1], 64)]


def test_a_continuation_of_one_of_two_users_behind_a_system_prompt():
    book = make_book(slots=8, pages=200)
    system = book.alloc()
    book.extend(system, 128)
    users = [book.alloc(system, 128) for _ in range(2)]
    for user in users:
        book.extend(user, 2600)
    continued = [book.alloc(user, 2560) for user in users]
    assert book.shared_groups([users[0], continued[0]]) == [([0, 1], 2560)]
    assert book.shared_groups([*users, *continued]) == [([0, 2], 2560), ([1, 3], 2560)]
    book.free(users[0])
    assert book.shared_groups([continued[0], users[1], continued[1], system]) == [([0, 3], 128), ([1, 2], 2560)]


def test_groups_follow_slots_that_come_and_go():
    """The same numbers of slots may be other sequences, and what a caller does to a result is its own."""
    book = make_book(slots=3, pages=60)
    a = book.alloc()
    book.extend(a, 200)
    b, c = book.alloc(a, 192), book.alloc(a, 64)
    first = book.shared_groups([a, b, c])
    assert first == [([0, 1], 192), ([2], 0)]
    first[-1][0].append(7)
    book.extend(c, 500)
    assert book.shared_groups([a, b, c]) == [([0, 1], 192), ([2], 0)]
    book.free(b)
    book.free(c)
    assert (book.alloc(), book.alloc(a, 128)) == (c, b)
    book.extend(c, 100)
    assert book.shared_groups([a, b, c]) == [([0, 1], 128), ([2], 0)]
    with pytest.raises(CacheError, match="not in use"):
        book.free(c)
        book.shared_groups([a, b, c])


def partitions(items):
    if not items:
        yield []
        return
    first, rest = items[0], items[1:]
    for partition in partitions(rest):
        yield [[first], *partition]
        for i in range(len(partition)):
            yield [*partition[:i], [first, *partition[i]], *partition[i + 1:]]


def test_the_grouping_is_the_best_one():
    """Random families of up to seven sequences against every way to part them."""
    rng = random.Random(9)
    for _ in range(150):
        book = make_book(slots=8, pages=200)
        for _ in range(rng.randint(2, 7)):
            live = [s for s in book.live_slots() if book.length(s) >= 64]
            if live and rng.random() < 0.85:
                source = rng.choice(live)
                slot = book.alloc(source, 64 * rng.randint(1, book.length(source) // 64))
            else:
                slot = book.alloc()
            book.extend(slot, book.length(slot) + rng.randint(0, 400))
        slots = book.live_slots()
        rng.shuffle(slots)
        pages = [book.pages(s, 0) for s in slots]

        def common(places):
            n = 0
            while all(len(pages[p]) > n and pages[p][n] == pages[places[0]][n] for p in places):
                n += 1
            return 64 * n
        groups = book.shared_groups(slots)
        for places, tokens in groups:
            assert tokens in (0, common(places))
        most = max(worth_of([(places, common(places)) for places in partition]) for partition in partitions(list(range(len(slots)))))
        assert worth_of(groups) == most
        assert not groups or sorted(p for places, _ in groups for p in places) == list(range(len(slots)))


def test_requests_that_are_alike_are_one_kind():
    """A list of equal parameters is the same call as one for all; a list that differs stays a list to the end."""
    class Sampler:
        def __init__(self):
            self.seen = []

        def sample(self, logits, params, requests, steps):
            self.seen.append(params)
            return logits.argmax(dim=-1).tolist()

    one = SamplingParams(temperature=0.5, seed=3)
    sampler = Sampler()
    generate(ScriptedEngine(), [[1], [2], [3]], max_new_tokens=2, sampling=[SamplingParams(temperature=0.5, seed=3) for _ in range(3)], sampler=sampler)
    assert sampler.seen and all(params == one for params in sampler.seen)
    sampler = Sampler()
    generate(ScriptedEngine(), [[46], [10], [20]], max_new_tokens=4, sampling=[SamplingParams(), one, one], sampler=sampler)
    assert sampler.seen[0] == [SamplingParams(), one, one] and sampler.seen[-1] == [one, one]      # the first ends early
