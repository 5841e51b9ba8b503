"""Which sequence holds which pages: the host side of the paged cache (no GPU)."""

import random

import pytest

from reskv_b200.paged import PAGE_TOKENS, PageBook


def check(book, pages):
    held = [0] * pages
    for e in book.sequences.values():
        assert len(e.pages) == -(-e.length // PAGE_TOKENS) and len(set(e.pages)) == len(e.pages)
        for p in e.pages:
            held[p] += 1
        if e.length % PAGE_TOKENS:  # a page that still takes tokens belongs to one sequence
            assert book.holders[e.pages[-1]] == 1
    assert held == book.holders
    assert sorted(book.free) == [p for p in range(pages) if not held[p]]


def test_extend_takes_the_lowest_pages_and_is_all_or_nothing():
    book = PageBook(4)
    a, b = book.add(2)
    book.extend([a, b], [64, 1])
    assert book.of(a).pages == [0] and book.of(b).pages == [1]
    book.extend([a, b], [1, 63])
    assert book.of(a).pages == [0, 2] and book.of(b).pages == [1]
    with pytest.raises(RuntimeError, match="out of pages: 2 needed, 1 free"):
        book.extend([a, b], [64, 1])
    assert book.of(a).length == 65 and book.of(b).length == 64
    check(book, 4)


def test_fork_shares_full_pages_and_copies_the_last():
    book = PageBook(8)
    (a,) = book.add(1)
    book.extend([a], [130])
    new, pairs = book.fork([a, a])
    assert pairs == [(2, 3), (2, 4)] and [book.of(s).pages for s in new] == [[0, 1, 3], [0, 1, 4]]
    assert book.holders[:5] == [3, 3, 1, 1, 1]
    book.release([a])
    check(book, 8)
    assert 2 in book.free and 0 not in book.free
    book.extend([new[0]], [62])
    assert book.fork([new[0]])[1] == []  # full: nothing to copy
    with pytest.raises(RuntimeError):
        book.fork([new[1]] * 9)
    check(book, 8)


def test_a_sequence_without_tokens_forks():
    book = PageBook(1)
    assert book.fork(book.add(1)) == ([1], [])


def test_compact_moves_pages_to_the_front_without_overlap():
    book = PageBook(10)
    a, b, c = book.add(3)
    for _ in range(3):
        book.extend([a, b, c], [64, 64, 64])
    book.release([b])
    used, pairs = book.compact()
    assert used == 6 and {s for s, _ in pairs} == {6, 8} and {d for _, d in pairs} == {1, 4}
    assert sorted(book.of(a).pages + book.of(c).pages) == list(range(6))
    check(book, 10)
    assert book.compact() == (6, [])


def test_random_traffic():
    rng, pages = random.Random(0), 40
    book = PageBook(pages)
    for _ in range(2000):
        live = list(book.sequences)
        what = rng.random()
        try:
            if what < 0.15 or not live:
                book.add(rng.randint(0, 2))
            elif what < 0.6:
                some = rng.sample(live, rng.randint(1, min(4, len(live))))
                book.extend(some, [rng.choice((0, 1, 5, 64, 100)) for _ in some])
            elif what < 0.75:
                book.fork([rng.choice(live) for _ in range(rng.randint(1, 3))])
            elif what < 0.9:
                book.release(rng.sample(live, rng.randint(1, min(3, len(live)))))
            else:
                used, pairs = book.compact()
                sources, targets = {s for s, _ in pairs}, {d for _, d in pairs}
                assert len(targets) == len(pairs) and not sources & targets and all(d < used <= s for s, d in pairs)
        except RuntimeError:
            pass
        check(book, pages)


def test_refusals():
    book = PageBook(4)
    a, b = book.add(2)
    for sequences, counts in (([7], [1]), ([a, a], [1, 1]), ([a], [1, 1]), ([a], [-1]), ([a], [1.0]), ([True], [1]), ([a], [2**31])):
        with pytest.raises(ValueError):
            book.extend(sequences, counts)
    for call in (book.fork, book.release):
        with pytest.raises(ValueError):
            call([9])
    with pytest.raises(ValueError):
        book.release([b, b])
    with pytest.raises(ValueError):
        book.add(-1)
    check(book, 4)


def test_the_library_refuses_bad_arguments_before_any_launch():
    import numpy as np

    from reskv_b200._extension import ERR_INVALID, ERR_LIMIT, ERR_WORKSPACE, library

    lib = library()
    buf = np.zeros(1 << 16, np.uint8)
    at = buf.ctypes.data + (-buf.ctypes.data) % 16
    ints = np.zeros(16, np.int32)
    i = ints.ctypes.data

    def write(k=at, step=128, sequences=1, total=1, heads=1, pages=at, width=1):
        return lib.reskv_paged_write(k, at, 0, step, 128, 128, 128, i, i, i, sequences, width, total, heads, pages, 1, i, None)

    assert write(sequences=-1) == ERR_INVALID and write(heads=0) == ERR_INVALID and write(width=-1) == ERR_INVALID
    assert write(pages=None) == ERR_INVALID and b"null" in lib.reskv_last_error()
    assert write(pages=at + 8) == ERR_INVALID
    assert write() == ERR_INVALID and b"paged_write: pages" in lib.reskv_last_error()  # host memory
    assert write(total=0) == 0 and write(sequences=0) == 0
    assert lib.reskv_paged_read(at, at, 0, i, i, i, 1, 1, 1, 1, at, 1, i, None) == ERR_INVALID

    need = lib.reskv_paged_attention_workspace_bytes(1, 1, 1)
    assert need > 0 and lib.reskv_paged_attention_workspace_bytes(-1, 1, 1) == 0

    def attend(q=at, heads=1, queries=1, scaling=0.1, ws=at, size=need, sequences=1, page_count=1, step=128):
        return lib.reskv_paged_attention(q, 0, step, 128, i, i, sequences, 1, heads, queries, at, page_count, scaling, ws, size, at,
                                         None, i, None)

    assert attend(queries=0) == ERR_INVALID and attend(heads=2, queries=3) == ERR_INVALID
    assert attend(queries=9) == ERR_LIMIT
    assert attend(scaling=0.0) == ERR_INVALID and attend(scaling=float("nan")) == ERR_INVALID
    assert attend(q=None) == ERR_INVALID and attend(step=12) == ERR_INVALID and attend(page_count=0) == ERR_INVALID
    assert attend(ws=None) == ERR_WORKSPACE and attend(size=need - 1) == ERR_WORKSPACE
    assert attend() == ERR_INVALID and b"paged_attention: q" in lib.reskv_last_error()
    assert attend(sequences=0) == 0

    def copy(src, dst, layers=1, page_bytes=16, pages=at):
        a, b = np.array(src, np.int32), np.array(dst, np.int32)
        return lib.reskv_copy_pages(pages, layers, 4, page_bytes, a.ctypes.data, b.ctypes.data, len(src), None)

    assert copy([0], [4]) == ERR_INVALID and copy([-1], [0]) == ERR_INVALID and copy([0], [1], page_bytes=8) == ERR_INVALID
    assert copy([0, 1], [2, 2]) == ERR_INVALID and b"destination twice" in lib.reskv_last_error()
    assert copy([0, 1], [1, 2]) == ERR_INVALID and b"source and a destination" in lib.reskv_last_error()
    assert copy([1], [1]) == ERR_INVALID
    assert copy([0], [1]) == ERR_INVALID and b"copy_pages: pages" in lib.reskv_last_error()
    assert copy([0], [1], layers=65536) == ERR_LIMIT
    assert copy([], []) == 0 and copy([0], [1], layers=0) == 0


def state(book):
    return (list(book.free), list(book.holders), {s: (list(e.pages), e.length, e.step) for s, e in book.sequences.items()}, book.epoch, book._next)


def test_a_copy_that_fails_changes_nothing():
    book, seen = PageBook(12), []
    a, b, c = book.add(3)
    book.extend([a, b, c], [130, 64, 70])
    book.release([b])

    def fails(pairs):
        seen.append(pairs)
        raise MemoryError

    before = state(book)
    for call in (lambda: book.fork([a, c, a], fails), lambda: book.compact(fails)):
        with pytest.raises(MemoryError):
            call()
        assert state(book) == before
    # the pages that a copy was offered are those that it gets
    assert book.fork([a, c, a])[1] == seen[0]
    check(book, 12)
    book.release([a])
    assert book.compact(lambda pairs: seen.append(pairs))[1] == seen[-1]
    check(book, 12)


def test_an_extension_is_taken_back():
    rng, book = random.Random(1), PageBook(40)
    sequences = book.add(5)
    for _ in range(200):
        counts = [rng.choice((0, 1, 63, 64, 65, 200)) for _ in sequences]
        before = state(book)
        try:
            entries = book.extend(sequences, counts)
        except RuntimeError:
            book.release(sequences)
            sequences = book.add(5)
            continue
        if rng.random() < 0.5:
            book.retract(entries, counts)
            assert state(book) == before
        check(book, 40)


def test_sequences_that_end_leave_their_pages_to_the_forked_ones():
    book = PageBook(5)
    a, b = book.add(2)
    book.extend([a, b], [130, 65])  # pages 0 1 2, 3 4: none free
    before = state(book)
    with pytest.raises(RuntimeError, match="out of pages: 1 needed, 0 free"):
        book.fork([a])
    with pytest.raises(RuntimeError, match="out of pages: 3 needed, 2 free"):
        book.fork([a, a, a], ending=[b])
    for sequences, ending in (([a], [a]), ([a], [b, b]), ([b], [a, b])):
        with pytest.raises(ValueError):
            book.fork(sequences, ending=ending)
    assert state(book) == before
    new, pairs = book.fork([a, a], ending=[b])
    assert [s for s, _ in pairs] == [2, 2] and {d for _, d in pairs} == {3, 4} and set(book.sequences) == {a, *new}
    check(book, 5)
    new, pairs = book.fork([new[0]], ending=[new[1], a])  # shared pages stay with the one that is left
    assert len(book.free) == 1 and book.of(new[0]).pages[:2] == [0, 1]
    check(book, 5)


def test_random_traffic_with_endings():
    rng, pages = random.Random(2), 30
    book = PageBook(pages)
    for _ in range(2000):
        live, before = list(book.sequences), None
        if not live or rng.random() < 0.3:
            book.add(rng.randint(1, 2))
        try:
            if live and rng.random() < 0.5:
                book.extend([rng.choice(live)], [rng.choice((1, 5, 64, 100))])
            elif live:
                ending = rng.sample(live, rng.randint(0, len(live) - 1))
                kept = [s for s in book.sequences if s not in ending]
                before, seen = state(book), []
                new, pairs = book.fork([rng.choice(kept) for _ in range(rng.randint(0, 3))], seen.extend, ending)
                before = None
                assert seen == pairs and not {s for s, _ in pairs} & {d for _, d in pairs} and len({d for _, d in pairs}) == len(pairs)
                assert set(book.sequences) == {*kept, *new}
        except RuntimeError:
            if before is not None:
                assert state(book) == before
        check(book, pages)
