"""The page book (tl_amd/csrc/page_book.h) through the C ABI: which pages sequences hold through
growth, forks, cuts, closes and compaction, its refusals, and random histories against a plain
model of it.  Host memory only: no GPU."""
import random

import pytest

from tl_amd import BackendError, PageBook, _lib


def test_grow_takes_the_lowest_pages_and_close_returns_them():
    b = PageBook(6, 16)
    x, y = b.open(), b.open()
    assert b.grow(x, 17) == [] and b.grow(y, 16) == [] and b.grow(x, 15) == []
    assert b.row(x, 3).tolist() == [0, 1, -1] and b.row(y, 1).tolist() == [2] and b.length(x) == 32
    b.close(x)
    assert b.free_pages == 5
    assert b.grow(y, 33) == [] and b.row(y, 4).tolist() == [2, 0, 1, 3]


def test_fork_shares_pages_and_writes_go_to_own_ones():
    b = PageBook(8, 16)
    x = b.open()
    b.grow(x, 20)
    y = b.fork(x)
    assert b.free_pages == 6 and b.row(y, 2).tolist() == [0, 1]
    assert b.grow(y, 1) == [(1, 2)]           # y writes into a shared tail page: a copy
    assert b.grow(x, 1) == []                 # x holds the old one alone now
    z = b.fork(x)
    assert b.grow(z, 0) == []
    b.cut(z, 16)
    assert b.grow(z, 1) == []                 # the shared page is full: the next one is new
    assert b.row(z, 2).tolist() == [0, 3] and b.row(x, 2).tolist() == [0, 1]
    b.close(x)
    b.close(y)
    assert b.free_pages == 6 and b.row(z, 2).tolist() == [0, 3]


def test_compact_moves_the_highest_pages_down():
    b = PageBook(10, 16)
    s = [b.open() for _ in range(4)]
    for i in s:
        b.grow(i, 32)
    t = b.fork(s[3])
    b.close(s[0])
    b.close(s[2])
    assert b.compact() == [(6, 0), (7, 1)]
    assert b.row(s[3], 2).tolist() == [0, 1] and b.row(t, 2).tolist() == [0, 1] and b.row(s[1], 2).tolist() == [2, 3]
    assert b.compact() == []
    n = b.open()
    b.grow(n, 16)
    assert b.row(n, 1).tolist() == [4]


def test_refusals():
    lib = _lib.load()
    for pages, size in ((0, 16), (1 << 31, 16), (4, 0), (4, 65536)):
        assert not lib.tl_hip_page_book_new(pages, size) and lib.tl_hip_last_status() == 8
    b = PageBook(3, 16)
    x = b.open()
    b.grow(x, 33)
    for call, variant in (((lambda: b.grow(x, 16)), "AllocationError"), ((lambda: b.grow(x, 1 << 62)), "AllocationError"),
                          ((lambda: b.grow(x, -1)), "ArgumentError"), ((lambda: b.grow(9, 1)), "IndexOutOfBounds"),
                          ((lambda: b.fork(9)), "IndexOutOfBounds"), ((lambda: b.close(9)), "IndexOutOfBounds"),
                          ((lambda: b.length(9)), "IndexOutOfBounds"), ((lambda: b.row(9, 3)), "IndexOutOfBounds"),
                          ((lambda: b.row(x, 2)), "ArgumentError"), ((lambda: b.cut(x, 34)), "ArgumentError"),
                          ((lambda: b.cut(x, -1)), "ArgumentError"), ((lambda: b.cut(9, 0)), "IndexOutOfBounds")):
        with pytest.raises(BackendError) as e:
            call()
        assert e.value.variant == variant
    assert b.length(x) == 33 and b.free_pages == 0 and b.row(x, 3).tolist() == [0, 1, 2]
    # a fork that cannot get a page of its own changes nothing
    y = b.fork(x)
    with pytest.raises(BackendError):
        b.grow(y, 1)
    assert b.row(y, 3).tolist() == [0, 1, 2]
    for f in (lib.tl_hip_page_book_open, lib.tl_hip_page_book_free_pages):
        assert f(None) == -1 and lib.tl_hip_last_status() == 4
    assert lib.tl_hip_page_book_close(None, 0) == 4 and lib.tl_hip_page_book_release(None) == 0
    # too little room for compaction's pairs: nothing moves
    import ctypes as C
    b.close(x)
    b.cut(y, 0)
    z = b.open()
    b.grow(z, 48)
    w = b.fork(z)
    b.close(z)
    assert b.row(w, 3).tolist() == [0, 1, 2]
    c = PageBook(4, 16)
    p, q = c.open(), c.open()
    c.grow(p, 32)
    c.grow(q, 32)
    c.close(p)
    n = C.c_int64()
    assert lib.tl_hip_page_book_compact(c._h, None, None, 0, C.byref(n)) == 8 and n.value == 2
    assert c.row(q, 2).tolist() == [2, 3] and c.compact() == [(2, 0), (3, 1)]


@pytest.mark.parametrize("seed", range(4))
def test_random_histories_keep_every_position_where_the_model_has_it(seed):
    """What each position of each sequence holds, through the book's pages and copies carried out
    on a list, against a plain dict of token lists."""
    r = random.Random(seed)
    size, n_pages = r.choice([1, 4, 16]), 40
    b, mem, model, token = PageBook(n_pages, size), [[None] * size for _ in range(n_pages)], {}, 0

    def carry(pairs):
        old = [list(p) for p in mem]
        assert len({d for _, d in pairs}) == len(pairs) and not {s for s, _ in pairs} & {d for _, d in pairs}
        for s, d in pairs:
            mem[d] = old[s]

    for _ in range(600):
        what = r.random()
        if not model or what < 0.15:
            model[b.open()] = []
        elif what < 0.6:
            s, n = r.choice(list(model)), r.randint(0, 3 * size)
            try:
                pairs = b.grow(s, n)
            except BackendError as e:
                assert e.variant == "AllocationError"
                continue
            carry(pairs)
            row = b.row(s, n_pages)
            for _ in range(n):
                mem[row[len(model[s]) // size]][len(model[s]) % size] = token
                model[s].append(token)
                token += 1
        elif what < 0.72:
            s = r.choice(list(model))
            model[b.fork(s)] = list(model[s])
        elif what < 0.84:
            s = r.choice(list(model))
            model[s] = model[s][: r.randint(0, len(model[s]))]
            b.cut(s, len(model[s]))
        elif what < 0.95:
            s = r.choice(list(model))
            b.close(s)
            del model[s]
        else:
            carry(b.compact())
            used = {p for s in model for p in b.row(s, n_pages).tolist() if p >= 0}
            assert used == set(range(len(used)))
        used = set()
        for s, tokens in model.items():
            row = b.row(s, n_pages).tolist()
            assert b.length(s) == len(tokens)
            assert [mem[row[j // size]][j % size] for j in range(len(tokens))] == tokens
            used |= {p for p in row if p >= 0}
        assert b.free_pages == n_pages - len(used)
