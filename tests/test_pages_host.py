"""The page book of a paged model (lengths, tables, reference counts, free pages) without a GPU: nothing is lost and nothing unwritten counts,
whichever way an evaluation ends."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def helper(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    so = str(tmp_path_factory.mktemp("pages") / "libpages_host.so")
    subprocess.run([nvcc, "-O1", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-o", so, os.path.join(ROOT, "tests", "pages_host.cu")], check=True,
                   capture_output=True)
    L = C.CDLL(so)
    L.book_new.restype = C.c_void_p
    return L


class Book:
    def __init__(self, lib, page, n_pages, n_seq, n_ctx):
        self.L, self.page, self.n_pages, self.n = lib, page, n_pages, n_seq
        self.h = C.c_void_p(lib.book_new(page, n_pages, n_seq, n_ctx))

    def __del__(self):
        self.L.book_delete(self.h)

    def ints(self, x):
        return (C.c_int * len(x))(*[int(v) for v in x])

    def eval(self, rows, stop=-1):
        """rows: {sequence: (first, count)}"""
        first, count = [0] * self.n, [0] * self.n
        for s, (p, c) in rows.items():
            first[s], count[s] = p, c
        return self.L.book_eval(self.h, self.n, self.ints(first), self.ints(count), stop)

    def reorder(self, parent):
        """The pages of the copies (-1: none), or None when there are too few."""
        spare = self.ints([-7] * self.n)
        return list(spare) if self.L.book_reorder(self.h, self.n, self.ints(parent), spare) else None

    @property
    def free(self):
        return self.L.book_free(self.h)

    def len(self, s):
        return self.L.book_len(self.h, s)

    def pages(self, s):
        out = (C.c_int * 1024)()
        n = self.L.book_pages(self.h, s, out)
        return list(out[:n])

    def sound(self):
        """Every page is free or in tables, and counted as often as it is in one; tables hold what the lengths say."""
        used = [p for s in range(self.n) for p in self.pages(s)]
        assert self.free == self.n_pages - len(set(used))
        for p in range(self.n_pages):
            assert self.L.book_refs(self.h, p) == used.count(p)
        for s in range(self.n):
            assert len(self.pages(s)) == -(-self.len(s) // self.page)
        return True


def test_an_evaluation_that_fails_leaves_its_sequences_where_its_rows_began(helper):
    b = Book(helper, 16, 12, 4, 200)
    assert b.eval({0: (0, 20), 1: (0, 33), 2: (0, 5)}) == 1 and b.sound()
    for stop in (0, 1, 2, 3):
        before = [b.pages(s) for s in range(3)]
        assert b.eval({0: (20, 30), 1: (33, 1), 3: (0, 17)}, stop) == -1 and b.sound()
        assert [b.len(s) for s in range(4)] == [20, 33, 5, 0] and [b.pages(s) for s in range(3)] == before
    assert b.eval({0: (7, 30), 2: (5, 5)}, 1) == -1 and b.sound()  # the cut of a sequence's positions stays
    assert [b.len(s) for s in range(4)] == [7, 33, 5, 0]
    assert b.eval({0: (7, 300)}) == 0 and b.sound() and b.len(0) == 7


def test_random_evaluations_keep_the_book_sound(helper):
    rng = np.random.default_rng(0)
    for page in (16, 32):
        b = Book(helper, page, 20, 5, 300)
        for _ in range(600):
            if rng.random() < 0.1:
                helper.book_drop(b.h, int(rng.integers(5)))
            rows = {}
            for s in rng.permutation(5)[:rng.integers(1, 5)]:
                n = b.len(int(s))
                first = n if rng.random() < 0.7 else int(rng.integers(0, n + 1))
                rows[int(s)] = (first, int(rng.integers(1, 40)))
            was = [b.len(s) for s in range(5)]
            stop = int(rng.integers(-1, 5)) if rng.random() < 0.3 else -1
            got = b.eval(rows, stop)
            assert b.sound()
            for s in range(5):
                if s not in rows or got == 0:
                    assert b.len(s) == was[s]
                else:
                    assert b.len(s) == (sum(rows[s]) if got == 1 else rows[s][0])


def test_beams_that_fill_the_pool_go_on_from_one_of_them(helper):
    """Four beams share a prompt's page and have a half-filled one each, none is free: three of the four are given up by the call itself."""
    b = Book(helper, 16, 5, 4, 64)
    assert b.eval({0: (0, 16)}) == 1 and b.reorder([0, 0, 0, 0]) == [-1] * 4
    assert b.eval({s: (16, 5) for s in range(4)}) == 1 and b.free == 0
    last = [b.pages(s)[1] for s in range(4)]
    got = b.reorder([2, 2, 2, 2])
    assert got[0] == -1 and sorted(got[1:]) == sorted(p for p in last if p != last[2])
    assert [b.pages(s)[1] for s in range(4)] == [last[2]] + got[1:] and b.free == 0 and b.sound()
    # two parents stay: what the others give up is not enough for three copies of one more
    b = Book(helper, 16, 4, 4, 64)
    assert b.eval({0: (0, 5), 1: (0, 5), 2: (0, 5), 3: (0, 5)}) == 1
    assert b.reorder([0, 0, 2, 2]) is not None and b.sound()
    b = Book(helper, 16, 3, 4, 64)
    assert b.eval({0: (0, 5), 1: (0, 5), 2: (0, 5)}) == 1
    assert b.reorder([0, 1, 1, 0]) is None and b.sound() and [b.len(s) for s in range(4)] == [5, 5, 5, 0]


@pytest.mark.parametrize("n_pages", (9, 14, 40))
def test_random_searches_keep_every_history(helper, n_pages):
    """Evaluations, reorderings and drops in a small pool, with what every position holds kept beside the book: no copy reads what another
    one writes, a refusal is right, and every sequence finds its own past."""
    rng = np.random.default_rng(n_pages)
    page, n, refused, recycled = 4, 5, 0, 0
    b = Book(helper, page, n_pages, n, 40)
    held, past, stamp = {}, [[] for _ in range(n)], 0
    for _ in range(3000):
        what = rng.random()
        old, lens = [b.pages(s) for s in range(n)], [b.len(s) for s in range(n)]
        if what < 0.05:
            s = int(rng.integers(n))
            helper.book_drop(b.h, s)
            past[s] = []
        elif what < 0.5:
            parent = rng.integers(0, n, n).tolist()
            free = b.free
            got = b.reorder(parent)
            copies = [r for r, q in enumerate(parent) if lens[q] % page and q in parent[:r]]
            kept = {p for r, q in enumerate(parent) for p in old[q][:len(old[q]) - (r in copies)]}
            assert (got is None) == (len(kept) + len(copies) > n_pages)
            if got is None:
                refused += 1
                assert [b.pages(s) for s in range(n)] == old
            else:
                assert [r for r in range(n) if got[r] >= 0] == copies
                spare = [got[r] for r in copies]
                assert len(set(spare)) == len(spare) and not set(spare) & kept
                recycled += len(spare) > free
                for r in copies:
                    held.update({(got[r], i): held[(old[parent[r]][-1], i)] for i in range(lens[parent[r]] % page)})
                past = [list(past[q]) for q in parent]
        else:
            s = int(rng.integers(n))
            first, m = (lens[s] if rng.random() < 0.8 else int(rng.integers(0, lens[s] + 1))), int(rng.integers(1, 7))
            if first + m <= 40 and b.eval({s: (first, m)}) == 1:
                now = b.pages(s)
                for i, (x, y) in enumerate(zip(old[s], now)):
                    if x != y and i == first // page:
                        held.update({(y, j): held[(x, j)] for j in range(first % page)})
                past[s] = past[s][:first]
                for i in range(first, first + m):
                    stamp += 1
                    held[(now[i // page], i % page)] = stamp
                    past[s].append(stamp)
        assert b.sound()
        for s in range(n):
            assert [held[(b.pages(s)[i // page], i % page)] for i in range(b.len(s))] == past[s]
    assert n_pages == 40 or (refused and recycled)
