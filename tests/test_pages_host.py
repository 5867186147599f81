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
