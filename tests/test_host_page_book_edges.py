"""Pages of a pool and the contexts that have them: several threads at once, copies."""
import copy
import pickle
import sys
import threading

import pytest

from glinthawk_amd.pages import PageBook


@pytest.fixture
def fast_switches():
    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    yield
    sys.setswitchinterval(before)


def together(work, n=8):
    failed, gate = [], threading.Barrier(n)

    def run(i):
        try:
            gate.wait()
            work(i)
        except Exception as e:      # for the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


def test_contexts_that_threads_begin_have_pages_of_their_own(fast_switches):
    book = PageBook(8 * 2000, 4)

    def work(i):
        for k in range(1000):
            assert book.extend((i, k), 5) == []

    together(work)
    seen = [p for i in range(8) for k in range(1000) for p in book.line((i, k))]
    assert len(seen) == len(set(seen)) == 8 * 2000 and book.free() == 0


def test_threads_that_fork_extend_and_release(fast_switches):
    book = PageBook(4000, 4)
    book.extend("parent", 6)

    def work(i):
        for k in range(300):
            book.fork("parent", (i, k))
            assert book.line((i, k)) == book.line("parent")
            pairs = book.extend((i, k), 1)
            assert len(pairs) == 1 and pairs[0][0] == book.line("parent")[-1]
            assert book.length((i, k)) == 7 and book.table([(i, k), "parent"], 3).shape == (2, 3)
            if k % 2:
                book.release((i, k))

    together(work)
    assert book.free() == 4000 - 2 - 8 * 150
    lasts = [book.line((i, k))[-1] for i in range(8) for k in range(0, 300, 2)]
    assert len(set(lasts)) == len(lasts)


def test_arguments_by_name():
    book = PageBook(n_pages=9, page_tokens=4)
    assert book.extend(name="a", tokens=5) == [] and book.fork(parent="a", child="b") is None
    assert book.line(name="b") == [0, 1] and book.length(name="b") == 5 and book.table(names=["a"], entries=2).tolist() == [[0, 1]]
    book.release(name="a")
    assert book.free() == 7


def test_one_name_that_threads_begin_at_once_is_one_context(fast_switches):
    for turn in range(200):
        book = PageBook(64, 4)
        together(lambda i: book.extend("a", 4), 4)
        assert book.length("a") == 16 and book.free() == 60, turn


def test_copies_are_refused():
    book = PageBook(9, 4)
    book.extend("a", 5)
    for make in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="not copied"):
            make(book)
    assert book.line("a") == [0, 1] and book.free() == 7
