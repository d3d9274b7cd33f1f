"""Pages of a pool and the contexts that have them: against a plain model of lists and counts, on random runs of calls."""
import random

import pytest

from glinthawk_amd.pages import PageBook


class Plain:
    """Every page's contents as a list of (context, token) it was written with; contexts as lists of what they should read."""

    def __init__(self, n_pages, tokens):
        self.pages = [[None] * tokens for _ in range(n_pages)]
        self.tokens, self.want = tokens, {}

    def copy(self, pairs):
        sources, destinations = [a for a, _ in pairs], [b for _, b in pairs]
        assert len(set(destinations)) == len(destinations) and not set(sources) & set(destinations)
        for a, b in pairs:
            self.pages[b] = list(self.pages[a])

    def append(self, book, name, n, mark):
        line, old = book.line(name), self.want.setdefault(name, [])
        for t in range(len(old), len(old) + n):
            self.pages[line[t // self.tokens]][t % self.tokens] = (mark, t)
            old.append((mark, t))

    def check(self, book):
        seen = set()
        for name, want in self.want.items():
            line = book.line(name)
            seen.update(line)
            assert len(line) == -(-len(want) // self.tokens) and book.length(name) == len(want)
            assert [self.pages[line[t // self.tokens]][t % self.tokens] for t in range(len(want))] == want
        assert book.free() == len(self.pages) - len(seen)


@pytest.mark.parametrize("n_pages,tokens", [(1, 1), (7, 1), (12, 4), (40, 16), (9, 64)])
def test_random_runs(n_pages, tokens):
    for seed in range(30):
        rng = random.Random(1000 * n_pages + seed)
        book, plain, mark = PageBook(n_pages, tokens), Plain(n_pages, tokens), 0
        for _ in range(150):
            op, names = rng.random(), list(plain.want)
            mark += 1
            if op < 0.55:
                name, n = rng.choice(names + [f"c{mark}"]), rng.choice([0, 1, 1, 2, tokens - 1, tokens, 3 * tokens + 1])
                before, free = book.line(name) if name in plain.want else None, book.free()
                pairs = book.extend(name, n)
                if pairs is None:
                    assert book.free() == free and (book.line(name) if name in plain.want else None) == before
                    # it needs more than there are: new pages, and one for a shared last page that is written
                    have = len(plain.want.get(name, []))
                    new = -(-(have + n) // tokens) - -(-have // tokens)
                    shared = have % tokens and sum(before[-1] in book.line(other) for other in names) > 1
                    assert new + (1 if shared and n else 0) > free
                    continue
                plain.copy(pairs)
                plain.append(book, name, n, mark)
            elif op < 0.75 and names:
                parent = rng.choice(names)
                book.fork(parent, f"f{mark}")
                plain.want[f"f{mark}"] = list(plain.want[parent])
            elif op < 0.93 and names:
                name = rng.choice(names)
                book.release(name)
                del plain.want[name]
            else:
                pairs = book.compact()
                plain.copy(pairs)
                used = n_pages - book.free()
                assert all(p < used for name in plain.want for p in book.line(name))
            plain.check(book)


def test_what_is_refused():
    for n, tokens in ((0, 16), (4, 0), (4, 12), (-1, 16)):
        with pytest.raises(ValueError):
            PageBook(n, tokens)
    book = PageBook(4, 16)
    for call in (lambda: book.fork("a", "b"), lambda: book.release("a"), lambda: book.line("a"), lambda: book.length("a"), lambda: book.table(["a"], 4)):
        with pytest.raises(KeyError):
            call()
    with pytest.raises(ValueError):
        book.extend("a", -1)
    assert book.extend("a", 65) is None and book.extend("a", 2 ** 62) is None and book.extend("a", 2 ** 64 - 1) is None and book.free() == 4
    assert book.extend("a", 64) == [] and book.extend("a", 0) == [] and book.extend("a", 1) is None
    book.fork("a", "b")
    with pytest.raises(ValueError):
        book.fork("a", "b")
    with pytest.raises(ValueError):
        book.table(["a"], 3)
    assert book.table(["a", "b"], 5).tolist() == [[0, 1, 2, 3, 0]] * 2


def test_the_first_to_write_a_shared_page_gets_the_copy():
    book = PageBook(6, 16)
    assert book.extend("a", 20) == []
    book.fork("a", "b")
    assert book.line("a") == book.line("b") == [0, 1] and book.free() == 4
    assert book.extend("b", 0) == [] and book.extend("b", 1) == [(1, 2)] and book.extend("a", 1) == []
    assert book.line("a") == [0, 1] and book.line("b") == [0, 2]
    book.release("a")
    assert book.free() == 4 and book.compact() == [(2, 1)] and book.line("b") == [0, 1]
    book.fork("b", "c")
    assert book.extend("c", 12) == [(1, 2)]          # 21 tokens and 12: to the 33rd
    assert book.line("c") == [0, 2, 3] and book.length("c") == 33
