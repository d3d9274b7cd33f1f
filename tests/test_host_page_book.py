"""Pages of a pool and the contexts that have them: against a plain model of lists and counts, on random runs of calls."""
import os
import random
import subprocess

import pytest

import glinthawk_amd
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


FAILING = r"""
#include "glint/pages.hh"
#include <cstdio>
#include <cstdlib>
#include <new>

static long left = -1; // allocations until one fails; -1: none does
void* operator new( std::size_t n )
{
  if ( left == 0 ) {
    throw std::bad_alloc {};
  }
  left -= left > 0;
  void* p = std::malloc( n );
  if ( p == nullptr ) {
    throw std::bad_alloc {};
  }
  return p;
}
void operator delete( void* p ) noexcept { std::free( p ); }
void operator delete( void* p, std::size_t ) noexcept { std::free( p ); }

int main()
{
  int failed = 0;
  for ( int op = 0; op < 5; op++ ) {
    for ( long n = 0; n < 12; n++ ) {
      glint::PageBook book { 40, 4 };
      book.extend( 1, 30 );
      book.extend( 2, 9 );
      book.fork( 2, 3 );
      book.release( 1 );
      const auto line2 = book.context( 2 )->pages, line3 = book.context( 3 )->pages;
      const auto free = book.free();
      left = n;
      bool threw = false;
      try {
        switch ( op ) {
          case 0: book.extend( 9, 20 ); break;
          case 1: book.extend( 3, 60 ); break;
          case 2: book.fork( 2, 9 ); break;
          case 3: book.compact(); break;
          default: book.release( 3 ); break;
        }
      } catch ( const std::bad_alloc& ) {
        threw = true;
      }
      left = -1;
      failed += threw;
      if ( threw && ( book.free() != free || book.context( 9 ) || book.context( 2 )->pages != line2 || book.context( 3 )->pages != line3 || op == 4 ) ) {
        std::printf( "op %d, allocation %ld\n", op, n );
        return 1;
      }
      book.release( 2 );
      book.release( 3 );
      book.release( 9 );
      if ( book.free() != 40 || !book.extend( 1, 160 ) || book.free() != 0 ) {
        std::printf( "op %d, allocation %ld: pages lost\n", op, n );
        return 1;
      }
    }
  }
  return failed >= 8 ? 0 : 2;
}
"""


def test_calls_that_memory_runs_out_in_change_nothing(tmp_path):
    source, exe = tmp_path / "failing.cc", tmp_path / "failing"
    source.write_text(FAILING)
    host = os.path.join(os.path.dirname(os.path.abspath(glinthawk_amd.__file__)), "host")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-I" + host, str(source), "-o", str(exe)], check=True, timeout=120)
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout
