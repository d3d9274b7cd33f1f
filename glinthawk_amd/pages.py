"""Bookkeeping of a cache in pages: which pages of a pool the contexts have (the C++ glint::PageBook).  The pages themselves are a torch tensor that
ops.pages describes; the copies a call here asks for are ops.copy_pages's to make, before the pages are written or read.

    book = PageBook(n_pages, page_tokens)
    pairs = book.extend("a", 100)                   # None: not enough pages
    book.fork("a", "b")                             # b shares a's pages
    pairs = book.extend("b", 1)                     # [(source, destination)] where a shared page is written: ops.copy_pages(pool, pairs)
    table = book.table(["a", "b"], entries)         # numpy (2, entries) int32, for the device
"""
from __future__ import annotations

import ctypes as C
import functools
import threading
from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import numpy as np

from .stage import host_lib

Pairs = List[Tuple[int, int]]


def _alone(method):
    """One call of a book at a time: a name and the number it goes by belong together."""
    @functools.wraps(method)
    def call(self, *args, **named):
        with self._lock:
            return method(self, *args, **named)
    return call


class PageBook:
    """Contexts go by any hashable name.  Threads may share a book."""

    def __init__(self, n_pages: int, page_tokens: int):
        if not 0 < n_pages < 2 ** 32 or not 0 < page_tokens < 2 ** 31 or page_tokens & (page_tokens - 1):
            raise ValueError(f"{n_pages} pages of {page_tokens} tokens: some pages, of a power of two of tokens, expected")
        self._b = host_lib().glint_pages_new(n_pages, page_tokens)
        if not self._b:
            raise MemoryError("no memory for the page book")
        self.n_pages, self.page_tokens, self._lock = n_pages, page_tokens, threading.RLock()
        self._ids: Dict[Hashable, int] = {}
        self._next = 0          # numbers are not used again

    def __del__(self):
        if getattr(self, "_b", None):
            host_lib().glint_pages_delete(self._b)
            self._b = None

    def __reduce__(self):
        raise TypeError("a page book is not copied or pickled: two would delete the same pages")

    def _known(self, name: Hashable) -> int:
        if name not in self._ids:
            raise KeyError(name)
        return self._ids[name]

    @staticmethod
    def _held(answer: int) -> int:
        if answer < 0:          # of a context that is known
            raise MemoryError("no memory for the page book's answer")
        return answer

    def _new(self) -> int:
        self._next += 1
        return self._next

    @_alone
    def extend(self, name: Hashable, tokens: int) -> Optional[Pairs]:
        """Room for `tokens` more tokens; the copies to make, or None, and nothing changed, where the pages do not suffice."""
        if tokens < 0:
            raise ValueError(f"{tokens} tokens")
        if tokens >= 2 ** 31:
            return None
        known = self._ids.get(name)
        number = self._new() if known is None else known
        pair = (C.c_uint32 * 2)()
        got = host_lib().glint_pages_extend(self._b, number, tokens, pair)
        if got < 0:
            return None
        self._ids[name] = number
        return [(pair[0], pair[1])] if got else []

    @_alone
    def fork(self, parent: Hashable, child: Hashable) -> None:
        number = self._known(parent)
        if child in self._ids:
            raise ValueError(f"context {child!r} is there already")
        new = self._new()
        if host_lib().glint_pages_fork(self._b, number, new) != 1:
            raise MemoryError("no memory for the fork")
        self._ids[child] = new

    @_alone
    def release(self, name: Hashable) -> None:
        host_lib().glint_pages_release(self._b, self._known(name))
        del self._ids[name]

    @_alone
    def compact(self) -> Pairs:
        """Pages in use move to the front of the pool; the copies to make.  Tables made before are out of date."""
        pairs = (C.c_uint32 * (2 * self.n_pages))()
        n = self._held(host_lib().glint_pages_compact(self._b, pairs, self.n_pages))
        return [(pairs[2 * i], pairs[2 * i + 1]) for i in range(n)]

    @_alone
    def length(self, name: Hashable) -> int:
        return int(self._held(host_lib().glint_pages_length(self._b, self._known(name))))

    @_alone
    def line(self, name: Hashable) -> List[int]:
        n = -(-self.length(name) // self.page_tokens)
        out = (C.c_uint32 * max(n, 1))()
        self._held(host_lib().glint_pages_line(self._b, self._known(name), out, n))
        return list(out[:n])

    @_alone
    def table(self, names: Sequence[Hashable], entries: int) -> np.ndarray:
        """(names, entries) page numbers, 0 behind a context's last."""
        out = np.zeros((len(names), entries), dtype=np.int32)
        for row, name in zip(out, names):
            n = self._held(host_lib().glint_pages_line(self._b, self._known(name), row.ctypes.data_as(C.POINTER(C.c_uint32)), entries))
            if n > entries:
                raise ValueError(f"context {name!r} has {n} pages, the table {entries} entries")
        return out

    def free(self) -> int:
        return int(host_lib().glint_pages_free(self._b))
