"""Operators over a paged cache at the edges of their arguments, without a GPU."""
import subprocess
import sys

import pytest
import torch

import glinthawk_amd
from glinthawk_amd import Shape, ops

FAILING = r"""
import ctypes, resource, sys
lib = ctypes.CDLL(sys.argv[1])
lib.gh_copy_pages_host.argtypes = [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p]
lib.gh_last_error.restype = ctypes.c_char_p
pairs = (ctypes.c_uint32 * 2)(0, 1)
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (1 << 30),) * 2)      # the check of so many pairs wants 8 GiB
rc = lib.gh_copy_pages_host(1 << 20, 64, 64, 8, 1, 0, pairs, 2 ** 31 - 1, None)
print(rc, lib.gh_last_error().decode())
"""


def test_pairs_that_memory_does_not_suffice_for_are_refused():
    """An error, and no exception across the C interface, which would end the process."""
    ran = subprocess.run([sys.executable, "-c", FAILING, glinthawk_amd.lib_path()], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0, (ran.returncode, ran.stderr)
    rc, said = ran.stdout.split(" ", 1)
    assert int(rc) < 0 and "no memory" in said


@pytest.mark.parametrize("most", [2 ** 32, 2 ** 32 + 16, -1, 2 ** 40])
def test_bounds_that_32_bits_do_not_hold_are_refused(most):
    """They are not cut to a smaller bound, whose keys alone would be attended."""
    shape = Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=2, hidden_dim=8, seq_len=8)
    p = ops.pages(torch.zeros(4, 16, 512, dtype=torch.float16), torch.zeros((2, 3), dtype=torch.int32))
    q, ints, room = torch.zeros(2, 1024, dtype=torch.float16), torch.ones(3, dtype=torch.int32), torch.zeros(16, dtype=torch.uint8)
    for call in (lambda: ops.attn_decode_paged(q, p, ints[:2], q.clone(), most, shape, room), lambda: ops.attn_packed(q, p, ints, None, q.clone(), most, shape, room),
                 lambda: ops.attn_decode_paged_workspace(2, most, shape, torch.float16), lambda: ops.attn_packed_workspace(2, 9, most, shape, torch.float16),
                 lambda: ops.token_logprobs_workspace(2, 100, most)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    with pytest.raises(ValueError, match="alternatives"):
        ops.token_logprobs(torch.zeros(2, 9), ints[:2], most, room)


def test_descriptors_of_many_shapes_are_not_all_kept():
    for n in range(1, 300):
        shape = Shape(dim=8 * n, n_layers=1, n_heads=n, n_kv_heads=n, hidden_dim=8, seq_len=8)
        assert ops.attn_decode_paged_workspace(1, 128, shape, torch.float16) == 2 * n * (8 + 2) * 4
    assert ops._shape_ref.cache_info().currsize <= 64


@pytest.mark.parametrize("heads,kv_heads,size", [(8, 2, 128), (64, 8, 128), (6, 6, 48), (33, 1, 64), (2, 2, 256)])
def test_workspaces_of_larger_calls_cover_smaller_ones(heads, kv_heads, size):
    """No smaller batch, number of tokens or bound asks for more, across the 64 keys that take no splits and the bound of partial results."""
    shape = Shape(dim=heads * size, n_layers=1, n_heads=heads, n_kv_heads=kv_heads, hidden_dim=8, seq_len=8)
    rows, keys = [1, 2, 3, 15, 16, 17, 63, 64, 100, 255, 1000, 1023, 1024, 4000, 70000], [0, 1, 63, 64, 65, 128, 129, 1000, 4096, 40000, 2 ** 24, 2 ** 31 - 1]
    for size_of in (lambda n, k: ops.attn_decode_paged_workspace(n, k, shape, torch.float16), lambda n, k: ops.attn_packed_workspace(min(n, 3), n, k, shape, torch.float16)):
        table = [[size_of(n, k) for k in keys] for n in rows]
        assert all(a <= b for line in table for a, b in zip(line, line[1:])) and all(a <= b for low, high in zip(table, table[1:]) for a, b in zip(low, high))
        assert all(v == 0 for line in table for v in line[:4]) and 0 < table[0][4] and table[-1][-1] <= 65536 * (size + 2) * 4
    for vocab in (1, 100, 32768, 32769, 65537, 130001, 2 ** 21):
        tops = [n for n in (0, 1, 5, 20, 64) if n <= vocab]
        table = [[ops.token_logprobs_workspace(n, vocab, k) for k in tops] for n in (1, 2, 7, 300, 65535)]
        assert all(a <= b for line in table for a, b in zip(line, line[1:])) and all(a <= b for low, high in zip(table, table[1:]) for a, b in zip(low, high))
        assert all((v == 0) == (vocab <= 32768) for line in table for v in line)
