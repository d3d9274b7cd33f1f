"""Operators over a paged cache at the edges of their arguments, without a GPU."""
import subprocess
import sys

import glinthawk_amd

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
