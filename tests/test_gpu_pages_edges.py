"""Attention over a cache in pages at the edges of what the calls take: far positions."""
import pytest
import torch

from glinthawk_amd import Shape, ops
from pages_plain import HALF_STEP, STEP32

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


def shape_of(heads, kv_heads, size):
    return Shape(dim=heads * size, n_layers=1, n_heads=heads, n_kv_heads=kv_heads, hidden_dim=8, seq_len=8)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("start", [2 ** 30 - 2, 2 ** 30 + 5])
def test_a_prompt_behind_more_than_2_30_keys(start, dtype):
    """Three tokens whose own keys have all the weight (e^40 against 2^30 equal ones), the pages of the past being one page: each sees its own key, and none behind it."""
    size, page = 8, 1 << 20
    pool = torch.zeros((2, page, 2 * size), dtype=dtype, device="cuda")
    entries = start // page + 2
    table = torch.zeros((1, entries), dtype=torch.int32, device="cuda")
    table[0, -2 if (start + 2) // page == start // page else -1] = 1
    new = pool.reshape(2 * page, 2 * size)
    at = [int(table[0, (start + t) // page]) * page + (start + t) % page for t in range(3)]
    for t, row in enumerate(at):
        new[row, t] = 16.0                     # keys at right angles: token t looks for its own, and token 2 for token 1's
        new[row, size:] = t + 1.0
    q = torch.zeros((3, size), dtype=dtype, device="cuda")
    for t, looks in enumerate((0, 1, 1)):
        q[t, looks] = 40.0 / 16.0 * size ** 0.5
    xb = torch.zeros_like(q)
    shared = sum(int(table[0, e]) == 0 and at[0] < page for e in range(entries))
    ops.attn_packed(q, ops.pages(pool, table), ints(0, 3), ints(start), xb, start + 3, shape_of(1, 1, size))
    # (the keys of a page that stands for others too are seen as often as the page stands there, all with the same value)
    assert shared or bool((pool[0] == 0).all())
    want = torch.tensor([1.0, 2.0, 2.0], device="cuda")[:, None].expand(3, size)
    assert float((xb.float() - want).abs().max()) <= 2 * (2 ** 30 * 2.718281828 ** -40 + 64 * STEP32 * 40 + 2 * HALF_STEP[dtype])
