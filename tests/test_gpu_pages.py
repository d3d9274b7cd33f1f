"""Attention over a cache in pages, pages copied, rows of packed tokens: against plain forms in 64 bits, at the sizes, masks and places where they can go wrong."""
import pytest
import torch

from glinthawk_amd import Shape, ops
from pages_plain import Pool, attention, hold

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


def shape_of(heads, kv_heads, size):
    return Shape(dim=heads * size, n_layers=1, n_heads=heads, n_kv_heads=kv_heads, hidden_dim=8, seq_len=8)


def queries(rows, heads, size, dtype, seed=1):
    return torch.randn((rows, heads * size), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def decode(pool, heads, lengths, q=None, max_length=None, workspace=None):
    """The kernel's rows, over a sentinel."""
    shape = shape_of(heads, pool.kv_heads, pool.size)
    q = queries(len(lengths), heads, pool.size, pool.pool.dtype) if q is None else q
    xb = torch.full_like(q, 7.0)
    p = ops.pages(pool.pool, pool.table)
    ops.attn_decode_paged(q, p, torch.tensor(lengths, dtype=torch.int32).cuda(), xb, max(lengths) if max_length is None else max_length, shape, workspace)
    return q, xb


def check_decode(pool, heads, lengths, **how):
    q, xb = decode(pool, heads, lengths, **how)
    dtype, size = pool.pool.dtype, pool.size
    for i, n in enumerate(lengths):
        if n == 0:
            assert bool((xb[i] == 7.0).all()), "the row of an empty context is left as it is"
            continue
        want, off = attention(q[i:i + 1].reshape(1, heads, size), pool.k(i)[:n], pool.v(i)[:n], n - 1, dtype, dtype != F32)
        hold(xb[i].reshape(1, heads, size), want, off, f"context {i} of {n} keys")


HEADS = [(8, 1, 128), (4, 4, 128), (6, 2, 128), (16, 1, 128), (20, 1, 128), (33, 1, 64), (12, 12, 64), (6, 6, 48), (5, 1, 64), (4, 2, 8), (4, 2, 16), (10, 5, 80), (8, 4, 36),
         (3, 1, 5), (2, 2, 160), (4, 1, 256), (2, 1, 249)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", HEADS)
def test_decode_heads(heads, kv_heads, size, dtype):
    lengths = [1, 0, 63, 64, 65, 33, 130, 2, 17]
    check_decode(Pool(lengths, kv_heads, size, dtype), heads, lengths)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 64, 128, 1024])
def test_decode_pages(page, dtype):
    lengths = [1, 15, 16, 17, 31, 47, 128, 200, 0]
    check_decode(Pool(lengths, 2, 128, dtype, page), 8, lengths)
    check_decode(Pool(lengths, 3, 64, dtype, page), 3, lengths)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", [(8, 1, 128), (2, 2, 64), (3, 1, 36), (4, 1, 200), (5, 1, 256), (4, 4, 136)])
def test_decode_of_long_contexts_in_splits(heads, kv_heads, size, dtype):
    lengths = [3001, 257, 1, 0, 1024, 2047]
    check_decode(Pool(lengths, kv_heads, size, dtype, 32), heads, lengths)
    check_decode(Pool(lengths[:1], kv_heads, size, dtype, 16, seed=3), heads, lengths[:1])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_of_many_contexts(dtype):
    lengths = [1 + 37 * i % 300 for i in range(300)]
    check_decode(Pool(lengths, 1, 64, dtype), 4, lengths)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch", [2, 63, 64, 65])
def test_decode_in_order_of_length(batch, dtype):
    """More work-groups than run at a time, lengths that are equal, zero, ascending and beyond the bound: each context once, whatever the order they are taken in."""
    lengths = [(0, 5, 5, 17 + i, 40, 0, 90 - i)[i % 7] for i in range(batch - 2)] + [1024, 1100]
    pool = Pool(lengths, 64 if batch > 2 else 1040, 8, dtype)
    q, xb = decode(pool, pool.kv_heads, lengths, max_length=1024)
    for i, n in enumerate(lengths):
        n = min(n, 1024)
        if n == 0:
            assert bool((xb[i] == 7.0).all())
            continue
        want, off = attention(q[i:i + 1].reshape(1, pool.kv_heads, 8), pool.k(i)[:n], pool.v(i)[:n], n - 1, dtype, dtype != F32)
        hold(xb[i].reshape(1, pool.kv_heads, 8), want, off, f"context {i} of {n} keys")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("spare,shift", [(1, 0), (0, 1), (8, 8), (24, 16), (3, 5)])
def test_pages_that_lie_apart_or_unaligned(spare, shift, dtype):
    lengths = [40, 100, 7]
    pool = Pool(lengths, 2, 128, dtype, spare=spare, shift=shift)
    check_decode(pool, 8, lengths)
    check_packed(pool, 8, [40, 60, 7], [0, 40, 0])


def test_keys_beyond_the_bound_are_not_attended():
    pool = Pool([200, 90], 2, 128, F16)
    q, xb = decode(pool, 8, [200, 90], max_length=100)
    for i, n in enumerate((100, 90)):
        want, off = attention(q[i:i + 1].reshape(1, 8, 128), pool.k(i)[:n], pool.v(i)[:n], n - 1, F16, True)
        hold(xb[i].reshape(1, 8, 128), want, off)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_numbers_that_name_no_page_touch_nothing_else(dtype):
    """A context whose table names no page: its own row is not specified, the others are as they were, and nothing is written but rows of xb."""
    lengths = [100, 100, 100]
    pool = Pool(lengths, 2, 128, dtype)
    q, clean = decode(pool, 8, lengths)
    pool.table[1, 2:] = torch.tensor([-1, 2 ** 31 - 1, pool.n_pages, 1, -(2 ** 31)], dtype=torch.int32).cuda()
    before = pool.memory.clone()
    _, xb = decode(pool, 8, lengths, q=q)
    assert torch.equal(xb[0], clean[0]) and torch.equal(xb[2], clean[2])
    assert torch.equal(pool.memory.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_decode_scores_of_every_size(dtype):
    """Scores far apart (one key has all the weight), all equal, all at the type's lowest value, and infinities where the formula gives NaN."""
    pool = Pool([100] * 4, 1, 128, dtype)
    q = queries(4, 8, 128, dtype) * 30
    q[1] = 0
    q[2] = -torch.finfo(dtype).max if dtype == F16 else -3.0e4
    check_decode(pool, 8, [100] * 4, q=q)
    q[3, 5] = INF
    _, xb = decode(pool, 8, [100] * 4, q=q)
    assert bool(torch.isnan(xb[3, :128]).all()) and bool(torch.isfinite(xb[3, 128:]).all())


# ---- packed prompts ------------------------------------------------------------------------------
def packed(pool, heads, tokens, start, q=None, max_keys=None, extra=2, workspace=None):
    shape = shape_of(heads, pool.kv_heads, pool.size)
    first = torch.tensor([0] + tokens).cumsum(0).int()
    q = queries(sum(tokens) + extra, heads, pool.size, pool.pool.dtype) if q is None else q
    xb = torch.full_like(q, 7.0)
    p = ops.pages(pool.pool, pool.table)
    where = None if start is None else torch.tensor(start, dtype=torch.int32).cuda()
    ops.attn_packed(q, p, first.cuda(), where, xb, max(pool.keys) if max_keys is None else max_keys, shape, workspace)
    return q, xb, first.tolist()


def check_packed(pool, heads, tokens, start, **how):
    q, xb, first = packed(pool, heads, tokens, start, **how)
    dtype, size = pool.pool.dtype, pool.size
    assert bool((xb[first[-1]:] == 7.0).all()), "rows behind the last sequence are left as they were"
    for i, n in enumerate(tokens):
        rows = slice(first[i], first[i] + n)
        want, off = attention(q[rows].reshape(n, heads, size), pool.k(i), pool.v(i), start[i] if start else 0, dtype, dtype != F32)
        hold(xb[rows].reshape(n, heads, size), want, off, f"sequence {i} of {n} tokens")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", HEADS)
def test_packed_heads(heads, kv_heads, size, dtype):
    tokens, start = [1, 0, 17, 40, 3], [0, 0, 0, 30, 64]
    check_packed(Pool([n + s for n, s in zip(tokens, start)], kv_heads, size, dtype), heads, tokens, start)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("page", [1, 8, 16, 32, 64, 512])
def test_packed_pages(page, dtype):
    tokens = [31, 65, 0, 64, 130, 1]
    check_packed(Pool(tokens, 2, 128, dtype, page), 2, tokens, None)
    start = [5, 17, 0, 1, 16, 100]
    check_packed(Pool([n + s for n, s in zip(tokens, start)], 1, 64, dtype, page), 3, tokens, start)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", [(8, 1, 128), (2, 2, 64), (3, 1, 36), (3, 1, 256), (2, 2, 136)])
def test_packed_over_many_stages_and_splits(heads, kv_heads, size, dtype):
    tokens, start = [300, 2, 129], [0, 1500, 700]
    check_packed(Pool([n + s for n, s in zip(tokens, start)], kv_heads, size, dtype, 32), heads, tokens, start)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_packed_many_sequences(dtype):
    tokens = [(7 * i) % 23 for i in range(150)]
    check_packed(Pool(tokens, 1, 64, dtype), 4, tokens, None)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", [(8, 1, 128), (2, 2, 128), (2, 1, 64), (3, 1, 36), (2, 1, 200)])
@pytest.mark.parametrize("start", [0, 900])
def test_what_stands_behind_a_token_does_not_reach_it(heads, kv_heads, size, dtype, start):
    """Infinities and NaN in a later token's row: the tokens before it are as if they were not there, those from it on are what the formula gives."""
    tokens, bad = [70], start + 37
    pool = Pool([start + 70], kv_heads, size, dtype)
    kv = kv_heads * size
    q, xb, _ = packed(pool, heads, tokens, [start])
    spoilt = pool.rows[0].clone()
    spoilt[bad, kv:] = INF
    spoilt[bad, kv + 1] = NAN
    spoilt[bad + 20, :kv] = NAN
    pool.store(pool.table[0], spoilt, 0)
    _, got, _ = packed(pool, heads, tokens, [start], q=q)
    want, off = attention(q[:37].reshape(37, heads, size), pool.k(0), pool.v(0), start, dtype, dtype != F32)
    hold(got[:37].reshape(37, heads, size), want, off)
    hold(xb[:37].reshape(37, heads, size), want, off)
    later = got[37:57].reshape(20, heads, size)
    assert bool(torch.isnan(later[:, :heads // kv_heads, 1]).all()) and bool(torch.isinf(later[:, :heads // kv_heads, 2]).all())
    assert bool(torch.isnan(got[57:70]).all())


def test_packed_equals_decode_of_its_tokens():
    """A prompt's last rows, and the same tokens decoded one by one: equal but for how the sums are cut."""
    pool = Pool([150], 2, 128, F16)
    q, xb, _ = packed(pool, 8, [150], [0], extra=0)
    for n in (1, 64, 149, 150):
        _, one = decode(pool, 8, [n], q=q[n - 1:n].contiguous())
        assert float((one[0].float() - xb[n - 1].float()).abs().max()) <= 4 * 2.0 ** -11 * 4


def test_first_that_goes_past_the_rows():
    """Tables that claim more tokens than there are rows: only rows that exist are written."""
    pool = Pool([64, 64], 1, 128, F16)
    shape = shape_of(8, 1, 128)
    q = queries(50, 8, 128, F16)
    whole = torch.full((60, 8 * 128), 7.0, dtype=F16, device="cuda")
    ops.attn_packed(q, ops.pages(pool.pool, pool.table), torch.tensor([0, 40, 1000], dtype=torch.int32).cuda(), None, whole[:50], 64, shape)
    assert bool((whole[50:] == 7.0).all())
    for i, (a, b) in enumerate(((0, 40), (40, 50))):
        want, off = attention(q[a:b].reshape(b - a, 8, 128), pool.k(i), pool.v(i), 0, F16, True)
        hold(whole[a:b].reshape(b - a, 8, 128), want, off)


# ---- rows of packed tokens, pages copied -------------------------------------------------------------
def test_page_rows():
    tokens, start = [5, 0, 33, 1], [14, 3, 0, 100]
    pool = Pool([n + s for n, s in zip(tokens, start)], 2, 8, F16, spare=16)
    pool.table[2, 1] = pool.n_pages                     # no such page
    first = torch.tensor([0, 5, 5, 38, 39], dtype=torch.int32).cuda()
    rows, pos = ops.page_rows(ops.pages(pool.pool, pool.table), first, torch.tensor(start, dtype=torch.int32).cuda(), 41)
    want_rows, want_pos = [], []
    for i, n in enumerate(tokens):
        for t in range(start[i], start[i] + n):
            page = int(pool.table[i, t // 16])
            want_rows.append(pool.pool[page, t % 16].data_ptr() if page < pool.n_pages else 0)
            want_pos.append(t if page < pool.n_pages else 0)
    assert rows.tolist() == want_rows + [0, 0] and pos.tolist() == want_pos + [0, 0]
    rows, pos = ops.page_rows(ops.pages(pool.pool, pool.table), first, torch.tensor([200, 0, 2 ** 31 - 1, 0], dtype=torch.int32).cuda(), 39)
    assert rows[:38].tolist() == [0] * 38 and rows[38] != 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("layers,pages,page,row,gap", [(1, 9, 16, 64, 0), (3, 9, 16, 64, 32), (2, 5, 2, 3, 0), (2, 5, 2, 3, 1), (4, 300, 16, 128, 0)])
def test_copy_pages(layers, pages, page, row, gap, dtype):
    memory = torch.randn(layers * pages * (page * row + gap)).to(dtype).cuda()
    pool = torch.as_strided(memory, (layers, pages, page, row), (pages * (page * row + gap), page * row + gap, row, 1))
    order = torch.randperm(pages)
    n = pages // 3
    pairs = torch.stack([order[:n], order[-n:]], 1)
    want = memory.clone()
    torch.as_strided(want, pool.shape, pool.stride())[:, pairs[:, 1].cuda()] = pool[:, pairs[:, 0].cuda()]
    once = memory.clone()
    for given in (pairs.int().cuda(), pairs.tolist()):
        memory.copy_(once)
        ops.copy_pages(pool, given)
        assert torch.equal(memory, want)
    interleaved = memory.clone()[:pages * layers * page * row].reshape(pages, layers, page, row).transpose(0, 1)      # the layers of a page side by side
    want = interleaved.clone()
    want[:, pairs[:, 1].cuda()] = want[:, pairs[:, 0].cuda()]
    ops.copy_pages(interleaved, pairs.int().cuda())
    assert torch.equal(interleaved, want)


def test_copy_leaves_out_numbers_that_name_no_page():
    pool = torch.randn(6, 4, 8).cuda()
    want = pool.clone()
    want[1] = want[0]
    ops.copy_pages(pool, torch.tensor([[0, 6], [7, 2], [0, 1], [-1, 3], [2, -1]], dtype=torch.int32).cuda())
    assert torch.equal(pool, want)


def test_copy_of_more_pairs_than_a_staging_slot_holds():
    n = 5000
    pool = torch.arange(2 * n, dtype=torch.float32).cuda()[:, None, None].expand(2 * n, 1, 4).contiguous()
    ops.copy_pages(pool, [(i, n + (i * 7919) % n) for i in range(n)])
    for i in (0, 1, 2047, 2048, 4999):
        assert float(pool[n + (i * 7919) % n, 0, 3]) == i
