"""Attention over a cache in pages at the edges of what the calls take: far positions, weights far below the largest, values that are no numbers, many sequences."""
import pytest
import torch

from glinthawk_amd import Shape, ops
from pages_plain import HALF_STEP, STEP32, Pool, attention, hold

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


def shape_of(heads, kv_heads, size):
    return Shape(dim=heads * size, n_layers=1, n_heads=heads, n_kv_heads=kv_heads, hidden_dim=8, seq_len=8)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def fastest(call, runs=5):
    call()
    times = []
    for _ in range(runs):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        call()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times)


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


def sink(dtype, keys, size=128, kv_heads=1):
    """A pool of one context whose key 0 lies 25.4 powers of two above all others, with values 0 there and 1 elsewhere; the queries' element, the exact result for n keys."""
    pool = torch.zeros((-(-keys // 16), 16, 2 * kv_heads * size), dtype=dtype, device="cuda")
    pool[:, :, kv_heads * size:] = 1.0
    pool[0, 0, kv_heads * size:] = 0.0
    pool[0, 0, 0:kv_heads * size:size] = 14.125          # the same in all types
    x = 14.125
    low = 2.718281828459045 ** (-x * x * size ** -0.5)
    return pool, x, lambda n: (n - 1) * low / (1 + (n - 1) * low)


def room_for(dtype, n, exact):
    # weights: relative, or where they are small for the type half its least difference, 2^-25 of 2^7; sums of n terms; the result
    return exact * (3 * HALF_STEP[dtype] + 2 * n * STEP32 + 64 * STEP32 * 26) + (n * 2.0 ** -32 + 2.0 ** -25 if dtype == F16 else 0)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_one_key_far_above_a_long_context_decode(dtype):
    keys, batch, heads = 40000, 1024, 64
    pool, x, exact = sink(dtype, keys)
    table = torch.arange(pool.shape[0], dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()      # contexts that share all pages
    q = torch.zeros((batch, heads, 128), dtype=dtype, device="cuda")
    q[:, :, 0] = x
    lengths = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    lengths[0], lengths[1] = 30001, 100
    xb = torch.zeros((batch, heads * 128), dtype=dtype, device="cuda")
    ops.attn_decode_paged(q.reshape(batch, -1), ops.pages(pool, table), lengths, xb, keys, shape_of(heads, 1, 128))
    for row, n in ((0, 30001), (1, 100), (2, keys), (batch - 1, keys)):
        assert float((xb[row].double() - exact(n)).abs().max()) <= room_for(dtype, n, exact(n)), n


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens", [3, 1024])
def test_one_key_far_above_a_long_context_packed(tokens, dtype):
    keys, heads, kv_heads = 40000, 16, 2
    pool, x, exact = sink(dtype, keys, kv_heads=kv_heads)
    table = torch.arange(pool.shape[0], dtype=torch.int32, device="cuda")[None].contiguous()
    q = torch.zeros((tokens, heads, 128), dtype=dtype, device="cuda")
    q[:, :, 0] = x
    xb = torch.zeros((tokens, heads * 128), dtype=dtype, device="cuda")
    start = keys - tokens
    ops.attn_packed(q.reshape(tokens, -1), ops.pages(pool, table), ints(0, tokens), ints(start), xb, keys, shape_of(heads, kv_heads, 128))
    for t in sorted({0, 1, tokens // 2, tokens - 1}):
        n = start + t + 1
        assert float((xb[t].double() - exact(n)).abs().max()) <= room_for(dtype, n, exact(n)), t


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", [(8, 1, 128), (4, 4, 64), (3, 1, 36), (2, 1, 200)])
def test_packed_scores_of_every_size(heads, kv_heads, size, dtype):
    """Scores far apart (one key has all the weight, others next to none), all equal, all at the type's lowest value, and an infinity where the formula gives NaN."""
    tokens, start = 70, 600
    pool = Pool([start + tokens], kv_heads, size, dtype)
    q = torch.randn((tokens, heads * size), generator=torch.Generator().manual_seed(1)).to(dtype).cuda() * 30
    q[20:30] = 0
    q[30:40] = -torch.finfo(dtype).max if dtype == F16 else -3.0e4
    q[40:50] = q[40:50] / 10

    def run():
        xb = torch.full_like(q, 7.0)
        ops.attn_packed(q, ops.pages(pool.pool, pool.table), ints(0, tokens), ints(start), xb, start + tokens, shape_of(heads, kv_heads, size))
        return xb.reshape(tokens, heads, size)

    want, off = attention(q.reshape(tokens, heads, size), pool.k(0), pool.v(0), start, dtype, dtype != F32)
    hold(run(), want, off)
    q[60, 5] = INF
    got = run()
    assert bool(torch.isnan(got[60, 0]).all()) and bool(torch.isfinite(got[60, 1:]).all())
    rest = [t for t in range(tokens) if t != 60]
    hold(got[rest], want[rest], off[rest])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,size", [(8, 1, 128), (4, 4, 64), (3, 1, 256), (5, 1, 24), (4, 2, 36)])
def test_decode_of_infinite_values(heads, kv_heads, size, dtype):
    """An infinite value that a token attends is infinite in its result, with its sign, also in splits and beside others; two of both signs are NaN."""
    lengths = [40, 3000, 700]
    pool, kv = Pool(lengths, kv_heads, size, dtype), kv_heads * size
    for i, n in enumerate(lengths):
        rows = pool.rows[i].clone()
        rows[n // 3, kv + 1], rows[n // 2, kv + 1], rows[n - 1, kv + 2] = INF, INF, -INF
        rows[5, kv + 3], rows[6, kv + 3] = INF, -INF
        pool.store(pool.table[i], rows, 0)
    q = torch.randn((len(lengths), heads * size), generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    xb = torch.zeros_like(q)
    ops.attn_decode_paged(q, ops.pages(pool.pool, pool.table), ints(*lengths), xb, max(lengths), shape_of(heads, kv_heads, size))
    got = xb.reshape(len(lengths), heads, size)
    group = got[:, :heads // kv_heads]
    assert bool((group[:, :, 1] == INF).all()) and bool((group[:, :, 2] == -INF).all()) and bool(torch.isnan(group[:, :, 3]).all())
    assert bool(torch.isfinite(group[:, :, 4:]).all()) and bool(torch.isfinite(got[:, heads // kv_heads:]).all())


@pytest.mark.parametrize("dtype,heads,kv_heads,size,tokens", [(F16, 8, 1, 128, 2048), (BF16, 8, 8, 64, 2048), (F16, 4, 1, 256, 1024), (F32, 8, 8, 64, 1024), (F32, 4, 2, 128, 1024),
                                                              (F16, 8, 4, 36, 1024)])
@pytest.mark.parametrize("what", ["row", "values", "every value", "one dim"])
def test_a_poisoned_prompt_is_no_long_call(what, dtype, heads, kv_heads, size, tokens):
    """NaN near a prompt's beginning reaches every token from there on and none before, in a call about as long as another, and the next sequence is as it was."""
    kv, other, bad = kv_heads * size, 50, 37
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = -(-tokens // 16)
    pool = torch.randn((pages + 4, 16, 2 * kv), generator=g, device="cuda").to(dtype)
    table = torch.zeros((2, pages), dtype=torch.int32, device="cuda")
    table[0] = torch.arange(pages)
    table[1, :4] = torch.arange(pages, pages + 4)
    q = torch.randn((tokens + other, heads * size), generator=g, device="cuda").to(dtype)
    first, shape = ints(0, tokens, tokens + other), shape_of(heads, kv_heads, size)
    room = torch.empty(max(16, ops.attn_packed_workspace(2, tokens + other, tokens, shape, dtype)), dtype=torch.uint8, device="cuda")

    def run(xb):
        ops.attn_packed(q, ops.pages(pool, table), first, None, xb, tokens, shape, room)
        return xb

    clean = run(torch.full_like(q, 7.0))
    usual = fastest(lambda: run(torch.empty_like(q)))
    rows = pool[:pages].reshape(-1, 2 * kv)
    if what == "row":
        rows[bad] = NAN
    elif what == "values":
        rows[bad, kv:] = NAN
    elif what == "every value":
        rows[bad:, kv:] = INF
    else:
        rows[bad, kv + 1] = NAN
    got = run(torch.full_like(q, 7.0))
    poisoned = fastest(lambda: run(torch.empty_like(q)))
    a, b = got.reshape(-1, heads, size), clean.reshape(-1, heads, size)
    assert torch.equal(a[tokens:], b[tokens:]), "the other sequence"
    # rows of the same keys in another way of summing: both within what rounding allows of the exact result
    want, off = attention(q[:bad].reshape(bad, heads, size), rows[:bad, :kv].double().reshape(bad, kv_heads, size), rows[:bad, kv:].double().reshape(bad, kv_heads, size), 0, dtype, dtype != F32)
    hold(a[:bad], want, off, "before the bad token")
    later, group = a[bad:tokens], heads // kv_heads
    if what in ("row", "values"):
        assert bool(torch.isnan(later).all())
    elif what == "every value":
        assert bool(torch.isinf(later).all())
    else:
        assert bool(torch.isnan(later[:, :group, 1]).all())
        keep = torch.ones((heads, size), dtype=torch.bool, device="cuda")
        keep[:group, 1] = False
        assert float((later[:, keep].double() - b[bad:tokens][:, keep].double()).abs().max()) <= 8 * HALF_STEP[dtype] * 4 + 4000 * STEP32
    assert poisoned < 25 * usual, f"{poisoned * 1e3:.0f} us, without NaN {usual * 1e3:.0f}"


@pytest.mark.parametrize("dtype,heads,kv_heads,size", [(F16, 8, 1, 128), (BF16, 4, 4, 64), (F32, 4, 2, 64), (F16, 4, 2, 36)])
@pytest.mark.parametrize("batch", [64, 65, 256, 257, 3000])
@pytest.mark.parametrize("tokens", [(0, 1, 1, 5, 0, 33, 1), (1, 0, 1, 1), (0,) * 10 + (2,)])
def test_many_sequences(tokens, batch, dtype, heads, kv_heads, size):
    """Single tokens, prompts and sequences without tokens in one call, contexts that share pages; and nothing of the rows behind."""
    new = [tokens[i % len(tokens)] for i in range(batch)]
    past = [(i * 37) % 90 for i in range(batch)]
    pool = Pool([130], kv_heads, size, dtype)
    table = pool.table.expand(batch, -1).contiguous()
    first = torch.tensor([0] + new).cumsum(0).int().cuda()
    q = torch.randn((sum(new) + 3, heads * size), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    xb = torch.full_like(q, 7.0)
    ops.attn_packed(q, ops.pages(pool.pool, table), first, ints(*past), xb, 130, shape_of(heads, kv_heads, size))
    assert bool((xb[sum(new):] == 7.0).all()) and bool((xb[:sum(new)] != 7.0).any(1).all())
    group = heads // kv_heads
    k, v = pool.k(0).repeat_interleave(group, 1), pool.v(0).repeat_interleave(group, 1)
    where = torch.tensor([past[i] + t for i in range(batch) for t in range(new[i])], device="cuda")
    x = q[:sum(new)].double().reshape(-1, heads, size)
    scores = (x.transpose(0, 1).float().double() @ k.permute(1, 2, 0).contiguous()) * size ** -0.5                     # (heads, tokens, keys)
    w = torch.softmax(scores.masked_fill(torch.arange(130, device="cuda") > where[:, None], -INF), -1)
    v = v.transpose(0, 1).contiguous()
    want, mean = (w @ v).transpose(0, 1), (w @ v.abs()).transpose(0, 1)
    off = mean * (3 * HALF_STEP[dtype] + 2 * (size + 16 + 130) * STEP32 * (1 + float(scores.abs().max()))) + HALF_STEP[dtype] * want.abs() + (200 * 2.0 ** -25 * 4 if dtype == F16 else 0)
    hold(xb[:sum(new)].reshape(-1, heads, size), want, off)


def test_the_time_of_many_sequences_grows_with_their_number():
    times = {}
    for batch in (512, 4096):
        pool = torch.randn((64, 16, 2048), device="cuda").half()
        table = torch.randint(64, (batch, 4), dtype=torch.int32, device="cuda")
        q, first, start = torch.randn((batch, 8192), device="cuda").half(), torch.arange(batch + 1, dtype=torch.int32, device="cuda"), torch.full((batch,), 40, dtype=torch.int32, device="cuda")
        xb, p, shape = torch.empty_like(q), ops.pages(pool, table), shape_of(64, 8, 128)
        times[batch] = fastest(lambda: ops.attn_packed(q, p, first, start, xb, 64, shape))
    assert times[4096] < 2 * 8 * times[512], times
