"""The operators over a paged cache as a server uses them: prompts of different lengths in one call, contexts forked and decoded with copies of shared pages,
a pool compacted under them, log probabilities of what comes out; in graphs, on streams of their own, two at a time."""
import numpy as np
import pytest
import torch

from glinthawk_amd import Shape, ops
from glinthawk_amd.pages import PageBook
from pages_plain import HALF_STEP, Pool, attention, hold, logprobs

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


class Server:
    """A few layers of attention over pages, with every context's tokens kept beside them."""

    def __init__(self, dtype, heads, kv_heads, size, n_pages, page, layers=2, most=256):
        self.shape = Shape(dim=heads * size, n_layers=layers, n_heads=heads, n_kv_heads=kv_heads, hidden_dim=8, seq_len=most)
        self.dtype, self.page, self.most, self.size = dtype, page, most, size
        self.pool = torch.full((layers, n_pages, page, 2 * self.shape.kv_dim), float("nan"), dtype=dtype, device="cuda")
        self.book, self.entries = PageBook(n_pages, page), -(-most // page)
        angle = torch.arange(most)[:, None].double() * 10000.0 ** (-torch.arange(size // 2).double() / (size // 2))[None]
        self.real, self.imag = angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()
        self.g = torch.Generator().manual_seed(3)
        self.kept = {}          # name -> per layer: list of (unrotated K, V) of every token

    def copy(self, pairs):
        if pairs:
            ops.copy_pages(self.pool, pairs)

    def step(self, new, packed):
        """new: {name: tokens}; all of them appended and attended to, layer by layer, and checked."""
        names = list(new)
        start = {n: self.book.length(n) if n in self.kept else 0 for n in names}
        for n in names:
            pairs = self.book.extend(n, new[n])
            assert pairs is not None
            self.copy(pairs)
            self.kept.setdefault(n, [[] for _ in range(len(self.pool))])
        table = torch.from_numpy(self.book.table(names, self.entries)).cuda()
        first = torch.tensor([0] + [new[n] for n in names]).cumsum(0).int().cuda()
        begin = torch.tensor([start[n] for n in names], dtype=torch.int32).cuda()
        total, shape, size = sum(new.values()), self.shape, self.size
        outputs = []
        for layer, pool in enumerate(self.pool):
            p = ops.pages(pool, table)
            q, kv = (torch.randn((total, w), generator=self.g).to(self.dtype).cuda() for w in (shape.dim, 2 * shape.kv_dim))
            plain_q = q.clone()
            rows, pos = ops.page_rows(p, first, begin, total)
            ops.kv_append(rows, kv, shape.kv_dim)
            ops.rope(pos, self.real, self.imag, q, rows, shape)
            xb = torch.full_like(q, float("nan"))
            if packed:
                ops.attn_packed(q, p, first, begin, xb, max(self.book.length(n) for n in names), shape)
            else:
                ops.attn_decode_paged(q, p, begin + 1, xb, max(self.book.length(n) for n in names), shape)
            outputs.append(xb)
            at = 0
            for i, n in enumerate(names):
                self.kept[n][layer] += [row for row in kv[at:at + new[n]]]
                k, v = self.read(pool, self.book.line(n), self.kept[n][layer])
                got = slice(at, at + new[n])
                turned = self.turned(plain_q[got].reshape(new[n], -1, size), range(start[n], start[n] + new[n]))
                self.near(q[got].reshape(new[n], -1, size), turned)
                want, off = attention(q[got].reshape(new[n], -1, size), k, v, start[n], self.dtype, self.dtype != F32)
                hold(xb[got].reshape(new[n], -1, size), want, off, f"{n}, layer {layer}")
                at += new[n]
        return outputs[-1]

    def turned(self, x, positions):
        re, im = self.real[list(positions)].double()[:, None], self.imag[list(positions)].double()[:, None]
        a, b = x.double()[..., 0::2], x.double()[..., 1::2]
        return torch.stack([a * re - b * im, a * im + b * re], -1).flatten(-2)

    def near(self, got, want):      # two products and a sum in fp32, one rounding
        assert bool(((got.double() - want).abs() <= HALF_STEP[self.dtype] * want.abs() + 4 * 2.0 ** -24 * 12).all())

    def read(self, pool, line, kept):
        """A context's K and V as its pages hold them, which are its tokens' own: V bit for bit, K turned by its position."""
        n, kv = len(kept), self.shape.kv_dim
        rows = pool[line].reshape(-1, 2 * kv)[:n]
        want = torch.stack(kept)
        assert torch.equal(rows[:, kv:], want[:, kv:])
        self.near(rows[:, :kv].reshape(n, -1, self.size), self.turned(want[:, :kv].reshape(n, -1, self.size), range(n)))
        return rows[:, :kv].double().reshape(n, -1, self.size), rows[:, kv:].double().reshape(n, -1, self.size)

    def fork(self, parent, child):
        self.book.fork(parent, child)
        self.kept[child] = [list(rows) for rows in self.kept[parent]]


@pytest.mark.parametrize("dtype,heads,kv_heads,size,page", [(F16, 8, 2, 128, 16), (BF16, 8, 4, 64, 32), (F32, 6, 6, 48, 16), (F16, 6, 2, 24, 8)])
def test_a_server(dtype, heads, kv_heads, size, page):
    s = Server(dtype, heads, kv_heads, size, n_pages=640 // page, page=page)
    s.step({"a": 70, "b": 33, "c": 1}, packed=True)
    s.fork("a", "d")
    s.fork("a", "e")
    assert s.book.line("d") == s.book.line("a")
    for _ in range(3):
        s.step({n: 1 for n in "abcde"}, packed=False)       # the forks part where they write on
    s.step({"b": 1, "d": 19, "c": 40}, packed=True)         # decoding and prompts in one call
    s.book.release("a")
    s.kept.pop("a")
    moved = s.book.compact()
    s.copy(moved)
    assert moved and all(p < s.book.n_pages - s.book.free() for n in s.kept for p in s.book.line(n))
    xb = s.step({n: 1 for n in "bcde"}, packed=False)

    w = torch.randn((777, heads * size), generator=s.g).to(dtype).cuda()
    logits = ops.matmul(xb, w)
    tokens = torch.tensor([0, 5, 776, 100], dtype=torch.int32).cuda()
    given, entropy, ids, values = ops.token_logprobs(logits, tokens, 7)
    want = logprobs(logits, tokens, 7)
    assert torch.equal(ids.long(), want[2]) and ops.argmax(logits) == ids[:, 0].tolist() if dtype != BF16 else True
    for got, exact in zip((given, entropy, values), (want[0], want[1], want[3])):
        assert float((got.double() - exact).abs().max()) <= 1e-6 * (10 + float(logits.float().abs().max()))


def parts(seed, dtype=F16, lengths=(900, 40, 1, 300)):
    pool = Pool(lengths, 2, 128, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed + 50)
    shape = Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=2, hidden_dim=8, seq_len=8)
    q = torch.randn((len(lengths), 1024), generator=g).to(dtype).cuda()
    logits = torch.randn((3, 70000), generator=g).cuda()
    return pool, shape, ops.pages(pool.pool, pool.table), q, torch.tensor(lengths, dtype=torch.int32).cuda(), logits, torch.tensor([1, 2, 3], dtype=torch.int32).cuda()


def calls(made, workspaces, xb, packed_xb):
    pool, shape, p, q, lengths, logits, tokens = made
    ops.attn_decode_paged(q, p, lengths, xb, 900, shape, workspaces[0])
    first = torch.arange(q.shape[0] + 1, dtype=torch.int32, device="cuda")
    ops.attn_packed(q, p, first, (lengths - 1).clamp(min=0), packed_xb, 900, shape, workspaces[1])
    return ops.token_logprobs(logits, tokens, 5, workspaces[2])


def rooms(made):
    pool, shape, p, q, lengths, logits, _ = made
    n = q.shape[0]
    return [torch.empty(max(16, v), dtype=torch.uint8, device="cuda") for v in (ops.attn_decode_paged_workspace(n, 900, shape, q.dtype), ops.attn_packed_workspace(n, n, 900, shape, q.dtype),
                                                                               ops.token_logprobs_workspace(3, 70000, 5))]


@pytest.mark.parametrize("dtype", [F16, F32])
def test_graphs_that_are_replayed(dtype):
    """Captured calls, replayed with other lengths and queries, eager work and waits between; every replay as the eager calls."""
    made = parts(1, dtype)
    pool, shape, p, q, lengths, logits, tokens = made
    room, xb, px = rooms(made), torch.zeros_like(q), torch.zeros_like(q)
    calls(made, room, xb, px)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(made, room, xb, px)
    for i, now in enumerate([(900, 40, 1, 300), (1, 1, 1, 1), (899, 0, 1, 17), (64, 33, 1, 128), (900, 40, 1, 300)]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        logits.copy_(torch.randn(logits.shape, generator=torch.Generator().manual_seed(i)))
        xb.fill_(3.0)
        px.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (xb, px, *got)]
        eager, packed_eager = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
        others = calls(made, rooms(made), eager, packed_eager)
        torch.cuda.synchronize()
        for a, b in zip(kept, (eager, packed_eager, *others)):
            assert torch.equal(a, b)
        for c, n in enumerate(now):
            if n:
                want, off = attention(q[c:c + 1].reshape(1, 8, 128), pool.k(c)[:n], pool.v(c)[:n], n - 1, dtype, dtype != F32)
                hold(kept[0][c].reshape(1, 8, 128), want, off)
                hold(kept[1][c].reshape(1, 8, 128), want, off)
            else:
                assert bool((kept[0][c] == 3.0).all())


def test_pairs_in_host_memory_are_not_captured():
    from glinthawk_amd._lib import GlintError

    pool = torch.arange(6, dtype=torch.float32).cuda()[:, None, None].expand(6, 4, 8).contiguous()
    pairs, graph = torch.tensor([[0, 3]], dtype=torch.int32).cuda(), torch.cuda.CUDAGraph()
    ops.copy_pages(pool, [(5, 4)])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(GlintError, match="captured"):
            ops.copy_pages(pool, [(1, 2)])
        ops.copy_pages(pool, pairs)
    for source in (1, 2, 0):
        pairs[0, 0] = source
        graph.replay()
        torch.cuda.synchronize()
        assert pool[:, 0, 0].tolist() == [0, 1, 2, source, 5, 5]


def test_two_at_a_time():
    """Two graphs with workspaces of their own, and eager calls on a third stream, at once."""
    made = [parts(i) for i in (1, 2, 3)]
    alone = []
    for m in made:
        xb, px = torch.zeros_like(m[3]), torch.zeros_like(m[3])
        alone.append((xb, px, *calls(m, rooms(m), xb, px)))
    torch.cuda.synchronize()
    graphs = []
    for m in made[:2]:
        xb, px, graph, room = torch.zeros_like(m[3]), torch.zeros_like(m[3]), torch.cuda.CUDAGraph(), rooms(m)
        with torch.cuda.graph(graph):
            got = calls(m, room, xb, px)
        graphs.append((graph, (xb, px, *got), room))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            xb, px = torch.zeros_like(made[2][3]), torch.zeros_like(made[2][3])
            third = (xb, px, *calls(made[2], rooms(made[2]), xb, px))
        torch.cuda.synchronize()
        for got, want in zip([g[1] for g in graphs] + [third], alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_the_same_call_gives_the_same_bits(dtype):
    made = parts(4, dtype)
    results = []
    for _ in range(5):
        xb, px = torch.zeros_like(made[3]), torch.zeros_like(made[3])
        results.append((xb, px, *calls(made, rooms(made), xb, px)))
    assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(results[0], other))


def test_work_queued_before_on_the_same_stream_is_seen():
    made = parts(5)
    pool, shape, p, q, lengths, logits, tokens = made
    xb, px = torch.zeros_like(q), torch.zeros_like(q)
    want = calls(made, rooms(made), xb, px)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        late_q, late_lengths = torch.zeros_like(q), torch.zeros_like(lengths)
        for _ in range(50):
            late_q.add_(1.0)
        late_q.copy_(q)
        late_lengths.copy_(lengths)
        a, b = torch.zeros_like(q), torch.zeros_like(q)
        got = calls((pool, shape, p, late_q, late_lengths, logits, tokens), rooms(made), a, b)
    stream.synchronize()
    assert torch.equal(a, xb) and torch.equal(b, px) and all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_workspace_serves_smaller_calls_and_none_smaller_is_taken():
    from glinthawk_amd._lib import GlintError

    pool = Pool([3000, 2900, 10], 1, 128, F16)
    shape = Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=1, hidden_dim=8, seq_len=8)
    p = ops.pages(pool.pool, pool.table)
    q = torch.randn((3, 1024), generator=torch.Generator().manual_seed(1)).half().cuda()
    size = ops.attn_decode_paged_workspace(3, 3000, shape, F16)
    guard = torch.full((size + 4096,), 77, dtype=torch.uint8, device="cuda")
    for batch in (1, 2, 3):
        for most in (1, 63, 64, 65, 500, 1000, 2000, 2999, 3000):
            assert ops.attn_decode_paged_workspace(batch, most, shape, F16) <= size
            lengths = torch.tensor([min(n, most) for n in pool.keys[:batch]], dtype=torch.int32).cuda()
            xb = torch.zeros((batch, 1024), dtype=F16, device="cuda")
            ops.attn_decode_paged(q[:batch], p, lengths, xb, most, shape, guard[:size])
            px = torch.zeros_like(xb)
            first = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
            ops.attn_packed(q[:batch], p, first, lengths - 1, px, most, shape, guard[:max(size, 16)])
            for i, n in enumerate(lengths.tolist()):
                want, off = attention(q[i:i + 1].reshape(1, 8, 128), pool.k(i)[:n], pool.v(i)[:n], n - 1, F16, True)
                hold(xb[i].reshape(1, 8, 128), want, off)
                hold(px[i].reshape(1, 8, 128), want, off)
    assert bool((guard[size:] == 77).all())
    lengths = torch.tensor(pool.keys, dtype=torch.int32).cuda()
    with pytest.raises(GlintError, match="workspace"):
        ops.attn_decode_paged(q, p, lengths, torch.zeros_like(q), 3000, shape, guard[:64])
    with pytest.raises(GlintError, match="16-byte"):
        ops.attn_decode_paged(q, p, lengths, torch.zeros_like(q), 3000, shape, guard[8:size])


def test_a_pool_beyond_32_bits():
    """Pages whose offsets pass 32 bits: a few tokens of a context at the far end of a pool of more than 4 GiB."""
    kv, page = 1024, 64
    n_pages = (5 << 30) // (2 * kv * 2 * page)
    pool = torch.empty((n_pages, page, 2 * kv), dtype=F16, device="cuda")
    small = Pool([200], 8, 128, F16, page)
    table = torch.tensor([[n_pages - 1, 3, n_pages - 2, n_pages // 2 + 7]], dtype=torch.int32).cuda()
    small.pool, line = pool, table[0].tolist()
    small.store(line, small.rows[0], 0)
    shape = Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=8, hidden_dim=8, seq_len=8)
    p = ops.pages(pool, table)
    q = torch.randn((200, 1024), generator=torch.Generator().manual_seed(1)).half().cuda()
    xb, px = torch.zeros_like(q[:1]), torch.zeros_like(q)
    ops.attn_decode_paged(q[199:], p, torch.tensor([200], dtype=torch.int32).cuda(), xb, 200, shape)
    ops.attn_packed(q, p, torch.tensor([0, 200], dtype=torch.int32).cuda(), None, px, 200, shape)
    want, off = attention(q.reshape(200, 8, 128), small.k(0), small.v(0), 0, F16, True)
    hold(px.reshape(200, 8, 128), want, off)
    hold(xb.reshape(1, 8, 128), want[199:], off[199:])
    ops.copy_pages(pool, [(n_pages - 1, 5)])
    assert torch.equal(pool[5], pool[n_pages - 1])
    rows, pos = ops.page_rows(p, torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.tensor([130], dtype=torch.int32).cuda(), 1)
    assert rows.tolist() == [pool[n_pages - 2, 2].data_ptr()] and pos.tolist() == [130]
