"""Log probabilities of given tokens, entropy and the largest alternatives against 64 bits."""
import math

import pytest
import torch

from glinthawk_amd import ops
from pages_plain import STEP32, logprobs

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


def check(logits, tokens, n_top, got=None):
    given, entropy, ids, values = ops.token_logprobs(logits, tokens, n_top) if got is None else got
    want = logprobs(logits, tokens, n_top)
    assert torch.equal(ids.long(), want[2])
    # differences of fp32 values as large as the logits, each rounded; the sum of V weights, each off by its exponent's rounding, in chains of V / 1024 and a tree;
    # the logarithm's own step
    finite = torch.where(torch.isfinite(logits), logits, 0.0).double().abs().amax(1)
    sums = (8 + 4 * finite + logits.shape[1] / 1024 + 12) * STEP32
    for a, b in ((given, want[0]), (values, want[3])):
        room = sums if a.dim() == 1 else sums[:, None]
        off = room + 4 * STEP32 * torch.where(torch.isfinite(b), b, 0.0).abs()
        assert bool((((a.double() - b).abs() <= off) | (a.double() == b)).all())
    assert bool(((entropy.double() - want[1]).abs() <= sums * (2 + math.log(logits.shape[1]))).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 63), (2, 65), (4, 1000), (1, 4096), (9, 4097), (300, 777), (1, 32000), (33, 32000), (2, 32001), (1, 130001), (700, 8200)])
def test_sizes(rows, vocab, dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    logits = (4 * torch.randn((rows, vocab), generator=g)).to(dtype).cuda()
    tokens = torch.randint(vocab, (rows,), generator=g, dtype=torch.int32).cuda()
    for n_top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        check(logits, tokens, n_top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [100, 5000, 32000])
def test_equal_values_masked_values_and_nan(vocab, dtype):
    g = torch.Generator().manual_seed(5)
    logits = torch.randint(-2, 3, (8, vocab), generator=g).float()      # nothing but equal values
    logits[1] = 0.0
    logits[1, ::2] = -0.0
    logits[2] = -INF
    logits[2, 17] = 3.0
    logits[3, 1:] = torch.finfo(dtype).min                              # the type's lowest value
    logits[4, : vocab // 2] = -INF
    logits[5] = torch.linspace(-30, 30, vocab)                          # one thread after the other has the largest
    logits[6] = torch.linspace(30, -30, vocab)
    logits = logits.to(dtype).cuda()
    tokens = torch.full((8,), 17, dtype=torch.int32).cuda()
    for n_top in (1, 7, 64):
        check(logits, tokens, n_top)
    logits[7, 3] = NAN
    given, entropy, ids, values = ops.token_logprobs(logits, tokens, 64)
    check(logits[:7], tokens[:7], 64, (given[:7], entropy[:7], ids[:7], values[:7]))
    assert math.isnan(given[7]) and math.isnan(entropy[7]) and bool(torch.isnan(values[7]).all())
    assert torch.equal(ids[7].long(), logprobs(logits[7:], tokens[7:], 64)[2][0])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [33, 1000, 32000, 40000])
def test_rows_of_the_largest_and_lowest_values(vocab, dtype):
    """Whole rows at the ends of the type, where a value times log2(e) leaves fp32, and what is about 1e30 away from 0."""
    logits = torch.zeros((7, vocab))
    ends = torch.finfo(dtype)
    logits[0] = ends.min
    logits[1] = ends.max
    logits[2, ::2] = ends.min
    logits[2, 1::2] = -INF
    logits[3] = ends.min
    logits[3, 5] = ends.max
    big = min(1e30, float(ends.max) / 4)
    logits[4] = -big
    logits[4, 7] = -0.7 * big
    logits[5] = 0.5 * big
    logits[5, ::3] = 0.6 * big
    logits[6] = -0.69 * big
    logits = logits.to(dtype).cuda()
    given, entropy, ids, values = ops.token_logprobs(logits, torch.full((7,), 7, dtype=torch.int32).cuda(), 20)
    want = logprobs(logits, torch.full((7,), 7, dtype=torch.int32).cuda(), 20)
    assert torch.equal(ids.long(), want[2])
    # equal values have one weight each and the others none, so a row's sums are a whole number n; what is left is the logarithm and the difference to the maximum,
    # each off by its own step (both below 12 where they are finite in fp32, or the difference is all there is)
    for got, exact in ((given, want[0]), (entropy, want[1]), (values, want[3])):
        exact = exact.float().double()
        assert bool((((got.double() - exact).abs() <= 4 * STEP32 * (12 + exact.abs())) | (got.double() == exact)).all())


@pytest.mark.parametrize("vocab", [900, 32000, 40000])
def test_values_far_from_zero(vocab):
    g = torch.Generator().manual_seed(9)
    base = torch.tensor([sign * 10.0 ** e for e in (3, 5, 6, 6.05, 7, 9, 12, 20, 30, 37) for sign in (1, -1)])
    logits = (base[:, None].double() + 3 * torch.randn((20, vocab), generator=g).double()).float().cuda()
    tokens = torch.randint(vocab, (20,), generator=g, dtype=torch.int32).cuda()
    for n_top in (1, 20, 64):
        check(logits, tokens, n_top)


def test_nan_and_infinities_only():
    logits = torch.tensor([[NAN] * 70, [-INF] * 70, [INF] * 2 + [0.0] * 68]).cuda()
    given, entropy, ids, values = ops.token_logprobs(logits, torch.zeros(3, dtype=torch.int32).cuda(), 64)
    assert bool(torch.isnan(given).all()) and bool(torch.isnan(entropy).all())
    assert ids.tolist() == [list(range(64))] * 3


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,vocab,stride", [(3, 500, 512), (5, 32000, 32007), (2, 70001, 70016)])
def test_rows_that_lie_apart_and_tokens_that_are_none(rows, vocab, stride, dtype):
    wide = torch.full((rows, stride), NAN, dtype=dtype, device="cuda")
    wide[:, :vocab] = torch.randn((rows, vocab), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    tokens = torch.randint(vocab, (rows,), dtype=torch.int32).cuda()
    check(wide[:, :vocab], tokens, 10)
    check(wide[:, 1:vocab], tokens.clamp(max=vocab - 2), 10)
    given = torch.full((rows,), 5.0, device="cuda")
    tokens[0], tokens[1] = vocab, -1
    from glinthawk_amd._lib import check as ok, lib
    room = torch.empty(max(16, ops.token_logprobs_workspace(rows, vocab, 0)), dtype=torch.uint8, device="cuda")
    ok(lib().gh_token_logprobs(given.data_ptr(), None, None, None, wide.data_ptr(), stride, tokens.data_ptr(), vocab, rows, 0, ops._dt(wide), room.data_ptr(), room.numel(),
                               ops._stream()))
    assert given[0] == 5.0 and given[1] == 5.0 and bool((given[2:] < 0).all())


def test_only_what_is_wanted():
    from glinthawk_amd._lib import check as ok, lib
    logits = torch.randn(4, 40000).cuda()
    room = torch.empty(ops.token_logprobs_workspace(4, 40000, 3), dtype=torch.uint8, device="cuda")
    ids, values, entropy = torch.zeros((4, 3), dtype=torch.int32).cuda(), torch.zeros((4, 3)).cuda(), torch.zeros(4).cuda()
    common = logits.data_ptr(), 40000
    ok(lib().gh_token_logprobs(None, None, ids.data_ptr(), values.data_ptr(), *common, None, 40000, 4, 3, 1, room.data_ptr(), room.numel(), ops._stream()))
    ok(lib().gh_token_logprobs(None, entropy.data_ptr(), None, None, *common, None, 40000, 4, 0, 1, room.data_ptr(), room.numel(), ops._stream()))
    want = logprobs(logits, torch.zeros(4, dtype=torch.int32).cuda(), 3)
    assert torch.equal(ids.long(), want[2]) and float((entropy - want[1]).abs().max()) < 1e-4
