"""Log probabilities at the edges of what the call takes: tokens that are none, rows with one value."""
import pytest
import torch

from glinthawk_amd import ops
from pages_plain import STEP32, logprobs

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.init(0)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(5, 40), (300, 500), (40, 32000), (6, 70001)])
def test_tokens_that_are_none_have_nan(rows, vocab, dtype):
    """Padding in a batch that is scored: what stood in the result's memory before does not come out, and the other rows are as they are without it."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g).to(dtype).cuda()
    tokens = torch.randint(vocab, (rows,), generator=g, dtype=torch.int32).cuda()
    want = ops.token_logprobs(logits, tokens, 3)
    none = torch.zeros(rows, dtype=torch.bool, device="cuda")
    padded = tokens.clone()
    for row, token in ((0, -1), (2, vocab), (rows - 1, 2 ** 31 - 1), (rows // 2, -(2 ** 31))):
        padded[row], none[row] = token, True
    for _ in range(3):
        left = [torch.full((rows,), 5.0, device="cuda") for _ in range(16)]      # memory of the results' size, given back with values in it
        del left
        got = ops.token_logprobs(logits, padded, 3)
        assert torch.equal(torch.isnan(got[0]), none)
        assert torch.equal(got[0][~none], want[0][~none]) and all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


def test_the_value_for_tokens_that_are_none():
    from glinthawk_amd._lib import check as ok, lib
    logits, tokens = torch.randn(4, 100).cuda(), torch.tensor([3, -1, 100, 99], dtype=torch.int32).cuda()
    given = torch.zeros(4).cuda()
    ok(lib().gh_token_logprobs_fill(given.data_ptr(), -2.5, None, None, None, logits.data_ptr(), 100, tokens.data_ptr(), 100, 4, 0, 1, None, 0, ops._stream()))
    want = logprobs(logits, tokens.clamp(0, 99), 1)[0]
    assert given[1] == -2.5 and given[2] == -2.5
    assert float((given.double() - want)[[0, 3]].abs().max()) <= 32 * STEP32 * 8


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab,values", [(40, 60000), (5000, 3000), (40000, 1000)])
def test_one_finite_value_has_the_whole_weight(vocab, values, dtype):
    """A constrained step that leaves one token: its log probability is 0, not above, and the entropy 0, not below (f16: powers of 2 relative to a rounded point within
    2^-16 (300 log2(e) < 2^9), one product with it off by its last place, 2^-24 of it)."""
    x = torch.full((values, vocab), -INF, dtype=dtype, device="cuda")
    x[:, 3] = torch.linspace(-300, 300, values).to(dtype).cuda()
    given, entropy, ids, top = ops.token_logprobs(x, torch.full((values,), 3, dtype=torch.int32, device="cuda"), 1)
    assert bool((given == 0).all()) and bool((entropy >= 0).all()) and float(entropy.max()) <= (2.0 ** -40 if dtype == F16 else 0) and bool((top == 0).all()) and bool((ids == 3).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_log_probabilities_are_never_above_zero(dtype):
    """One value far above the others, whose weights do not reach the sum's last place."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn((4000, 900), generator=g).to(dtype).cuda()
    x[:, 5] = torch.linspace(15, 60, 4000).to(dtype).cuda()
    given, entropy, _, top = ops.token_logprobs(x, torch.full((4000,), 5, dtype=torch.int32, device="cuda"), 2)
    assert bool((given <= 0).all()) and bool((top <= 0).all()) and bool((entropy >= 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_alternatives_of_a_product(dtype):
    """Logits as the dense product gives them: the alternatives' indices in every type, the first of them what the argmax says where that takes the type."""
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn((4, 512), generator=g).to(dtype).cuda(), torch.randn((777, 512), generator=g).to(dtype).cuda()
    logits = ops.matmul(x, w)
    ids = ops.token_logprobs(logits, torch.tensor([0, 5, 776, 100], dtype=torch.int32).cuda(), 7)[2]
    assert torch.equal(ids.long(), logprobs(logits, torch.zeros(4, dtype=torch.int32).cuda(), 7)[2])
    if dtype != BF16:
        assert ops.argmax(logits) == ids[:, 0].tolist()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1500, 5000, 32000, 70001])
def test_rows_that_let_few_tokens_through(vocab, dtype):
    """Grammar masks: some values, -inf elsewhere, NaN among it or not, fewer values than alternatives or more, in one place or apart; and rows where most values are equal."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((12, vocab), generator=g)
    rows = torch.full((12, vocab), -INF)
    for row, allowed in enumerate((range(100, 130), [vocab - 1], range(3, vocab, vocab // 5), range(0, vocab, 3), [], range(vocab - 70, vocab), [0, 1, 2])):
        rows[row, list(allowed)] = x[row, list(allowed)]
    rows[7] = 2.0
    rows[7, 40:vocab:700] = 3.0
    rows[8] = torch.where(x[8] > 1.5, x[8], 1.0)
    rows[9] = -0.0
    rows[9, ::2] = 0.0
    rows[9, 77] = -1.0
    rows[10, 5:9] = x[10, 5:9]
    rows[10, vocab // 2:] = float("nan")
    rows[11] = float("nan")
    rows[11, vocab - 2] = 1.0
    rows[11, 300] = -INF
    rows = rows.to(dtype).cuda()
    for n_top in (1, 5, 20, 64):
        ids = ops.token_logprobs(rows, torch.zeros(12, dtype=torch.int32, device="cuda"), n_top)[2]
        want = logprobs(rows, torch.zeros(12, dtype=torch.int32, device="cuda"), n_top)[2]
        for row in range(12):
            assert ids[row].tolist() == want[row].tolist(), (row, n_top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n_top", [5, 64])
def test_rows_that_let_few_tokens_through_are_no_long_call(n_top, dtype):
    x = torch.randn((1000, 32000), device="cuda").to(dtype)
    masked = torch.full_like(x, -INF)
    masked[:, 100:130] = x[:, 100:130]
    tokens = torch.zeros(1000, dtype=torch.int32, device="cuda")

    def fastest(logits):
        times = []
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            ops.token_logprobs(logits, tokens, n_top)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times[1:])

    usual, few = fastest(x), fastest(masked)
    assert few < 6 * usual, f"{few * 1e3:.0f} us, without a mask {usual * 1e3:.0f}"
