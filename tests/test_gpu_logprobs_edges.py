"""Log probabilities at the edges of what the call takes: tokens that are none."""
import pytest
import torch

from glinthawk_amd import ops
from pages_plain import STEP32, logprobs

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


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
