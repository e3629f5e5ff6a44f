"""Tokens whose values or keys are much larger than the others' and whose weight is nothing: the answers are those of the
tokens that count, as exact as without them (tests/kv4_planted.py has the bound)."""
import pytest
import torch

from tests.kv4_planted import Planted

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
BETA = {64: 26.0, 128: 36.0, 256: 50.0}  # an unlikely token is under e^-95 then: nothing even where values are 2^100 larger


@pytest.fixture(scope="module")
def C():
    from torch_ans_b200 import _C
    _C.set_sync_check(False)
    _C.device_status()
    return _C


COUNTS_ROWS, COUNTS_PROMPT = [[1, 1], [5, 6]], [[70, 64], [300, 257]]


def unlikely_values(C, dim, dtype, counts, exponent):
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    for b, tokens in enumerate(([3, 290], [0, 500, 1029])):
        c.unlikely(b, tokens)
        c.resize(b, tokens, 1, exponent)
    c.check(C, counts, 4, dtype, beta=BETA[dim])


def hidden_values(C, dim, dtype, counts, exponent):
    """The last token, which only a sequence's last query sees, has large values; that query's answer is checked too."""
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    for b, n in enumerate(c.lengths):
        c.unlikely(b, [n - 1])
        c.resize(b, [n - 1], 1, exponent)
    c.check(C, counts, 4, dtype, beta=BETA[dim])


def small_values(C, dim, dtype, counts, exponent):
    """Among tokens of ordinary values whose weight is nothing, tokens with small ones are the whole answer."""
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    for b, n in enumerate(c.lengths):
        few = [t for t in range(n) if t // 32 % 4 == 1]
        c.resize(b, [t for t in range(n) if t not in few], 1, exponent)
        c.unlikely(b, [t for t in range(n) if t not in few])
    q, wanted = c.queries(counts, 4, dtype, beta=BETA[dim])
    at, sees = 0, []
    for b, n in enumerate(counts):  # the block of small values is what each query wants
        sees += [i + c.lengths[b] - n >= 63 for i in range(n)]
        pattern = c.pattern[b][torch.arange(c.kv).repeat_interleave(4), 1].float() * {64: 8.0, 128: 4.0, 256: 2.0}[dim]
        pattern[:, :16] = BETA[dim]
        q[at: at + n], wanted[at: at + n] = pattern.to(dtype), 1
        at += n
    out, bound = c.answers(q, wanted, counts)
    sees = torch.tensor(sees, device="cuda")  # the others have none of the block before them
    assert out[sees].square().mean().sqrt() > 30 * bound[sees].mean()
    bad = c.wrong(c.attend(C, q, counts), out, bound)
    assert not bad[sees].any() and C.device_status() == 0


@pytest.mark.parametrize("exponent", [0, 5, 7, 12, 20, 40, 100])
@pytest.mark.parametrize("dim,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("how", [unlikely_values, hidden_values, small_values])
@pytest.mark.parametrize("counts", COUNTS_ROWS)
def test_values_that_do_not_count_few_rows(C, counts, how, dim, dtype, exponent):
    how(C, dim, dtype, counts, exponent)
