"""As tests/test_gpu_kv4_value_range.py, where many query rows share a key/value head; and keys of hidden tokens."""
import pytest
import torch

from tests.kv4_planted import Planted
from tests.test_gpu_kv4_value_range import (BETA, BF, COUNTS_PROMPT, FP, C, hidden_values, small_values,  # noqa: F401
                                            unlikely_values)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [0, 5, 7, 12, 20, 40, 100])
@pytest.mark.parametrize("dim,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("how", [unlikely_values, hidden_values, small_values])
@pytest.mark.parametrize("counts", COUNTS_PROMPT)
def test_values_that_do_not_count_many_rows(C, counts, how, dim, dtype, exponent):  # noqa: F811
    how(C, dim, dtype, counts, exponent)


@pytest.mark.parametrize("exponent", [5, 12, 24, 40, 100])
@pytest.mark.parametrize("dim,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("counts", [[5, 6], [70, 64]])
def test_large_keys_of_hidden_tokens(C, counts, dim, dtype, exponent):  # noqa: F811
    """A token after a query's own has a key of any size: the answers do not change."""
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    q, wanted = c.queries(counts, 4, dtype, beta=BETA[dim])
    out, bound = c.answers(q, wanted, counts)
    for b, n in enumerate(c.lengths):
        c.resize(b, [n - 1], 0, exponent)
    bad = c.wrong(c.attend(C, q, counts), out, bound)
    last = torch.tensor([counts[0] - 1, sum(counts) - 1], device="cuda")  # these see the token
    bad[last] = False
    assert not bad.any() and C.device_status() == 0


@pytest.mark.parametrize("dim,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("counts", [[70, 64], [300, 257]])
def test_values_of_all_sizes_in_one_context(C, counts, dim, dtype):  # noqa: F811
    """Blocks of 32 tokens whose values are 2^-8 .. 2^8 times the ordinary, each wanted by some query."""
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    for b, n in enumerate(c.lengths):
        for t in range(n):
            c.resize(b, [t], 1, (t // 32 * 5) % 17 - 8)
    q, wanted = c.queries(counts, 4, dtype)
    out, bound = c.answers(q, wanted, counts)
    bad = c.wrong(c.attend(C, q, counts), out, bound)
    assert not bad.any() and C.device_status() == 0
