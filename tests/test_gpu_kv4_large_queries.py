"""Finite queries of any size give finite answers: a softmax with all its weight on one block of tokens.  Scores reach 2^124, so
only tokens with equal keys are within an error of one another, and the bound of tests/kv4_planted.py holds as it is."""
import pytest
import torch

from tests.kv4_planted import Planted

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    from torch_ans_b200 import _C
    _C.set_sync_check(False)
    _C.device_status()
    return _C


@pytest.mark.parametrize("exponent,keys", [(8, 0), (30, 0), (60, 0), (100, 0), (112, 0), (116, 0), (118, 0), (122, -30), (-100, 100), (-116, 116)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1], [6], [100]])
def test_queries_of_any_size(C, counts, dim, exponent, keys):
    c = Planted([300], 16, 1, dim, 32, seed=dim)
    c.resize(0, range(300), 0, keys)
    q, wanted = c.queries(counts, 4, torch.bfloat16, size=2.0 ** exponent)
    assert q.isfinite().all()
    out, bound = c.answers(q, wanted, counts)
    got = c.attend(C, q, counts)
    assert got.isfinite().all()
    assert out.square().mean().sqrt() > 30 * bound.mean()
    assert not c.wrong(got, out, bound).any() and C.device_status() == 0


@pytest.mark.parametrize("exponent", [3, 4, 5, 6, 7, 12, 16, 20, 22, 24, 40])
@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16)])
@pytest.mark.parametrize("counts", [[1, 1], [5, 6], [70, 64], [300, 257]])
def test_large_scores_with_values_of_all_sizes(C, counts, dim, dtype, exponent):
    """Scores of 2^8 to 2^46 (keys grow, so float16 queries reach them too) and blocks whose values are 2^-32 .. 2^32 times the
    ordinary."""
    c = Planted([300, 1030], 16, 2, dim, 32, seed=dim)
    for b, n in enumerate(c.lengths):
        c.resize(b, range(n), 0, exponent)
        for t in range(n):
            c.resize(b, [t], 1, ((t // 32 * 5) % 17 - 8) * (4 if dtype == torch.bfloat16 else 1))
    q, wanted = c.queries(counts, 4, dtype)
    out, bound = c.answers(q, wanted, counts)
    assert not c.wrong(c.attend(C, q, counts), out, bound).any() and C.device_status() == 0


@pytest.mark.parametrize("exponent", [10, 14, 20, 40, 60])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1, 1, 1], [7, 3, 5], [300, 143, 718]])
def test_equal_large_scores_wherever_they_are(C, counts, dim, exponent):
    """Blocks of 128 tokens, which many warps share: their equal scores stay equal beside others that are far away, and after steps
    whose values differ by more than 2^12."""
    c = Planted([353, 143, 1880], 32, 2, dim, 128, seed=dim + 1)
    for b, n in enumerate(c.lengths):
        c.resize(b, range(n), 0, exponent)
    c.unlikely(2, [700, 1100, 1200])
    c.resize(2, [700, 1100, 1200], 1, 16)
    for first in (0, 5, 11):
        q, wanted = c.queries(counts, 4, torch.bfloat16, beta={64: 26.0, 128: 36.0, 256: 50.0}[dim], first=first)
        out, bound = c.answers(q, wanted, counts)
        assert not c.wrong(c.attend(C, q, counts), out, bound).any() and C.device_status() == 0
