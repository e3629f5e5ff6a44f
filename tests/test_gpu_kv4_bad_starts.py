"""Queries that no sequence answers, because its starts are out of order or past the queries, are zeros beside the flag."""
import pytest
import torch

from tests import kv4_plain as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts,owned", [
    ([0, 4, 900], [(0, 0, 4)]),          # the second ends past the queries
    ([0, 700, 12], []),                  # the first does, and the second goes back
    ([-3, 5, 12], [(1, 5, 12)]),         # the first begins before them
    ([3, 3, 12], [(1, 3, 12)]),          # in order: the first three belong to nobody
    ([900, 901, 902], []),
    ([6, 2, 10], [(1, 6, 10)]),          # the first ends before it begins: 2 to 5 are before the first start, too
])
@pytest.mark.parametrize("heads", [2, 16, 128])
def test_rows_of_skipped_sequences_are_zeros(starts, owned, heads):
    from torch_ans_b200 import _C
    _C.device_status()
    pages, total = P.table([100, 40], 16)
    codes, params = P.pool(total, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(12, heads, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    ln, st = torch.tensor([100, 40], **i32), torch.tensor(starts, **i32)
    want = torch.zeros_like(q)
    if starts == [6, 2, 10]:
        both = _C.kv4_attend(q[2:10], codes, params, pages[1:].contiguous(), ln[1:].contiguous(),
                             q_starts=torch.tensor([0, 8], **i32), max_queries=12)[:4].float()[None]
    for b, lo, hi in owned:
        first = starts[b] if starts[b] >= 0 else lo
        want[lo:hi] = _C.kv4_attend(q[first:hi], codes, params, pages[b: b + 1].contiguous(), ln[b: b + 1].contiguous(),
                                    q_starts=torch.tensor([0, hi - first], **i32), max_queries=12)[lo - first:]
    assert _C.device_status() == 0
    for _ in range(3):
        dirt = torch.full_like(q, float("nan"))  # what the output's memory may hold
        del dirt
        lse = torch.full((12, heads), 7.0, device="cuda")
        out = _C.kv4_attend(q, codes, params, pages, ln, q_starts=st, max_queries=12, lse=lse)
        answered = torch.zeros(12, dtype=torch.bool)
        for b, lo, hi in owned:
            answered[lo:hi] = True
        if starts == [6, 2, 10]:
            early = out[2:6].float()
            assert ((early - both[0]).abs() <= 0.02).logical_or(early == 0).all()
            out[2:6], lse[2:6] = 0, float("-inf")
        assert out[~answered].eq(0).all() and torch.isneginf(lse[~answered]).all()
        assert torch.allclose(out.float(), want.float(), atol=0.02) and lse[answered].isfinite().all()
    assert _C.device_status() == (0 if starts == [3, 3, 12] else 2)


def test_sequences_that_overlap_leave_nothing_unwritten():
    """More row tiles than their number of queries allows for."""
    from torch_ans_b200 import _C
    _C.device_status()
    n, batch = 300, 40
    pages, total = P.table([50] * batch, 16)
    codes, params = P.pool(total, 1, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, n] * (batch // 2) + [n], **i32)
    q = torch.randn(n, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    for most in (1, n):
        for _ in range(3):
            dirt = torch.full_like(q, float("nan"))
            del dirt
            out = _C.kv4_attend(q, codes, params, pages, torch.full((batch,), 50, **i32), q_starts=starts, max_queries=most)
            assert out.isfinite().all()
            assert _C.device_status() == 2


def test_more_work_than_a_call_takes_gives_zeros():
    """80 sequences of 2^30 tokens (one page again and again): refused on the device, nothing is left unwritten."""
    from torch_ans_b200 import _C
    _C.device_status()
    page, batch = 1 << 20, 80
    codes = torch.zeros(1, 2, 1, page, 32, dtype=torch.uint8, device="cuda")
    params = torch.zeros(1, 2, 1, page, 2, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.ones(batch, 1, 64, dtype=torch.bfloat16, device="cuda")
    dirt = torch.full_like(q, float("nan"))
    del dirt
    lse = torch.zeros(batch, 1, device="cuda")
    out = _C.kv4_attend(q, codes, params, torch.zeros(batch, 1024, **i32), torch.full((batch,), 1 << 30, **i32), lse=lse)
    assert out.eq(0).all() and torch.isneginf(lse).all() and _C.device_status() == 2
