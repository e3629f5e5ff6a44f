"""Waits that run out: the call ends, with the flag, whichever of its warps came through and which did not, the workspace's
counts are zero, and the next call with it is right, whether or not anybody read the flag.  (Waits are bounded: with a limit of 0 each ends at once.)"""
import ctypes

import pytest
import torch

from tests import kv4_plain as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,counts", [([700, 300], [700, 300]), ([9000], [300]), ([20000], [70]), ([300] * 40, [60] * 40)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_calls_end_and_the_next_one_is_right(monkeypatch, lengths, counts, dim):
    from torch_ans_b200 import _C, capi
    lib = capi.load()
    heads, kv = 8, 2
    pages, total = P.table(lengths, 16)
    codes, params = P.pool(total, kv, 16, dim)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], **i32)
    n, batch, most, ln = sum(counts), len(lengths), max(counts), torch.tensor(lengths, **i32)
    q = torch.randn(n, heads, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    size = lib.tans_kv4_attend_workspace_size(n, heads, kv, dim, batch, pages.shape[1], 16, most)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, **i32)

    def call():
        out = torch.zeros_like(q)
        rc = lib.tans_kv4_attend(q.data_ptr(), heads * dim, dim, n, heads, 0, codes.data_ptr(), params.data_ptr(), total, kv, 16,
                                 dim, pages.data_ptr(), batch, pages.shape[1], ln.data_ptr(), starts.data_ptr(), most,
                                 ctypes.c_float(dim ** -0.5), 1, out.data_ptr(), None, ws.data_ptr(), size, status.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        return out

    first = call()
    assert status.item() == 0 and ws[:10240].eq(0).all()
    for limit in ["0"] + ["1", "2", "3"] * 10:  # in between, some blocks of a row tile come through and some do not
        monkeypatch.setenv("TORCH_ANS_B200_WAIT_LIMIT", limit)
        call()
        assert ws[:10240].eq(0).all(), limit
        assert limit != "0" or status.item() == 64
        monkeypatch.delenv("TORCH_ANS_B200_WAIT_LIMIT")
        status.zero_()
        assert torch.equal(call(), first) and status.item() == 0
    assert _C.device_status() == 0


def test_a_long_piece_of_work_is_not_a_stall(monkeypatch):
    """The warp that looks work up waits while a row tile's tokens are gone through, which takes as long as they are many:
    524,288 here (one page again and again), some ten milliseconds, under a limit of less than one."""
    from torch_ans_b200 import _C
    _C.device_status()
    page, heads, n = 1 << 14, 64, 700
    codes, params = P.pool(1, 1, page, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, 32, **i32)
    q = torch.randn(n, heads, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    args = (q, codes, params, pages, torch.tensor([32 * page], **i32))
    kw = dict(q_starts=torch.tensor([0, n], **i32), max_queries=n)
    first = _C.kv4_attend(*args, **kw)
    assert _C.device_status() == 0
    monkeypatch.setenv("TORCH_ANS_B200_WAIT_LIMIT", "700")
    assert torch.equal(_C.kv4_attend(*args, **kw), first)
    assert _C.device_status() == 0
