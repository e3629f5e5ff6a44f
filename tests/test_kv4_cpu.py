"""The 4-bit key/value cache without a GPU: the ops are there, refuse CPU tensors and bad arguments before any device
work, and the plain definitions that the GPU tests compare with agree with each other."""
import ctypes

import pytest
import torch

from tests import kv4_plain as P

OPS = ["kv4_append", "kv4_gather", "kv4_attend", "kv4_to_symbols", "kv4_from_symbols"]


def test_ops_are_there_and_refuse_cpu_tensors():
    from torch_ans_b200 import _C
    codes, params = P.pool(2, 1, 16, 64, device="cpu")
    rows, ids = torch.zeros(3, 1, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    i32 = dict(dtype=torch.int32)
    for op in OPS:
        assert hasattr(_C, op)
    for f in (lambda: _C.kv4_append(codes, params, rows, rows, ids), lambda: _C.kv4_gather(codes, params, ids, torch.float16),
              lambda: _C.kv4_attend(rows, codes, params, torch.zeros(3, 1, **i32), torch.zeros(3, **i32)),
              lambda: _C.kv4_to_symbols(codes, ids), lambda: _C.kv4_from_symbols(torch.zeros(2, 1024, **i32), codes, ids[:1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_capi_refuses_bad_arguments_without_touching_the_device():
    from torch_ans_b200 import capi
    lib = capi.load()
    p = 1 << 20  # an aligned address that no refused call reads
    ok = dict(codes=p, params=p, num_pages=4, kv_heads=2, page_size=16, head_dim=64, dtype=0)

    def append(tokens=3, k=p, rotation=None, rows=0, rotary=0, positions=None, q=None, q_heads=0, q_out=None, **kw):
        a = {**ok, **kw}
        return lib.tans_kv4_append(a["codes"], a["params"], a["num_pages"], a["kv_heads"], a["page_size"], a["head_dim"],
                                   a["dtype"], k, 128, 64, p, 128, 64, q, 128, 64, q_heads, q_out, p, tokens, rotation,
                                   rows, rotary, positions, 0, None, None)

    def attend(total=3, batch=3, q_heads=4, starts=None, most=1, q=p, out=p, ws=p, ws_bytes=0, max_pages=1, **kw):
        a = {**ok, **kw}
        return lib.tans_kv4_attend(q, 256, 64, total, q_heads, a["dtype"], a["codes"], a["params"], a["num_pages"],
                                   a["kv_heads"], a["page_size"], a["head_dim"], p, batch, max_pages, p, starts, most,
                                   ctypes.c_float(0.125), 1, out, None, ws, ws_bytes, None, None)

    assert append(tokens=0) == 0 and attend(total=0, batch=0) == 0  # nothing to do
    for bad in (dict(head_dim=96), dict(page_size=24), dict(page_size=0), dict(kv_heads=0), dict(num_pages=-1), dict(dtype=2),
                dict(codes=p + 4), dict(params=p + 8), dict(codes=None)):
        assert append(**bad) == 1, bad
        assert attend(**bad) == 1, bad
    for bad in (dict(tokens=-1), dict(k=None), dict(rotation=p, rows=5, rotary=24, positions=p),
                dict(rotation=p, rows=5, rotary=128, positions=p), dict(rotation=p, rows=0, rotary=64, positions=p),
                dict(rotation=p, rows=5, rotary=64), dict(rotation=p + 4, rows=5, rotary=64, positions=p),
                dict(q=p, q_heads=2), dict(q=p, q_heads=0, q_out=p), dict(q=p, q_heads=2, q_out=p + 2)):
        assert append(**bad) == 1, bad
    for bad in (dict(total=-1), dict(batch=-1), dict(batch=2), dict(q_heads=3), dict(q_heads=0), dict(most=-1), dict(q=None),
                dict(out=None), dict(out=p + 8), dict(max_pages=-1)):
        assert attend(**bad) == 1, bad
    assert attend() == 3  # a workspace that is too small
    assert attend(total=1 << 29, batch=1 << 29, q_heads=4) == 4
    size = lib.tans_kv4_attend_workspace_size
    assert size(3, 4, 2, 64, 3, 1, 16, 1) >= 10240 and size(0, 4, 2, 64, 0, 0, 16, 0) == 0
    assert lib.tans_kv4_to_symbols(p, 4, 2, 16, 80, p, 1, 0, p, p, None, None) == 1
    assert lib.tans_kv4_to_symbols(p, 4, 2, 16, 64, p, 1, 0, p + 4, p, None, None) == 1
    assert lib.tans_kv4_from_symbols(p, p, 4, 2, 16, 64, None, 1, None, None) == 1
    assert lib.tans_kv4_gather(p, p, 4, 2, 16, 64, 0, p, 1, p, None, None, None) == 1


def test_header_names_the_size_of_the_counts():
    from torch_ans_b200 import capi
    text = open(capi.HEADER).read()
    assert "#define TANS_KV4_ATTEND_COUNTS 10240" in text


@pytest.mark.parametrize("interleaved", [False, True])
def test_plain_rotation_keeps_lengths_and_products(interleaved):
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(5, 2, 64, dtype=torch.float64, generator=g) for _ in range(2))
    angle = torch.arange(9).double()[:, None] * 10000.0 ** (-torch.arange(0, 32, 2).double() / 32)
    rot = torch.cat([angle.cos(), angle.sin()], 1)  # in 64 bits: the premise is cos^2 + sin^2 = 1 to 1e-15
    pos = torch.tensor([0, 1, 8, 3, 3])
    a, b = P.rotate(x, pos, rot, interleaved), P.rotate(y, pos, rot, interleaved)
    assert torch.equal(a[0], x[0]) and torch.equal(a[..., 32:], x[..., 32:])
    assert torch.allclose((a * b).sum(-1), (x * y).sum(-1), rtol=0, atol=1e-12)  # the same turn on both sides


def test_plain_attention_against_a_loop():
    lengths, counts, page = [5, 0, 33], [2, 1, 33], 16
    pages, total = P.table(lengths, page, device="cpu")
    codes, params = P.pool(total, 2, page, 64, device="cpu")
    starts = [0, 2, 3, 36]
    q = torch.randn(36, 4, 64, generator=torch.Generator().manual_seed(1))
    out, lse, bound, _ = P.attend(q, codes, params, pages, lengths, starts, 0.2)
    for b in range(3):
        for i in range(counts[b]):
            for h in range(4):
                rows = range(max(0, lengths[b] - counts[b] + i + 1))
                at = [(int(pages[b, t // page]), t % page) for t in rows]
                k = [P.values(codes[p, 0, h // 2, s], params[p, 0, h // 2, s]) for p, s in at]
                v = [P.values(codes[p, 1, h // 2, s], params[p, 1, h // 2, s]) for p, s in at]
                row = starts[b] + i
                if not at:
                    assert out[row, h].eq(0).all() and lse[row, h] == float("-inf")
                    continue
                s = torch.stack([(q[row, h].double() * x).sum() * 0.2 for x in k])
                w = torch.exp(s - s.max())
                assert torch.allclose(out[row, h], (w[:, None] * torch.stack(v)).sum(0) / w.sum(), atol=1e-12)
                assert abs(float(lse[row, h] - s.max() - w.sum().log())) < 1e-12
    assert torch.equal(P.pack(P.unpack(codes)), codes)


def test_pages_are_given_out_and_taken_back():
    from torch_ans_b200.kv_cache import PagedKVCache4
    cache = PagedKVCache4(5, 1, 64, device="cpu")
    step = cache.reserve([1, 2, 3], [16, 0, 17])  # one page, none, two
    assert step.pages.shape == (3, 2) and step.slots.numel() == 33 and step.max_queries == 17
    assert len(set(step.slots.tolist())) == 33 and step.positions.tolist() == list(range(16)) + list(range(17))
    assert step.q_starts.tolist() == [0, 16, 16, 33] and step.lengths.tolist() == [16, 0, 17]
    assert step.pages[0, 1] == -1 and step.pages[1].tolist() == [-1, -1]
    with pytest.raises(RuntimeError, match="free pages"):
        cache.reserve([1, 2], [16, 17])  # three pages of the two that are free
    assert cache.length(1) == 16 and cache.length(2) == 0
    cache.free(3)
    step = cache.reserve([1, 2], [16, 17])  # three of four
    assert cache.length(1) == 32 and step.positions.tolist() == list(range(16, 32)) + list(range(17))
    with pytest.raises(RuntimeError, match="free pages"):
        cache.reserve([4], [17])
    assert cache.length(4) == 0
    for bad in (dict(head_dim=80), dict(page_size=24), dict(num_pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            PagedKVCache4(**{**dict(num_pages=1, kv_heads=1, head_dim=64, device="cpu"), **bad})
