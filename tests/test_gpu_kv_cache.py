"""PagedKVCache4 as a serving program uses it: prompts and single tokens in and answered, a sequence stored through
the entropy coder and loaded again."""
import pytest
import torch

from tests import kv4_plain as P

pytestmark = pytest.mark.gpu


def rotation(rows, r):
    angle = torch.arange(rows, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, r, 2, device="cuda") / r)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def projection(n, heads, kv, dim, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, (heads + 2 * kv) * dim, device="cuda", generator=g).to(dtype)
    return [t.unflatten(1, (-1, dim)) for t in x.split([heads * dim, kv * dim, kv * dim], 1)]


def reference(cache, names, counts, q):
    """The answer in 64 bits from what the cache holds, by sequence."""
    out, at = [], 0
    for name, n in zip(names, counts):
        k, v = (t.double() for t in cache.gather(name, torch.float16))
        m, qs = k.shape[0], q[at: at + n].double().unflatten(1, (cache.kv_heads, -1))
        s = torch.einsum("ikgd,jkd->ikgj", qs, k) * cache.head_dim ** -0.5
        hidden = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n)
        p = torch.softmax(s.masked_fill(hidden[:, None, None], float("-inf")), -1)
        out.append(torch.einsum("ikgj,jkd->ikgd", p, v).flatten(1, 2))
        at += n
    return torch.cat(out)


@pytest.mark.parametrize("heads,kv,dim,page,by_channel", [(8, 2, 128, 16, False), (4, 4, 64, 32, True)])
def test_serving_path_and_stored_sequences(heads, kv, dim, page, by_channel):
    from torch_ans_b200 import _C
    from torch_ans_b200.kv_cache import PagedKVCache4
    cache = PagedKVCache4(64, kv, dim, page_size=page)
    rot, lengths = rotation(2048, dim), {"a": 0, "b": 0}
    outs = {}
    rounds = [(["a", "b"], [301, 70])] + [(["b", "a"], [1, 1])] * 3 + [(["a"], [5])]
    for i, (names, counts) in enumerate(rounds):
        q, k, v = projection(sum(counts), heads, kv, dim, i)
        step = cache.reserve(names, counts)
        for n, c in zip(names, counts):
            lengths[n] += c
            assert cache.length(n) == lengths[n]
        q = cache.append(step, k, v, q=q, rotation=rot)
        out = cache.attend(step, q)
        # the gathered values are rounded to float16 (2^-11 of each) and the weights too; scores of about
        # dim / sqrt(dim) products of size 1 carry 2^-11 of their sum each
        ref = reference(cache, names, counts, q)
        top = max(float(cache.gather(n, torch.float16)[1].abs().max()) for n in names)
        size = float(q.double().abs().sum(-1).max()) * 8 * dim ** -0.5
        bound = top * (2.0 ** -10 + 2 * size * 2.0 ** -10) + ref.abs() * P.U[torch.bfloat16]
        assert ((out.double() - ref).abs() <= bound).all()
        outs = dict(step=step, q=q, out=out, names=names)
    raw = 2 * kv * lengths["a"] * (dim // 2 + 4)
    data = cache.store("a", by_channel=by_channel)
    assert _C.device_status() == 0
    if not by_channel:  # rounded bell-shaped rows have about 3.4 bits a code: smaller than what the pages hold
        assert len(data) < 2 * kv * -(-lengths["a"] // page) * page * (dim // 2 + 4)
    assert raw > 0
    ka, va = cache.gather("a")
    first = cache._pages["a"][0]
    cache.free("a")
    assert cache.length("a") == 0
    cache.load(cache_bytes := data, "c")
    assert cache._pages["c"][0] == first and cache.length("c") == lengths["a"]
    kc, vc = cache.gather("c")
    assert torch.equal(ka, kc) and torch.equal(va, vc)
    cache.load(cache_bytes, "d")  # and once more, in other pages
    kd, vd = cache.gather("d")
    assert torch.equal(ka, kd) and torch.equal(va, vd)
    i32 = dict(dtype=torch.int32, device="cuda")
    again = _C.kv4_attend(outs["q"], cache.codes, cache.params, torch.tensor([cache._pages["d"]], **i32),
                          torch.tensor([lengths["a"]], **i32), q_starts=torch.tensor([0, 5], **i32), max_queries=5)
    assert torch.equal(again, outs["out"])
    assert _C.device_status() == 0


def test_sequences_without_tokens_are_stored():
    from torch_ans_b200.kv_cache import PagedKVCache4
    cache = PagedKVCache4(5, 1, 64)
    cache.reserve([5], [0])
    cache.load(cache.store(5), 6)
    assert cache.length(6) == 0


def test_refusals():
    from torch_ans_b200.kv_cache import PagedKVCache4
    cache = PagedKVCache4(4, 1, 64)
    with pytest.raises(ValueError):
        cache.reserve([1, 1], [1, 1])
    with pytest.raises(ValueError):
        cache.reserve([1], [-1])
    with pytest.raises(KeyError):
        cache.store("nobody")
    step = cache.reserve([1], [20])
    _, k, v = projection(20, 1, 1, 64, 0)
    cache.append(step, k, v)
    data = cache.store(1)
    for bad in (b"", data[:20], b"XXXX" + data[4:], data[:200], data[:-9]):
        with pytest.raises((ValueError, RuntimeError)):
            cache.load(bad, 2)
    assert cache.length(2) == 0
    with pytest.raises(ValueError, match="in the cache"):
        cache.load(data, 1)
    with pytest.raises(ValueError, match="layout"):
        PagedKVCache4(4, 2, 64).load(data, 1)
    with pytest.raises(RuntimeError, match="free pages"):
        PagedKVCache4(1, 1, 64).load(data, 1)
    freqs = bytearray(data)
    freqs[28:30] = b"\x00\x00"
    with pytest.raises(ValueError, match="tables"):
        cache.load(bytes(freqs), 2)
