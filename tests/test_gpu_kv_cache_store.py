"""What a stored sequence's bytes hold: the sequence, and nothing of what its pages held before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def status():
    from torch_ans_b200 import _C
    _C.device_status()
    yield
    assert _C.device_status() == 0


def rows(n, kv, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, kv, dim, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]


@pytest.mark.parametrize("by_channel", [False, True])
@pytest.mark.parametrize("ordinary", [0, 1, 13, 24, 31])
def test_codes_that_are_nearly_all_the_same(ordinary, by_channel):
    """Rows without range (zeros, as a padded value has them) have one code: it may be most of a table or all of it."""
    from torch_ans_b200.kv_cache import PagedKVCache4
    cache = PagedKVCache4(9, 2, 64)
    k, v = rows(48, 2, 64, 3)
    k[ordinary:], v[: 48 - ordinary] = 0.0, 3.0
    cache.append(cache.reserve(["a"], [48]), k, v)
    held, codes = cache.gather("a"), cache.codes[cache._pages["a"]].clone()
    for name in ("b", "c"):
        cache.load(cache.store("a", by_channel=by_channel), name)
        assert torch.equal(cache.codes[cache._pages[name]], codes)
        assert all(torch.equal(x, y) for x, y in zip(held, cache.gather(name)))
        cache.free(name)


@pytest.mark.parametrize("by_channel", [False, True])
@pytest.mark.parametrize("kv,dim,page,tokens", [(2, 128, 16, 37), (1, 64, 64, 1), (3, 256, 32, 64), (2, 64, 48, 95)])
def test_bytes_do_not_depend_on_what_the_pages_held(kv, dim, page, tokens, by_channel):
    from torch_ans_b200.kv_cache import PagedKVCache4
    k, v = rows(tokens, kv, dim, 1)
    stored = []
    for before in ("zeros", "another sequence", "anything"):
        cache = PagedKVCache4(8, kv, dim, page_size=page)
        if before == "zeros":
            cache.codes.zero_()
            cache.params.zero_()
        elif before == "anything":
            cache.codes.fill_(0xa7)
            cache.params.fill_(float("nan"))
        else:
            step = cache.reserve(["other"], [8 * page])
            cache.append(step, *rows(8 * page, kv, dim, 2))
            cache.free("other")
        cache.append(cache.reserve(["a"], [tokens]), k, v)
        stored.append(cache.store("a", by_channel=by_channel))
        held = cache.gather("a")
        cache.load(stored[-1], "b")
        assert all(torch.equal(x, y) for x, y in zip(held, cache.gather("b")))
    assert stored[0] == stored[1] == stored[2]
