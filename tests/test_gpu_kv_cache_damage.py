"""Stored sequences that were damaged are refused before anything of the cache changes."""
import struct

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def stored():
    from torch_ans_b200 import _C
    from torch_ans_b200.kv_cache import PagedKVCache4
    _C.device_status()
    cache = PagedKVCache4(12, 2, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = [torch.randn(50, 2, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    cache.append(cache.reserve(["a"], [50]), k, v)
    yield cache, cache.store("a")
    assert _C.device_status() == 0


def refused(cache, data):
    codes, params = cache.codes.clone(), cache.params.clone()
    free = list(cache._free)
    with pytest.raises(ValueError):
        cache.load(data, "b")
    assert cache.length("b") == 0 and cache._free == free
    assert torch.equal(cache.codes, codes) and torch.equal(cache.params.view(torch.int16), params.view(torch.int16))


HEADER, TABLES, PARAMS = 28, 4 * 16 * 2, 4 * 2 * 2 * 16 * 4


@pytest.mark.parametrize("at", [4, 8, HEADER + 5, HEADER + TABLES, HEADER + TABLES + PARAMS - 1, HEADER + TABLES + PARAMS + 4,
                                HEADER + TABLES + PARAMS + 100, -300, -20, -5, -1])
@pytest.mark.parametrize("bit", [0, 6])
def test_one_bit_is_another(stored, at, bit):
    cache, data = stored
    bad = bytearray(data)
    bad[at] ^= 1 << bit
    refused(cache, bytes(bad))


def test_lengths_and_flags(stored):
    cache, data = stored
    refused(cache, data + b"\0")
    refused(cache, data[:24] + struct.pack("<I", 2) + data[28:])
    cache.reserve(["none"], [0])
    empty = cache.store("none")
    refused(cache, empty + b"\0")
    refused(cache, empty[:-1] + bytes([empty[-1] ^ 1]))


def test_strings_without_a_checksum(stored):
    """The first version of the format ended with the streams."""
    cache, data = stored
    old = b"KV4\x01" + data[4:-4]
    cache.load(old, "c")
    assert all(torch.equal(x, y) for x, y in zip(cache.gather("a"), cache.gather("c")))
    # its streams are cut to their last 8 bytes, which cannot hold 1,024 codes: the decoder says so
    body, at, cut = old[:HEADER + TABLES + PARAMS], HEADER + TABLES + PARAMS, b""
    for _ in range(16):
        n = struct.unpack_from("<I", old, at)[0]
        cut += struct.pack("<I", 8) + old[at + 4 + n - 8: at + 4 + n]
        at += 4 + n
    refused(cache, body + cut)
