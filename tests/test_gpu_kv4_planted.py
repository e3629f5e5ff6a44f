"""Attention over the 4-bit cache where each answer depends on a known block of tokens (tests/kv4_planted.py has the bound): a
part lost in a join, values of other tokens or a wrong rescale are far outside it at any length."""
import pytest
import torch

from tests.kv4_planted import Planted

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def C():
    from torch_ans_b200 import _C
    _C.set_sync_check(False)
    _C.device_status()
    return _C


@pytest.mark.parametrize("dim,dtype,kv,group,page,block", [(64, FP, 1, 8, 16, 32), (128, BF, 2, 4, 64, 64), (256, BF, 1, 2, 32, 128),
                                                           (128, FP, 1, 16, 48, 32), (64, BF, 2, 40, 16, 32)])
def test_every_block_of_a_long_context(C, dim, dtype, kv, group, page, block):
    """One token after another, until each block of the context was asked for."""
    c = Planted([20011 if dim < 256 else 9001], page, kv, dim, block, seed=dim)
    blocks = -(-c.lengths[0] // block)
    for first in range(0, blocks, kv * group):
        c.check(C, [1], group, dtype, first=first)


@pytest.mark.parametrize("dim,dtype,kv,group,counts", [(64, BF, 8, 1, 5), (128, FP, 2, 4, 3), (256, BF, 1, 3, 2), (128, BF, 1, 8, 8)])
def test_ragged_drafts(C, dim, dtype, kv, group, counts):
    lengths = [0, 1, 33, 2049, 7, 700, 128, 129, 4000, 64, 31]
    c = Planted(lengths, 16, kv, dim, 32, seed=1)
    for first in (0, 60):
        c.check(C, [counts if n else 0 for n in lengths], group, dtype, first=first)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,dtype,kv,group", [(64, FP, 4, 4), (128, BF, 2, 4), (256, FP, 1, 3)])
def test_prompts_and_chunks(C, dim, dtype, kv, group, causal):
    lengths = [700, 1, 0, 129, 300, 64]
    c = Planted(lengths, 16, kv, dim, 32, seed=2)
    c.check(C, lengths, group, dtype, causal=causal)
    c.check(C, [333, 1, 0, 100, 20, 64], group, dtype, causal=causal, first=5)


@pytest.mark.parametrize("dim,dtype,group,count,length", [(128, BF, 4, 200, 20000), (64, FP, 4, 129, 9001), (256, BF, 1, 130, 5000),
                                                          (64, BF, 32, 9, 12345)])
def test_every_block_before_a_chunk(C, dim, dtype, group, count, length):
    c = Planted([length], 64, 1, dim, 64, seed=3)
    c.check(C, [count], group, dtype)


@pytest.mark.parametrize("sequences", [129, 200, 295])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_sequences_than_threads_with_blocks_of_their_own(C, sequences, dim):
    """One key/value head and more sequences than a block has threads, still fewer items than half the blocks."""
    g = torch.Generator().manual_seed(sequences)
    lengths = torch.randint(0, 900, (sequences,), generator=g).tolist()
    lengths[5], lengths[sequences - 2] = 5000, 0
    c = Planted(lengths, 16, 1, dim, 64, seed=4)
    c.check(C, [1] * sequences, 8, BF)


@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, FP), (256, BF)])
def test_many_short_sequences_with_many_rows(C, dim, dtype):
    """Hundreds of sequences in the kernel for many rows: more row tiles than SMs, found beyond the first 32 sequences."""
    g = torch.Generator().manual_seed(7)
    lengths = torch.randint(1, 200, (300,), generator=g).tolist()
    counts = [min(n, 1 + i % 20) if i % 7 else 0 for i, n in enumerate(lengths)]
    c = Planted(lengths, 16, 2, dim, 32, seed=5)
    c.check(C, counts, 4, dtype)


@pytest.mark.parametrize("lengths,counts", [([3000, 11, 700, 5000], [1, 1, 1, 1]), ([4097, 900], [300, 64])])
def test_results_repeat(C, lengths, counts):
    c = Planted(lengths, 16, 2, 128, 64, seed=6)
    first = c.check(C, counts, 4, BF)
    for _ in range(3):
        assert torch.equal(c.check(C, counts, 4, BF), first)
