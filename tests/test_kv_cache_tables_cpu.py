"""The frequency tables of stored sequences, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("seed", range(5))
def test_tables_sum_to_the_precision_and_hold_every_code(seed):
    from torch_ans_b200.kv_cache import _cdfs, _frequencies
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, 1 << 40, (6, 16), generator=g) >> torch.randint(0, 40, (6, 16), generator=g)
    counts[0] = 0
    counts[0, seed] = 1  # one code only
    counts[1] = 7
    counts[2, 3] += 1 << 33
    freqs = _frequencies(counts)
    assert freqs.min() >= 1 and freqs.sum(1).eq(1 << 16).all() and freqs[0, seed] == (1 << 16) - 15
    # no symbol loses more than the 16 that go to the least ones and one by rounding, or gains more than what is left over
    exact = counts.double() / counts.sum(1, keepdim=True) * (1 << 16)
    assert ((freqs.double() - exact).abs() <= 16).all()
    cdfs = _cdfs(freqs)
    assert cdfs.dtype == torch.int32 and cdfs.shape == (6, 17) and cdfs[:, 0].eq(0).all() and cdfs[:, -1].eq(1 << 16).all()
    assert torch.equal(cdfs.diff(dim=1).long(), freqs)
