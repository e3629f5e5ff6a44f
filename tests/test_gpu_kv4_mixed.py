"""Attention over rows of mixed sizes, with weights that all differ: the root mean square error of each query and head is within
what independent roundings may add up to.

A token's share of the error is at most p_j R_j (2^-11 for its weight and value together with the other's 2^-11 in quadrature, here 2^-11 and
2 e_j), with e_j = 2^-11 sqrt(sum q^2 k^2), what the roundings of a key add up to, and 2^-19 sum |q||k| for the float sums; the shares
are independent.  Three times that, 2^-15 of sum p_j R_j for what is not independent, and the output's own rounding."""
import pytest
import torch

from tests import kv4_plain as P

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def check(q, codes, params, pages, lengths, counts, causal, hint):
    from torch_ans_b200 import _C
    _C.device_status()
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
    kv, page, dim = codes.shape[2], codes.shape[3], q.shape[2]
    got = _C.kv4_attend(q, codes, params, pages, torch.tensor(lengths, **i32), q_starts=torch.tensor(starts, **i32), max_queries=hint,
                        causal=causal)
    assert _C.device_status() == 0
    for b, m in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        if m == 0 or lo == hi:
            continue
        ids = pages[b, : -(-m // page)].long()
        held = P.values(codes[ids], params[ids]).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :m]
        step = params[ids, 1, :, :, 0].double().permute(1, 0, 2).flatten(1)[:, :m].abs()
        size = torch.maximum(held[1].abs().amax(-1), 7.5 * step)[:, None]
        qb, scale = q[lo:hi].double().unflatten(1, (kv, -1)), dim ** -0.5
        s = torch.einsum("ikgd,kjd->ikgj", qb, held[0]) * scale
        e = scale * (2.0 ** -11 * torch.einsum("ikgd,kjd->ikgj", qb ** 2, held[0] ** 2).sqrt() +
                     2.0 ** -19 * torch.einsum("ikgd,kjd->ikgj", qb.abs(), held[0].abs()))
        t = torch.arange(m, device="cuda")
        seen = t <= torch.arange(hi - lo, device="cuda")[:, None] + (m - hi + lo) if causal else torch.ones(hi - lo, m, dtype=torch.bool, device="cuda")
        p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen[:, None, None], float("-inf")), -1))
        out = torch.einsum("ikgj,kjd->ikgd", p, held[1])
        bound = 3 * (p * size * (2.0 ** -11 + 2 * e)).square().sum(-1).sqrt() + (p * size).sum(-1) * 2.0 ** -15
        bound = bound + out.square().mean(-1).sqrt() * P.U[q.dtype] + (2.0 ** -24 if q.dtype == FP else 0.0)
        err = (got[lo:hi].double().unflatten(1, (kv, -1)) - out).square().mean(-1).sqrt()
        assert (err <= bound).all(), (b, float((err / bound).max()), int((err > bound).sum()), err.numel())


@pytest.mark.parametrize("values,keys", [(0.0, 0.0), (1.0, 0.0), (1.0, 0.5), (1.5, 1.0), (3.0, 0.5), (8.0, 0.5)])
@pytest.mark.parametrize("dim,dtype", [(64, FP), (128, BF), (128, FP), (256, BF), (256, FP)])
@pytest.mark.parametrize("counts,causal", [([1, 1, 1], True), ([6, 3, 8], True), ([400, 90, 64], True), ([300, 100, 64], False)])
def test_rows_of_mixed_sizes(counts, causal, dim, dtype, values, keys):
    """Sizes of values and keys are 2^N(0, .) from token to token (cut at three deviations)."""
    if dtype == FP and values > 1.5:
        values = 1.5
    lengths = [1500, 333, 64]
    pages, total = P.table(lengths, 16, 3)
    codes, params = P.pool(total, 2, 16, dim, 5)
    g = torch.Generator(device="cuda").manual_seed(dim)
    f = torch.randn(params.shape[:-1], device="cuda", generator=g).clamp(-3, 3)
    params = (params.float() * torch.exp2(f * torch.tensor([keys, values], device="cuda")[None, :, None, None])[..., None]).to(BF)
    q = torch.randn(sum(counts), 8, dim, device="cuda", generator=g).to(dtype)
    check(q, codes, params, pages, lengths, counts, causal, max(counts))
