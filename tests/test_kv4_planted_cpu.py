"""The planted caches themselves: a plain 32-bit evaluation is within their bound, and answers with a fault that a kernel could
have are not."""
import pytest
import torch

from tests.kv4_planted import Planted

BF, FP = torch.bfloat16, torch.float16


def plain(c, q, counts, dtype, drop=(), half_products=False):
    """The attention in 32 bits.  half_products: weights times value scales in one float16 each, under the largest scale of all."""
    from tests import kv4_plain as P
    out, lo, group = torch.zeros(q.shape), 0, q.shape[1] // c.kv
    for b, (n, m) in enumerate(zip(counts, c.lengths)):
        ids = c.pages[b, : -(-m // c.page)].long()
        held = P.values(c.codes[ids], c.params[ids]).float().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :m]
        s = torch.einsum("ikgd,kjd->ikgj", q[lo: lo + n].float().unflatten(1, (c.kv, group)), held[0]) * c.dim ** -0.5
        t = torch.arange(m)
        seen = t <= torch.arange(n)[:, None] + (m - n)
        for d in drop:
            seen = seen & (t != d)
        p = torch.softmax(s.masked_fill(~seen[:, None, None], float("-inf")), -1)
        if half_products:
            top = held[1].abs().amax()
            out[lo: lo + n] = ((p[..., None] * (held[1] / top)[:, None]).half().float().sum(-2) * top).flatten(1, 2)
        else:
            out[lo: lo + n] = torch.einsum("ikgj,kjd->ikgd", p, held[1]).flatten(1, 2)
        lo += n
    return out.to(dtype)


@pytest.mark.parametrize("dim,dtype,lengths,counts", [(64, BF, [3000], [3]), (128, FP, [700, 129], [40, 129]), (256, BF, [40000], [1])])
def test_bound_holds_and_rejects(dim, dtype, lengths, counts):
    c = Planted(lengths, 16, 1, dim, 64, device="cpu")
    q, wanted = c.queries(counts, 2, dtype)
    out, bound = c.answers(q, wanted, counts)
    got = plain(c, q, counts, dtype)
    assert not c.wrong(got, out, bound).any()
    zeros = c.wrong(torch.zeros_like(got), out, bound)
    assert zeros.float().mean() > 0.95 and zeros.any(-1).all()
    assert (out.square().mean().sqrt() > 30 * bound.mean())  # the bound is small beside the answers
    # the second head wants the second block of its first query: without these 128 tokens that answer is another
    lost = plain(c, q, counts, dtype, drop=range(64, 192))
    assert c.wrong(lost, out, bound)[0, 1].float().mean() > 0.9


def test_bound_rejects_products_under_a_large_value_that_does_not_count():
    for exponent, found in ((0, False), (20, True), (60, True)):
        c = Planted([300], 16, 1, 64, 32, device="cpu")
        c.unlikely(0, [290])
        c.resize(0, [290], 1, exponent)
        q, wanted = c.queries([2], 2, BF, beta=26.0)
        out, bound = c.answers(q, wanted, [2])
        assert not c.wrong(plain(c, q, [2], BF), out, bound).any()
        assert bool(c.wrong(plain(c, q, [2], BF, half_products=True), out, bound).any()) == found
