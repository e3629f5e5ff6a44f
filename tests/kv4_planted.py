"""Caches whose answers are known to come from known tokens, and how far an answer may be from the 64-bit one.

The keys of a block of tokens are one pattern of -k and +k, another for each block; a query is the pattern of one block
(`wanted`), so its softmax lies on that block's tokens, all with the same score, but for about e^-20.  The values of a block
are about the same, those of different blocks are not.  An answer is then as large as the values, it is wrong altogether when
the block's tokens are lost, and the bound below is small beside it, whatever the length.

The first ANCHOR channels of ordinary keys are +k and of a query `beta`: a token with -k there (`unlikely`) has a score far
below all others, for every query.

The bound of an answer, before its own rounding.  R_j is the size of a token's values: the largest of them or 7.5 scales, if
that is more.
  * weight and value may each be rounded to float16: (2^-11 + 2^-11) sum p_j R_j, and 2^-16 of it for the float sums.  In a
    block the scores are the same number by the same arithmetic, so their errors cancel against the softmax's sum.
  * the tokens outside the block: their scores may be off by e (2^-11 of sum |q||k|, as in kv4_plain.attend_bounds), so their
    weights by a factor of expm1(2 e), and the sum by as much of their share.
  * a weight under float16's normal numbers carries an absolute error, 2^-25 of the largest product of a weight and a size that
    the query sees: 2^-24 for each token that it sees."""
import torch

from tests import kv4_plain as P

ANCHOR = 16
K = 0.9375  # 7.5 / 8
ALPHA = {64: 8.0, 128: 4.0, 256: 2.0}  # scores of the block at least 20 above the others (in e's), up to 1,000 blocks


class Planted:
    """A cache for `lengths`: codes, params, pages; `pattern` [sequences][kv, blocks, dim] of -1 and 1."""

    def __init__(self, lengths, page, kv, dim, block, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.kv, self.dim, self.block, self.device = lengths, page, kv, dim, block, device
        pages, total = P.table(lengths, page, seed, device="cpu")
        codes, params = torch.zeros(total, 2, kv, page, dim // 2, dtype=torch.uint8), torch.zeros(total, 2, kv, page, 2)
        self.pattern = []
        for b, n in enumerate(lengths):
            blocks = -(-n // block)
            u = torch.randint(0, 2, (kv, blocks, dim), generator=g) * 2 - 1
            u[..., :ANCHOR] = 1
            self.pattern.append(u.to(device))
            if n == 0:
                continue
            t = torch.arange(n)
            at = pages[b, t // page].long(), t % page
            kc = ((u[:, t // block] + 1) // 2 * 15)  # [kv, n, dim]
            base = torch.randint(2, 14, (kv, blocks, dim), generator=g)[:, t // block]
            vc = base + torch.randint(-2, 3, base.shape, generator=g)
            codes[at[0], :, :, at[1]] = torch.stack([P.pack(kc), P.pack(vc)]).permute(2, 0, 1, 3)
            vs = torch.rand(kv, n, generator=g) * 0.25 + 0.25
            vo = -7.5 * vs + torch.randn(kv, n, generator=g) * 0.3
            kp = torch.tensor([2 * K / 15, -K]).expand(kv, n, 2)
            params[at[0], :, :, at[1]] = torch.stack([kp, torch.stack([vs, vo], -1)]).permute(2, 0, 1, 3)
        self.codes, self.params, self.pages = codes.to(device), params.to(torch.bfloat16).to(device), pages.to(device)

    def place(self, b, t):
        return int(self.pages[b, t // self.page]), t % self.page

    def resize(self, b, tokens, side, exponent):
        """Rows of these tokens times 2^exponent."""
        for t in tokens:
            p, i = self.place(b, t)
            self.params[p, side, :, i] = (self.params[p, side, :, i].double() * 2.0 ** exponent).to(torch.bfloat16)

    def unlikely(self, b, tokens):
        for t in tokens:
            p, i = self.place(b, t)
            self.codes[p, 0, :, i, : ANCHOR // 2] = 0

    def queries(self, counts, group, dtype, seed=0, beta=0.0, size=1.0, causal=True, first=0):
        """Queries of each sequence, heads kv * group; (q, wanted [queries, heads]).  Every block that a query sees is
        wanted in turn, from number `first`."""
        q, wanted, turn = [], [], first
        for b, (n, m) in enumerate(zip(counts, self.lengths)):
            for i in range(n):
                sees = m - n + i + 1 if causal else m
                blocks = max(1, -(-sees // self.block))
                w = (turn + torch.arange(self.kv * group)) % blocks
                turn += self.kv * group
                row = torch.zeros(self.kv, group, self.dim, device=self.device)
                if m > 0:
                    row = self.pattern[b][torch.arange(self.kv).repeat_interleave(group), w].float().view(self.kv, group, self.dim)
                    row = row * ALPHA[self.dim]
                    row[..., :ANCHOR] = beta
                q.append((row * size).flatten(0, 1))
                wanted.append(w)
        return torch.stack(q).to(dtype).to(self.device), torch.stack(wanted).to(self.device)

    def answers(self, q, wanted, counts, causal=True, drop=()):
        """(out, bound) in 64 bits; tokens in `drop` are left out (a mistake to be found)."""
        out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
        scale, group, lo = self.dim ** -0.5, q.shape[1] // self.kv, 0
        for b, (n, m) in enumerate(zip(counts, self.lengths)):
            hi = lo + n
            if n and m:
                ids = self.pages[b, : -(-m // self.page)].long()
                held = P.values(self.codes[ids], self.params[ids]).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :m]
                step = self.params[ids, 1, :, :, 0].double().permute(1, 0, 2).flatten(1)[:, :m].abs()
                size = torch.maximum(held[1].abs().amax(-1), 7.5 * step)  # [kv, m]
                qb = q[lo:hi].double().unflatten(1, (self.kv, group))
                s = torch.einsum("ikgd,kjd->ikgj", qb, held[0]) * scale
                e = torch.einsum("ikgd,kjd->ikgj", qb.abs(), held[0].abs()) * scale * 2.0 ** -11
                t = torch.arange(m, device=q.device)
                seen = (t <= torch.arange(n, device=q.device)[:, None] + (m - n)) if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
                for d in drop:
                    seen = seen & (t != d)
                p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen[:, None, None], float("-inf")), -1))
                product = p * size[:, None]
                outside = (t // self.block != wanted[lo:hi, :, None]).unflatten(1, (self.kv, group))
                off = torch.expm1(2 * e.clamp(max=300)) * outside
                of = (product * (2.0 ** -10 + 2.0 ** -16 + off)).nan_to_num(0).sum(-1) + (p * off).nan_to_num(0).sum(-1) * product.sum(-1)
                of = of + seen.sum(-1)[:, None, None] * 2.0 ** -24 * product.amax(-1)
                out[lo:hi] = torch.einsum("ikgj,kjd->ikgd", p, held[1]).flatten(1, 2)
                bound[lo:hi] = of.flatten(1, 2)
            lo = hi
        return out, bound

    def wrong(self, got, out, bound):
        """The elements of `got` that are further from `out` than they may be."""
        least = 2.0 ** -24 if got.dtype == torch.float16 else 0.0  # float16's smallest step
        return ~((got.double() - out).abs() <= bound[..., None] * 1.01 + out.abs() * P.U[got.dtype] * 1.01 + least)

    def attend(self, C, q, counts, causal=True, max_queries=None):
        starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
        i32 = dict(dtype=torch.int32, device=q.device)
        return C.kv4_attend(q, self.codes, self.params, self.pages, torch.tensor(self.lengths, **i32),
                            q_starts=torch.tensor(starts, **i32), max_queries=max(counts) if max_queries is None else max_queries,
                            causal=causal)

    def check(self, C, counts, group, dtype, beta=0.0, size=1.0, causal=True, first=0):
        """The op's answers are within the bound, and the bound is small beside them."""
        q, wanted = self.queries(counts, group, dtype, beta=beta, size=size, causal=causal, first=first)
        out, bound = self.answers(q, wanted, counts, causal)
        got = self.attend(C, q, counts, causal)
        assert C.device_status() == 0
        assert out.square().mean().sqrt() > 30 * bound.mean()
        bad = self.wrong(got, out, bound)
        assert not bad.any(), (int(bad.sum()), bad.numel(), float((got.double() - out).square().mean().sqrt() / out.square().mean().sqrt()))
        return got
