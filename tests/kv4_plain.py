"""The 4-bit key/value cache in 64 bits: the definitions that its kernels are tested against, written with plain torch
operations (any device), and caches to test with."""
import torch

TINY = 2.0 ** -100
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a unit in the last place, relative: 8 and 11 significant bits


def rounding(x, dtype):
    """What x (64 bits) loses when it is rounded to dtype; a value that is off by e before it is rounded ends within
    rounding(x) + 2 e of x, since the nearest to it is no further from it than the nearest to x."""
    return (x.to(dtype).double() - x).abs()


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def pack(c):
    c = c.to(torch.uint8).unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def rotate(x, positions, rotation, interleaved):
    """x [tokens, heads, dim] in 64 bits, turned to its positions."""
    r = rotation.shape[1]
    cos, sin = (t.double()[positions][:, None] for t in (rotation[:, : r // 2], rotation[:, r // 2:]))
    x = x.double().clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2: r])
    a2, b2 = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        x[..., 0:r:2], x[..., 1:r:2] = a2, b2
    else:
        x[..., : r // 2], x[..., r // 2: r] = a2, b2
    return x


def params_of(x):
    """(scale, offset) of rows x in 64 bits, each rounded to bfloat16 as it is stored."""
    offset = x.amin(-1).float().to(torch.bfloat16).double()
    scale = ((x.amax(-1) - offset) / 15).float().to(torch.bfloat16).double()
    return torch.where(scale < TINY, 0.0, scale), offset


def values(codes, params):
    """What the rows stand for; codes [..., dim / 2], params [..., 2]."""
    return unpack(codes).double() * params[..., :1].double() + params[..., 1:].double()


def attend(q, codes, params, pages, lengths, q_starts, scale, causal=True):
    """(out, lse, bound, score_bound) in 64 bits; lengths and q_starts are lists.  The bounds: see attend_bounds."""
    heads, dim, kv, page = q.shape[1], q.shape[2], codes.shape[2], codes.shape[3]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    score_bound = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for b, m in enumerate(lengths):
        lo, hi = q_starts[b], q_starts[b + 1]
        n = hi - lo
        if m == 0 or n == 0:
            continue
        ids = pages[b, : -(-m // page)].long()
        ok = (ids >= 0) & (ids < codes.shape[0])
        held = values(codes[ids.clamp(0, codes.shape[0] - 1)], params[ids.clamp(0, codes.shape[0] - 1)])
        held = held.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :m]  # [2, kv, m, dim]
        ok = ok.repeat_interleave(page)[:m]
        held = torch.where(ok[:, None], held, 0.0)
        qb = q[lo:hi].double().unflatten(1, (kv, heads // kv))
        s = torch.einsum("ikgd,kjd->ikgj", qb, held[0]) * scale
        seen = ok[None, :].expand(n, m)
        if causal:
            seen = seen & (torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n))
        s = s.masked_fill(~seen[:, None, None], float("-inf"))
        out[lo:hi] = torch.einsum("ikgj,kjd->ikgd", torch.nan_to_num(torch.softmax(s, -1)), held[1]).flatten(1, 2)
        lse[lo:hi] = torch.logsumexp(s, -1).flatten(1, 2)
        of_out, of_score = attend_bounds(qb, held, scale)
        bound[lo:hi], score_bound[lo:hi] = of_out.flatten(1, 2)[..., None], of_score.flatten(1, 2)
    return out, lse, bound, score_bound


def attend_bounds(qb, held, scale):
    """How far an output and a score may be from the 64-bit ones before the output's own rounding, for each query and head.

    A weight may carry half a unit of float16 (2^-11 relative at most) and a value too (2^-11 of the largest): 2^-10 of
    the largest value together.  A score may be off by the rounding of its factors to float16 (2^-11 of the sum of
    |q||k| that it adds up) and by the float sums and the hardware's 2^x (2^-18 of it, plus 2^-20); an error e of the
    scores changes the log of their sum by e, weights by a factor of at most exp(2 e), the result by about 2 e of the
    largest value."""
    top = held[1].abs().amax((1, 2))  # [kv]
    size = torch.einsum("ikgd,kd->ikg", qb.abs(), held[0].abs().amax(1)) * abs(scale)
    score = size * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -20
    return top[:, None] * (2.0 ** -10 + 2 * score), score


def pool(pages, kv, page, dim, seed=0, device="cuda"):
    """A cache of random rows of different sizes."""
    g = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(0, 256, (pages, 2, kv, page, dim // 2), dtype=torch.uint8, device=device, generator=g)
    scale = torch.exp(torch.randn(codes.shape[:-1], device=device, generator=g) * 0.4 - 1.5)
    offset = torch.randn(codes.shape[:-1], device=device, generator=g) * 0.5 - 7.5 * scale
    return codes, torch.stack([scale, offset], -1).to(torch.bfloat16)


def table(lengths, page, seed=0, extra=1, device="cuda"):
    """A page table over shuffled pages, -1 past each sequence's end; (pages, pool size)."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 1
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at: at + n] + [-1] * (max(need) + extra - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=device).reshape(len(lengths), max(need) + extra), total
