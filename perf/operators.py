"""The 4-bit key/value cache operators, as cases to measure: appending to a paged cache with the position rotation, attention
over the cache, and the cache's pages as symbols of the entropy coder (and back).

The cache of one layer is two tensors that the caller owns:
  codes   uint8    [pages, 2, kv_heads, page_size, head_dim / 2]   4-bit codes, the even channel in the low half of a byte;
                                                                   [:, 0] keys, [:, 1] values
  params  bfloat16 [pages, 2, kv_heads, page_size, 2]              (scale, offset) of each token's head
A code c stands for c * scale + offset. A row x is stored with offset = bf16(min x), scale = bf16((max x - offset) / 15), and
c = round((x - offset) / scale) clamped to 0..15; a scale under 2^-100 is stored as 0, a row that is not finite as NaN.

`run` with `own` false is the plain form: elementary torch operations in 32 bits, rounded once at the end.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TINY = 2.0 ** -100


def listed():
    return [
        # one sequence generates: the new token's projection goes into the cache. Latency is all there is.
        dict(name="append_one", op="append", tokens=1, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, page=16, padding=0, dtype="bf16"),
        # a decode step of a batch, padded to a fixed size for graph replay (slots of -1), neighbouring channels rotated together
        dict(name="append_batch", op="append", tokens=61, heads=12, kv_heads=4, dim=64, rotary=32, interleaved=True, page=32, padding=5, dtype="fp16"),
        # packed prompts enter the cache: bound by memory
        dict(name="append_prompts", op="append", tokens=16381, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, page=16, padding=0, dtype="bf16"),
        # one sequence generates over a short context: the smallest call
        dict(name="attend_one", op="attend", batch=1, queries=1, least=777, most=777, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a serving batch of very different context lengths, one of them empty
        dict(name="attend_batch", op="attend", batch=48, queries=1, least=0, most=16384, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a few very long contexts, eight query heads to a key head: few rows, a long axis
        dict(name="attend_long", op="attend", batch=3, queries=1, least=100003, most=131071, heads=16, kv_heads=2, dim=128, page=64, dtype="fp16"),
        # drafted tokens are verified: five queries a sequence, no shared heads
        dict(name="attend_drafts", op="attend", batch=29, queries=5, least=3, most=5000, heads=8, kv_heads=8, dim=64, page=32, dtype="bf16"),
        # packed prompts of different lengths attend to themselves
        dict(name="attend_prompts", op="attend", batch=4, queries=0, least=1100, most=3500, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a chunk of a long prompt attends to everything before it
        dict(name="attend_chunk", op="attend", batch=1, queries=511, least=32749, most=32749, heads=16, kv_heads=4, dim=64, page=128, dtype="fp16"),
        # a few pages leave for the entropy coder, one stream for each page, side and head
        dict(name="symbols_few", op="to_symbols", pages=3, kv_heads=8, dim=128, page=16, by_channel=False),
        # a long prefix leaves, with a table for each channel
        dict(name="symbols_many", op="to_symbols", pages=509, kv_heads=8, dim=128, page=64, by_channel=True),
        # decoded symbols come back into pages
        dict(name="symbols_back", op="from_symbols", pages=509, kv_heads=8, dim=128, page=64, by_channel=True),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([16, 32, 48, 64, 128])
    op = rng.choice(["append", "attend", "attend", "attend", "to_symbols", "from_symbols"])
    if op == "append":
        tokens = _between(rng, 1, max(2, (16381 * 48 * 128) // (dim * kv * (group + 2))))
        tokens = min(tokens, 65537)
        return dict(op=op, tokens=tokens, heads=kv * group, kv_heads=kv, dim=dim, rotary=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.5, page=page,
                    padding=rng.choice([0, tokens // 7]), dtype=dtype)
    if op in ("to_symbols", "from_symbols"):
        pages = _between(rng, 1, max(2, 60_000_000 // (2 * kv * page * dim)))
        return dict(op=op, pages=pages, kv_heads=kv, dim=dim, page=page, by_channel=rng.random() < 0.5)
    kind = rng.choice(["step", "drafts", "prompts", "chunk"])
    if kind in ("step", "drafts"):
        batch = _between(rng, 1, 96)
        queries = 1 if kind == "step" else rng.randint(2, 8)
        most = _between(rng, 16, max(17, min(131071, 250_000_000 // (batch * kv * dim * max(1, group * queries // 8)))))
        return dict(op=op, batch=batch, queries=queries, least=rng.choice([0, most // 3, most]), most=most, heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype)
    if kind == "prompts":
        batch = rng.randint(1, 5)
        most = _between(rng, 40, max(41, int(math.sqrt(1_400_000_000 / (batch * kv * group)))))
        most = min(most, 6000)
        return dict(op=op, batch=batch, queries=0, least=rng.choice([1, most // 2, most]), most=most, heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype)
    queries = _between(rng, 9, 1500)
    most = _between(rng, queries, max(queries + 1, min(40000, 1_400_000_000 // (queries * kv * group))))
    return dict(op=op, batch=1, queries=queries, least=most, most=most, heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype)


def _lengths(case):
    """Context lengths, on the host: spread over their logarithm, the longest among them; least=0 is a spread over a factor of 64 with one length of 0."""
    r = random.Random(case["batch"] * 1000003 + case["most"])
    lo, hi = case["least"] or max(1, case["most"] // 64), case["most"]
    n = [_between(r, lo, hi) for _ in range(case["batch"])]
    n[0] = hi
    if case["least"] == 0 and case["batch"] > 1:
        n[-1] = 0
    return n


def _queries(case):
    """Queries of each sequence: a whole prompt's (queries=0), or the same number for each."""
    return _lengths(case) if case["queries"] == 0 else [case["queries"]] * case["batch"]


def _pool(pages, case, gen):
    """A cache whose codes are spread as those of bell-shaped rows are, with rows of different sizes."""
    shape = (pages, 2, case["kv_heads"], case["page"], case["dim"] // 2)
    a, b = (torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=gen) for _ in range(2))
    lo = ((a & 15) + (b & 15)) >> 1
    codes = (((a >> 4) + (b >> 4)) >> 1).bitwise_left_shift_(4).bitwise_or_(lo)
    scale = torch.exp(torch.randn(shape[:-1], device="cuda", generator=gen) * 0.3 - 1.2)
    offset = torch.randn(shape[:-1], device="cuda", generator=gen) * 0.4 - 7.5 * scale
    return codes, torch.stack([scale, offset], -1).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] in ("to_symbols", "from_symbols"):
        total = case["pages"] + 7
        s["codes"], s["params"] = _pool(total, case, gen)
        s["pages"] = torch.randperm(total, device="cuda", generator=gen)[: case["pages"]]
        if case["op"] == "from_symbols":
            s["symbols"] = _symbols_plain(s["codes"], s["pages"].flip(0))
        return s
    heads, kv, dim, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        n = case["tokens"]
        # the projection's output holds queries, keys and values beside each other; some channels of the keys are much larger
        x = torch.randn(n, (heads + 2 * kv) * dim, device="cuda", generator=gen)
        size = torch.exp(torch.randn((heads + 2 * kv) * dim, device="cuda", generator=gen) * 0.6)
        x = (x * size).to(dtype)
        s["q"] = x[:, : heads * dim].view(n, heads, dim)
        s["k"] = x[:, heads * dim : (heads + kv) * dim].view(n, kv, dim)
        s["v"] = x[:, (heads + kv) * dim :].view(n, kv, dim)
        # page 0 is nobody's; the tokens of a sequence follow each other inside a page
        total = -(-n // page) + 9
        order = 1 + torch.randperm(total - 1, device="cuda", generator=gen)
        at = torch.arange(n, device="cuda") + 3
        s["slots"] = order[at // page] * page + at % page
        if case["padding"]:
            s["slots"][n - case["padding"] :] = -1
        s["positions"] = (torch.arange(n, device="cuda") + int(torch.randint(0, 999, (1,), device="cuda", generator=gen))) % 32768
        angle = torch.arange(32768, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda") / case["rotary"])
        s["rotation"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["codes"] = torch.zeros(total, 2, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
        s["params"] = torch.zeros(total, 2, kv, page, 2, dtype=torch.bfloat16, device="cuda")
        return s
    lengths, queries = _lengths(case), _queries(case)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 1
    s["codes"], s["params"] = _pool(total, case, gen)
    order = torch.randperm(total, device="cuda", generator=gen)
    width = max(need) + 1
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    col = torch.arange(width, device="cuda")
    used = col < torch.tensor(need, device="cuda")[:, None]
    s["pages"] = torch.where(used, order[(first[:, None] + col).clamp(max=total - 1)], -1).to(torch.int32)
    # what a last page holds after the sequence's end is whatever was in that memory
    at = s["lengths"][:, None] + torch.arange(page, device="cuda")
    tail = (at % page >= s["lengths"][:, None] % page) & (s["lengths"][:, None] % page > 0)
    slot = torch.where(tail, s["pages"].gather(1, (at // page).clamp(max=width - 1).long()), order[-1].int()).long()
    s["params"][slot, :, :, at % page] = float("nan")
    s["q_starts"] = torch.tensor([sum(queries[:b]) for b in range(len(queries) + 1)], dtype=torch.int32, device="cuda")
    s["max_queries"] = max(queries)
    s["q"] = torch.randn(sum(queries), heads, dim, device="cuda", generator=gen).to(dtype)
    s["scale"] = dim ** -0.5
    return s


def _unpack(codes):
    """[..., n] bytes to [..., 2 n] codes."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _pack(c):
    c = c.to(torch.uint8).unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def _values(codes, params):
    return _unpack(codes).float() * params[..., :1].float() + params[..., 1:].float()


def _quantised(x):
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    offset = lo.to(torch.bfloat16).float()
    scale = ((hi - offset) / 15).to(torch.bfloat16).float()
    scale = torch.where(scale < TINY, torch.zeros_like(scale), scale)
    finite = torch.isfinite(scale) & torch.isfinite(offset)
    c = ((x - offset) / scale).round().clamp(0, 15)
    c = torch.where(finite & (scale > 0), c, torch.zeros_like(c))
    params = torch.where(finite, torch.cat([scale, offset], -1), torch.full_like(scale, float("nan")))
    return _pack(c), params.to(torch.bfloat16)


def _rotated(x, table, rotary, interleaved):
    """[n, heads, dim] in 32 bits; table [n, rotary]: cosines, then sines."""
    cos, sin = table[:, None, : rotary // 2], table[:, None, rotary // 2 :]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : rotary // 2], x[..., rotary // 2 : rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _append_plain(s):
    case = s["case"]
    table = s["rotation"][s["positions"]]
    q = _rotated(s["q"].float(), table, case["rotary"], case["interleaved"])
    k = _rotated(s["k"].float(), table, case["rotary"], case["interleaved"])
    slot = s["slots"].clamp(min=0)  # page 0 takes what is not to be kept
    page, at = slot // case["page"], slot % case["page"]
    c, p = _quantised(torch.stack([k, s["v"].float()], 1))
    s["codes"][page, :, :, at] = c
    s["params"][page, :, :, at] = p
    held = _values(s["codes"][page, :, :, at], s["params"][page, :, :, at])
    held = torch.where((s["slots"] >= 0)[:, None, None, None], held, torch.zeros_like(held)).to(s["k"].dtype)
    return {"q": q.to(s["q"].dtype), "k": held[:, 0], "v": held[:, 1]}


def _attend_plain(s):
    case = s["case"]
    batch, kv, dim, group, most = case["batch"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"], s["max_queries"]
    pages = s["pages"].clamp(min=0).long()
    held = _values(s["codes"][pages], s["params"][pages])  # [batch, pages, 2, kv, page, dim]
    held = held.permute(0, 2, 3, 1, 4, 5).flatten(3, 4)  # [batch, 2, kv, tokens, dim]
    col = torch.arange(held.shape[3], device="cuda")
    there = col < s["lengths"][:, None]
    held = torch.where(there[:, None, None, :, None], held, torch.zeros_like(held[:1, :1, :1, :1, :1]))
    row = torch.arange(most, device="cuda")
    count = s["q_starts"][1:] - s["q_starts"][:-1]
    asked = row < count[:, None]
    at = torch.where(asked, s["q_starts"][:-1, None] + row, s["q"].shape[0])  # one row more takes what is not asked
    q = torch.cat([s["q"], torch.zeros_like(s["q"][:1])]).float()[at]  # [batch, most, heads, dim]
    q = q.unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, kv, group * most, dim]
    score = (q @ held[:, 0].transpose(-1, -2) * s["scale"]).unflatten(2, (group, most))
    last = s["lengths"][:, None] - count[:, None] + row  # the position of each query: it sees itself and what is before
    seen = (col <= last[:, :, None]) & there[:, None, :]
    score = torch.where(seen[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ held[:, 1]).unflatten(2, (group, most)) / torch.where(total > 0, total, torch.ones_like(total))
    full = torch.empty(s["q"].shape[0] + 1, case["heads"], dim, dtype=s["q"].dtype, device="cuda")
    full[at.flatten()] = out.permute(0, 3, 1, 2, 4).reshape(batch * most, case["heads"], dim).to(full.dtype)
    return full[:-1]


def _symbols_plain(codes, pages):
    return _unpack(codes[pages]).flatten(3).flatten(0, 2).int()


def _to_symbols_plain(s):
    case = s["case"]
    symbols = _symbols_plain(s["codes"], s["pages"])
    side = torch.arange(2 * case["kv_heads"], device="cuda", dtype=torch.int32)
    table = side[:, None, None]
    if case["by_channel"]:
        table = table * case["dim"] + torch.arange(case["dim"], device="cuda", dtype=torch.int32)
    return symbols, table.expand(2 * case["kv_heads"], case["page"], case["dim"]).flatten(1).repeat(case["pages"], 1)


def _from_symbols_plain(s):
    case = s["case"]
    s["codes"][s["pages"]] = _pack(s["symbols"].view(case["pages"], 2, case["kv_heads"], case["page"], case["dim"]))
    return s["codes"]


def run(s):
    case = s["case"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "to_symbols": _to_symbols_plain, "from_symbols": _from_symbols_plain}[case["op"]](s)
    from torch_ans_b200 import _C

    if case["op"] == "append":
        q = _C.kv4_append(s["codes"], s["params"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"], rotation=s["rotation"],
                          interleaved=case["interleaved"])
        k, v = _C.kv4_gather(s["codes"], s["params"], s["slots"], s["k"].dtype)
        return {"q": q, "k": k, "v": v}
    if case["op"] == "attend":
        return _C.kv4_attend(s["q"], s["codes"], s["params"], s["pages"], s["lengths"], q_starts=s["q_starts"], max_queries=s["max_queries"], scale=s["scale"])
    if case["op"] == "to_symbols":
        return _C.kv4_to_symbols(s["codes"], s["pages"], by_channel=case["by_channel"])
    _C.kv4_from_symbols(s["symbols"], s["codes"], s["pages"])
    return s["codes"]


def work(case):
    if case["op"] in ("to_symbols", "from_symbols"):
        n = case["pages"] * 2 * case["kv_heads"] * case["page"] * case["dim"]
        return {"bytes": n * (8.5 if case["op"] == "to_symbols" else 4.5) + 8 * case["pages"], "flops": 0}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    row = dim / 2 + 4  # a stored row: its codes and its parameters
    if case["op"] == "append":
        n, kept = case["tokens"], case["tokens"] - case["padding"]
        # in: queries, keys and values; out: the queries turned, the rows stored, and the values they stand for
        moved = n * (2 * heads + 2 * kv) * dim * 2 + kept * 2 * kv * (row + dim * 2) + n * (4 * case["rotary"] + 16)
        return {"bytes": moved, "flops": n * (heads + kv) * case["rotary"] * 3 + kept * 2 * kv * dim * 6}
    lengths, queries = _lengths(case), _queries(case)
    moved = sum(lengths) * 2 * kv * row + sum(queries) * heads * dim * 4
    pairs = sum(max(0, m - n + i + 1) for m, n in zip(lengths, queries) for i in range(n))
    return {"bytes": moved, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    if case["op"] in ("to_symbols", "from_symbols"):
        return None  # whole numbers
    s = prepare(case, seed)
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        half = case["rotary"] // 2
        turn = torch.complex(s["rotation"][:, :half].double(), s["rotation"][:, half:].double())[s["positions"]]

        def rotate(x):
            x = x.double().clone()
            r = x[..., : case["rotary"]]
            first, second = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., :half], r[..., half:])
            z = torch.complex(first, second) * turn[:, None]
            if case["interleaved"]:
                r[..., 0::2], r[..., 1::2] = z.real, z.imag
            else:
                r[..., :half], r[..., half:] = z.real, z.imag
            return x

        def stored(x):
            x = x.double()
            offset = x.min(-1, keepdim=True).values.to(torch.bfloat16).double()
            scale = ((x.max(-1, keepdim=True).values - offset) / 15).to(torch.bfloat16).double()
            scale[scale < TINY] = 0
            c = torch.where(scale > 0, torch.round((x - offset) / scale), torch.zeros_like(x)).clamp(0, 15)
            x = c * scale + offset
            x[s["slots"] < 0] = 0
            return x

        return {"q": rotate(s["q"]), "k": stored(rotate(s["k"])), "v": stored(s["v"])}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, start = case["heads"] // kv, 0
    for b, (m, n) in enumerate(zip(_lengths(case), _queries(case))):
        if m and n:
            pages = s["pages"][b, : -(-m // case["page"])].long()
            for h in range(kv):
                both = []
                for side in (0, 1):
                    byte = s["codes"][pages, side, h].reshape(-1, dim // 2)[:m].int()
                    p = s["params"][pages, side, h].reshape(-1, 2)[:m].double()
                    x = torch.empty(m, dim, dtype=torch.float64, device="cuda")
                    x[:, 0::2], x[:, 1::2] = byte % 16, byte // 16
                    both.append(x * p[:, :1] + p[:, 1:])
                q = s["q"][start : start + n, h * group : (h + 1) * group].double()
                hidden = torch.arange(m, device="cuda") > (torch.arange(n, device="cuda") + (m - n))[:, None]
                for g in range(group):
                    score = (q[:, g] @ both[0].T * s["scale"]).masked_fill(hidden, float("-inf"))
                    out[start : start + n, h * group + g] = torch.nan_to_num(torch.softmax(score, -1)) @ both[1]
        start += n
    return out
