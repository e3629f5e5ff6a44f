"""The 4-bit key/value cache on the GPU against its definition in 64 bits (tests/kv4_plain.py).

Tolerances.  A stored row: scale and offset are bfloat16 roundings of values computed in float, so they are within one
bfloat16 unit (2^-7 relative) of the 64-bit ones; a value is then within half a step of the row, plus what the two
roundings cut off at the ends (15 steps x 2^-8 and 2^-8 of the smallest value), plus the float rounding of the rotation
(2^-22 of the row's largest).  Attention: kv4_plain.attend_bounds, plus the output's own rounding."""
import pytest
import torch

from tests import kv4_plain as P

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def C():
    from torch_ans_b200 import _C
    _C.set_sync_check(False)
    _C.device_status()
    return _C


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rotation(rows, r):
    angle = torch.arange(rows, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, r, 2, device="cuda") / r)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def qkv(n, heads, kv, dim, dtype, seed, how="packed"):
    """Rows of a fused projection, as views: packed (strided tokens), odd (rows on odd addresses) or heads (heads first)."""
    x = torch.randn(n, (heads + 2 * kv) * dim + 1, device="cuda", generator=gen(seed)) * 2
    x = (x * torch.exp(torch.randn(x.shape[1], device="cuda", generator=gen(seed + 1)))).to(dtype)
    x = x[:, 1:] if how == "odd" else x[:, :-1].contiguous()
    q, k, v = (t.unflatten(1, (-1, dim)) for t in x.split([heads * dim, kv * dim, kv * dim], 1))
    if how == "heads":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    return q, k, v


APPEND = [(1, 8, 2, 64, BF, 64, False, 16, "packed"), (7, 3, 1, 128, FP, 64, True, 48, "odd"),
          (130, 32, 8, 128, BF, 128, False, 16, "packed"), (33, 4, 4, 256, FP, 256, False, 64, "heads"),
          (257, 6, 2, 64, FP, 32, True, 32, "packed"), (19, 5, 5, 256, BF, 48, False, 16, "odd"),
          (40, 2, 1, 128, BF, 0, False, 16, "packed"), (1025, 16, 8, 128, FP, 112, False, 128, "heads")]


@pytest.mark.parametrize("n,heads,kv,dim,dtype,r,interleaved,page,how", APPEND)
def test_append_stores_rotated_rows(C, n, heads, kv, dim, dtype, r, interleaved, page, how):
    q, k, v = qkv(n, heads, kv, dim, dtype, n, how)
    total = -(-n // page) + 3
    codes, params = P.pool(total, kv, page, dim, 5)
    before, before_p = codes.clone(), params.clone()
    slots = torch.randperm(total * page, device="cuda", generator=gen(2))[:n]
    skipped = torch.arange(n, device="cuda") % 5 == 3
    slots[skipped] = -1
    pos = torch.randint(0, 700, (n,), device="cuda", generator=gen(3))
    rot = rotation(700, r) if r else None
    turned = C.kv4_append(codes, params, k, v, slots, q=q, positions=pos if r else None, rotation=rot,
                          interleaved=interleaved)
    eq, ek = (P.rotate(t, pos, rot, interleaved) if r else t.double() for t in (q, k))
    size = eq.abs().amax(-1, keepdim=True)
    assert turned.dtype == dtype and turned.is_contiguous()
    assert ((turned.double() - eq).abs() <= P.rounding(eq, dtype) + 2 * size * 2.0 ** -22).all()
    hk, hv = C.kv4_gather(codes, params, slots, torch.bfloat16)
    keep = ~skipped
    for side, (x, held) in enumerate(((ek, hk), (v.double(), hv))):
        assert held[skipped].eq(0).all()
        s = slots[keep]
        got = params[s // page, side, :, s % page].double()
        scale, offset = P.params_of(x[keep])
        assert ((got[..., 0] - scale).abs() <= scale * 2.0 ** -7).all()
        assert ((got[..., 1] - offset).abs() <= offset.abs() * 2.0 ** -7).all()
        exact = P.values(codes[s // page, side, :, s % page], params[s // page, side, :, s % page])
        low = x[keep].amin(-1, keepdim=True).abs()
        most = x[keep].abs().amax(-1, keepdim=True)
        step = got[..., :1]
        assert ((exact - x[keep]).abs() <= step * (0.5 + 15 * 2.0 ** -8) + low * 2.0 ** -8 + most * 2.0 ** -22).all()
        # gathered values are those, rounded once
        assert ((held[keep].double() - exact).abs() <= P.rounding(exact, BF) + 2 * exact.abs() * 2.0 ** -24).all()
    # nothing else is written
    rest = torch.ones(total * page, dtype=torch.bool, device="cuda")
    rest[slots[keep]] = False
    rest = rest.view(total, page)[:, None, None, :].expand(total, 2, kv, page)
    assert torch.equal(codes[rest], before[rest]) and torch.equal(params[rest], before_p[rest])
    assert C.device_status() == 0


def test_append_rows_without_range_and_not_finite(C):
    dim, kv, page = 128, 1, 16
    k = torch.randn(9, kv, dim, device="cuda", generator=gen(1)).to(BF)
    v = k.clone()
    k[0], k[1], k[2], k[3] = 0.0, 3.25, -1e30, 1e-38  # no range: the row reads back as its bfloat16 value
    k[4, 0, 5], k[5, 0, 77], k[6, 0, 0] = float("nan"), float("inf"), float("-inf")
    k[7, 0, 3], k[7, 0, 4] = 3.0e38, -3.0e38  # a range past float
    v[8] = torch.arange(dim, device="cuda") % 16  # exactly the codes
    codes, params = P.pool(2, kv, page, dim)
    C.kv4_append(codes, params, k, v, torch.arange(9, device="cuda"))
    hk, hv = C.kv4_gather(codes, params, torch.arange(9, device="cuda"), BF)
    assert torch.equal(hk[:4], k[:4])
    assert hk[4:8].isnan().all()
    assert torch.equal(hv[8], v[8])
    assert C.device_status() == 0


def test_append_flags_bad_slots_and_positions(C):
    q, k, v = qkv(4, 2, 2, 64, BF, 0)
    codes, params = P.pool(3, 2, 16, 64)
    before = codes.clone()
    C.kv4_append(codes, params, k, v, torch.tensor([48, 1 << 40, -1, -(1 << 50)], device="cuda"))
    assert C.device_status() == 1 and torch.equal(codes, before)
    pos = torch.tensor([0, 10, -1, 3], device="cuda")
    out = C.kv4_append(codes, params, k, v, torch.arange(4, device="cuda"), q=q, positions=pos, rotation=rotation(10, 64))
    assert C.device_status() == 1
    assert torch.equal(out[1:3], q[1:3]) and not torch.equal(out[3], q[3])
    hk, _ = C.kv4_gather(codes, params, torch.tensor([48, 0], device="cuda"), BF)
    assert C.device_status() == 1 and hk[0].eq(0).all() and not hk[1].eq(0).all()


def run_attend(C, lengths, counts, heads, kv, dim, page, dtype, causal=True, seed=0, how="packed", max_queries=None,
               scale=None, q_scale=1.0, edit=None):
    pages, total = P.table(lengths, page, seed)
    codes, params = P.pool(total, kv, page, dim, seed)
    if edit:
        edit(codes, params, pages)
    starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
    q = (qkv(starts[-1], heads, kv, dim, dtype, seed, how)[0].float() * q_scale / 4).to(dtype)
    if how == "odd":
        q = torch.cat([q.new_zeros(q.shape[0], heads, 1), q], -1)[..., 1:]
    lse = torch.full((starts[-1], heads), 7.0, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    out = C.kv4_attend(q, codes, params, pages, torch.tensor(lengths, **i32),
                       q_starts=None if counts == [1] * len(counts) and how == "packed" else torch.tensor(starts, **i32),
                       max_queries=max_queries, causal=causal, scale=scale, lse=lse)
    ref, ref_lse, bound, score_bound = P.attend(q, codes, params, pages, lengths, starts, dim ** -0.5 if scale is None else scale, causal)
    assert out.shape == q.shape and out.dtype == dtype
    err = (out.double() - ref).abs()
    least = 2.0 ** -24 if dtype == FP else 0.0  # float16's smallest step
    assert (err <= bound + ref.abs() * P.U[dtype] * 1.01 + least).all(), (err / bound.clamp(min=1e-30)).max()
    none = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    if (~none).any():
        assert ((lse.double() - ref_lse)[~none].abs() <= (score_bound + ref_lse.abs() * 2.0 ** -20)[~none]).all()
    assert out[none].eq(0).all()
    assert C.device_status() == 0
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 1000]


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [
    (8, 8, 64, 16, BF), (32, 8, 128, 16, BF), (16, 2, 128, 64, FP), (6, 2, 256, 48, BF), (7, 1, 64, 32, FP),
    (64, 2, 128, 128, BF), (12, 1, 256, 16, FP), (71, 1, 64, 16, BF)])
def test_attend_one_query(C, heads, kv, dim, page, dtype):
    run_attend(C, EDGES, [1] * len(EDGES), heads, kv, dim, page, dtype, seed=heads)


@pytest.mark.parametrize("lengths", [[1], [40000], [5, 30011], [3] * 300])
@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(32, 8, 128, 16, BF), (8, 1, 64, 64, FP), (2, 2, 256, 32, FP)])
def test_attend_one_query_few_and_many_sequences(C, lengths, heads, kv, dim, page, dtype):
    run_attend(C, lengths, [1] * len(lengths), heads, kv, dim, page, dtype, seed=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,page,dtype,counts", [
    (8, 8, 64, 32, BF, 5), (16, 4, 128, 16, FP, 3), (9, 3, 256, 16, BF, 2), (16, 2, 128, 48, BF, 8), (5, 1, 64, 16, FP, 7)])
def test_attend_drafted_queries(C, heads, kv, dim, page, dtype, counts, causal):
    lengths = [0, 1, 2, 4, 16, 17, 40, 64, 129, 500, 2049]  # the first have more queries than tokens: rows that see nothing
    n = [counts, counts, 0, counts, counts, 1, counts, counts, counts - 1, counts, counts]
    run_attend(C, lengths, n, heads, kv, dim, page, dtype, causal, seed=counts)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(8, 2, 128, 16, BF), (4, 4, 64, 48, FP), (3, 1, 256, 32, BF),
                                                      (16, 2, 64, 128, BF), (6, 1, 128, 16, FP)])
def test_attend_prompts(C, heads, kv, dim, page, dtype, causal):
    lengths = [1, 300, 0, 129, 64, 700, 17]
    counts = [1, 300, 0, 129, 64, 700, 17]
    run_attend(C, lengths, counts, heads, kv, dim, page, dtype, causal, seed=4)
    counts = [3, 200, 70, 1, 64, 333, 0]  # chunks of prompts, some longer than what is there
    run_attend(C, lengths, counts, heads, kv, dim, page, dtype, causal, seed=5, how="heads")


@pytest.mark.parametrize("heads,kv,dim,page,dtype,count,length", [
    (4, 1, 128, 64, BF, 100, 20000), (16, 4, 64, 16, FP, 65, 9001), (2, 2, 256, 16, BF, 130, 5000), (32, 1, 128, 32, FP, 9, 12345)])
def test_attend_chunk_of_a_long_prompt(C, heads, kv, dim, page, dtype, count, length):
    run_attend(C, [length], [count], heads, kv, dim, page, dtype, seed=6)


@pytest.mark.parametrize("count", [1, 4, 150])
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (BF, 256)])
def test_attend_unaligned_rows_and_wrong_hint(C, dtype, dim, count):
    run_attend(C, [200, 333], [count, count], 4, 2, dim, 16, dtype, seed=7, how="odd")
    run_attend(C, [200, 333], [count, count], 4, 2, dim, 16, dtype, seed=7, how="heads", max_queries=1)
    run_attend(C, [200, 333], [count, count], 4, 2, dim, 16, dtype, seed=7, max_queries=100000)


@pytest.mark.parametrize("counts", [[1, 1], [6, 6], [100, 256]])
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (BF, 256)])
def test_attend_large_and_small_values(C, dtype, dim, counts):
    """Scores far apart (a softmax with one weight), rows of very different sizes, values past float16."""
    def sizes(codes, params, pages):
        f = torch.exp2(torch.randint(-12, 9, params.shape[:-1], device="cuda", generator=gen(9)).float())
        params[:, 1] = (params[:, 1].float() * f[:, 1, ..., None] * (2.0 ** 12 if dtype == BF else 1.0)).to(BF)
        params[:, 0] = (params[:, 0].float() * 4).to(BF)
    run_attend(C, [300, 257], counts, 4, 2, dim, 16, dtype, seed=8, q_scale=4.0, edit=sizes)

    def tiny(codes, params, pages):
        params[:, 1] = (params[:, 1].float() * 2.0 ** -60).to(BF)
    if dtype == BF:
        run_attend(C, [300, 257], counts, 4, 2, dim, 16, dtype, seed=8, edit=tiny)
        run_attend(C, [300, 257], counts, 4, 2, dim, 16, dtype, seed=8, scale=-0.05)


@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 5, 5], [90, 100, 20]])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attend_ignores_what_is_past_the_end(C, dim, counts):
    """Rows of the last page after a sequence's end, and pages that no sequence has, hold anything."""
    lengths = [100, 47, 16]

    def dirt(codes, params, pages):
        used = torch.zeros(params.shape[0], params.shape[3], dtype=torch.bool, device="cuda")
        for b, n in enumerate(lengths):
            for t in range(n):
                used[pages[b, t // 16], t % 16] = True
        params.copy_(torch.where(used[:, None, None, :, None], params, float("nan")))
    run_attend(C, lengths, counts, 4, 2, dim, 16, BF, seed=10, edit=dirt)


@pytest.mark.parametrize("count", [1, 70])
def test_attend_passes_stored_nan_to_the_queries_that_see_it(C, count):
    pages, total = P.table([200], 16)
    codes, params = P.pool(total, 2, 16, 128)
    params[pages[0, 8].item(), 0, 1, 2] = float("nan")  # token 130, a key of head 1
    q = torch.randn(count, 4, 128, device="cuda", generator=gen(1)).to(BF)
    i32 = dict(dtype=torch.int32, device="cuda")
    out = C.kv4_attend(q, codes, params, pages, torch.tensor([140], **i32), q_starts=torch.tensor([0, count], **i32))
    assert out[:, :2].isfinite().all()
    sees = torch.arange(count, device="cuda") + 140 - count >= 130
    assert out[sees][:, 2:].isnan().all() and out[~sees][:, 2:].isfinite().all()


@pytest.mark.parametrize("count", [1, 6, 80])
def test_attend_flags_bad_pages_lengths_and_starts(C, count):
    lengths = [100, 300]
    pages, total = P.table(lengths, 16)
    codes, params = P.pool(total, 2, 16, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(2 * count, 4, 128, device="cuda", generator=gen(1)).to(BF)
    starts = [0, count, 2 * count]
    ln, st = torch.tensor(lengths, **i32), torch.tensor(starts, **i32)
    good = C.kv4_attend(q, codes, params, pages, ln, q_starts=st)
    bad = pages.clone()
    bad[1, 2], bad[1, 5] = total, -7  # hidden, and flagged
    out = C.kv4_attend(q, codes, params, bad, ln, q_starts=st)
    assert C.device_status() == 1
    ref, _, bound, _ = P.attend(q, codes, params, bad, lengths, starts, 128 ** -0.5)
    assert ((out.double() - ref).abs() <= bound + ref.abs() * P.U[BF] * 1.01).all()
    assert torch.equal(out[:count], good[:count])
    out = C.kv4_attend(q, codes, params, pages, torch.tensor([100, -5], **i32), q_starts=st)
    assert C.device_status() == 2 and torch.equal(out[:count], good[:count]) and out[count:].eq(0).all()
    full = torch.zeros_like(pages)
    C.kv4_attend(q, codes, params, full, torch.tensor([100, 1 << 30], **i32), q_starts=st)
    assert C.device_status() == 2
    # queries after the last sequence's are zeros; starts that are out of order belong to nobody
    out = C.kv4_attend(q, codes, params, pages[:1].contiguous(), ln[:1].contiguous(), q_starts=st[:2].contiguous())
    assert C.device_status() == 0 and torch.equal(out[:count], good[:count]) and out[count:].eq(0).all()
    C.kv4_attend(q, codes, params, pages, ln, q_starts=torch.tensor([0, 1 << 29, 2 * count], **i32))
    assert C.device_status() & 2


def test_attend_past_32_bits(C):
    """Pages more than 2^32 bytes into the pool."""
    page, kv, dim = 64, 8, 128
    total = (1 << 32) // (2 * kv * page * dim // 2) + 9
    codes = torch.empty(total, 2, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
    params = torch.empty(total, 2, kv, page, 2, dtype=torch.bfloat16, device="cuda")
    k = torch.randn(200, kv, dim, device="cuda", generator=gen(0)).to(BF)
    v = torch.randn(200, kv, dim, device="cuda", generator=gen(1)).to(BF)
    ids = [total - 1, 0, total - 2, total - 5]
    pages = torch.tensor([ids], dtype=torch.int32, device="cuda")
    t = torch.arange(200, device="cuda")
    slots = pages[0].long()[t // page] * page + t % page
    C.kv4_append(codes, params, k, v, slots)
    small_codes, small_params = codes[pages[0].long()].clone(), params[pages[0].long()].clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    for n in (1, 3, 150):
        q = torch.randn(n, 16, dim, device="cuda", generator=gen(2)).to(BF)
        st, ln = torch.tensor([0, n], **i32), torch.tensor([200], **i32)
        a = C.kv4_attend(q, codes, params, pages, ln, q_starts=st)
        b = C.kv4_attend(q, small_codes, small_params, torch.arange(4, **i32)[None], ln, q_starts=st)
        assert torch.equal(a, b)
    ids = pages[0].long()
    sym, _ = C.kv4_to_symbols(codes, ids)
    assert torch.equal(sym, C.kv4_to_symbols(small_codes, torch.arange(4, device="cuda"))[0])
    C.kv4_from_symbols(15 - sym, codes, ids)
    assert torch.equal(codes[ids], ~small_codes)
    assert C.device_status() == 0


@pytest.mark.parametrize("count", [1, 5, 200])
def test_attend_is_reproducible_on_other_streams_and_in_graphs(C, count):
    lengths = [3000, 11, 700]
    pages, total = P.table(lengths, 16)
    codes, params = P.pool(total, 2, 16, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(3 * count, 8, 128, device="cuda", generator=gen(1)).to(BF)
    ln, st = torch.tensor(lengths, **i32), torch.tensor([0, count, 2 * count, 3 * count], **i32)
    call = lambda: C.kv4_attend(q, codes, params, pages, ln, q_starts=st, max_queries=count)  # noqa: E731
    first = call()
    torch.cuda.synchronize()
    for _ in range(5):
        assert torch.equal(call(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [call() for _ in range(3)]
    others = [call() for _ in range(3)]  # at the same time on this stream
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs + others)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = call()
    for _ in range(3):
        held.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, first)
    ln.copy_(torch.tensor([64, 11, 0], **i32))  # a graph reads the lengths when it runs
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, call()) and not torch.equal(held, first)
    torch.cuda.set_sync_debug_mode("error")
    try:
        call()
    finally:
        torch.cuda.set_sync_debug_mode(0)
    del g


@pytest.mark.parametrize("lengths,counts", [([700, 300], [700, 300]), ([9000], [300])])
def test_attend_wait_that_runs_out_is_reported(C, monkeypatch, lengths, counts):
    """Waits between a block's warps are bounded: one that runs out ends the call and flags TANS_DEV_STALLED, and the
    next call on the same stream is right."""
    pages, total = P.table(lengths, 16)
    codes, params = P.pool(total, 2, 16, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
    q = torch.randn(starts[-1], 8, 128, device="cuda", generator=gen(1)).to(BF)
    call = lambda: C.kv4_attend(q, codes, params, pages, torch.tensor(lengths, **i32),  # noqa: E731
                                q_starts=torch.tensor(starts, **i32))
    first = call()
    torch.cuda.synchronize()
    assert C.device_status() == 0
    monkeypatch.setenv("TORCH_ANS_B200_WAIT_LIMIT", "0")
    call()
    torch.cuda.synchronize()  # returns: no warp is still waiting
    assert C.device_status() & 64
    monkeypatch.delenv("TORCH_ANS_B200_WAIT_LIMIT")
    assert torch.equal(call(), first) and C.device_status() == 0


@pytest.mark.parametrize("n,kv,page,dim,by_channel", [(1, 1, 16, 64, False), (5, 3, 48, 128, True), (9, 8, 64, 256, False)])
def test_symbols(C, n, kv, page, dim, by_channel):
    codes, _ = P.pool(n + 4, kv, page, dim, n)
    ids = torch.randperm(n + 4, device="cuda", generator=gen(1))[:n]
    sym, idx = C.kv4_to_symbols(codes, ids, by_channel=by_channel)
    ref = P.unpack(codes[ids]).int()
    side = torch.arange(2 * kv, device="cuda", dtype=torch.int32).view(1, 2, kv, 1, 1)
    tab = side * dim + torch.arange(dim, device="cuda", dtype=torch.int32) if by_channel else side
    assert torch.equal(sym, ref.reshape(n * 2 * kv, page * dim))
    assert torch.equal(idx, tab.expand_as(ref).reshape(n * 2 * kv, page * dim))
    other = torch.zeros_like(codes)
    C.kv4_from_symbols(sym, other, ids)
    assert torch.equal(other[ids], codes[ids]) and int(other.count_nonzero()) == int(codes[ids].count_nonzero())
    assert C.device_status() == 0
    other.zero_()
    bad = ids.clone()
    bad[0] = n + 4
    sym2, _ = C.kv4_to_symbols(codes, bad)
    assert C.device_status() == 1 and sym2[: 2 * kv].eq(0).all() and torch.equal(sym2[2 * kv:], sym[2 * kv:])
    C.kv4_from_symbols(sym, other, bad)
    assert C.device_status() == 1 and other[ids[0]].eq(0).all() and torch.equal(other[ids[1:]], codes[ids[1:]])
    sym[0, 0] += 16
    C.kv4_from_symbols(sym, other, ids)
    assert C.device_status() == 2 and torch.equal(other[ids], codes[ids])


def test_empty_calls(C):
    codes, params = P.pool(2, 2, 16, 64)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = torch.empty(0, 2, 64, dtype=BF, device="cuda")
    out = C.kv4_append(codes, params, rows, rows, none, q=rows)
    assert out.shape == (0, 2, 64)
    assert C.kv4_gather(codes, params, none, FP)[0].shape == (0, 2, 64)
    empty = torch.empty(0, 3, **i32)
    assert C.kv4_attend(rows, codes, params, empty, torch.empty(0, **i32)).shape == (0, 2, 64)
    # sequences, but no page column: every length is 0
    q = torch.randn(2, 2, 64, device="cuda").to(BF)
    assert C.kv4_attend(q, codes, params, torch.empty(2, 0, **i32), torch.zeros(2, **i32)).eq(0).all()
    # queries, but no sequence
    assert C.kv4_attend(q, codes, params, empty, torch.empty(0, **i32), q_starts=torch.zeros(1, **i32)).eq(0).all()
    assert C.kv4_to_symbols(codes, none)[0].shape == (0, 16 * 64)
    C.kv4_from_symbols(torch.empty(0, 16 * 64, **i32), codes, none)
    assert C.device_status() == 0


def test_refusals(C):
    codes, params = P.pool(2, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros(3, 2, 64, dtype=BF, device="cuda")
    q = torch.zeros(3, 4, 64, dtype=BF, device="cuda")
    slots = torch.arange(3, device="cuda")
    ln, pages = torch.ones(3, **i32), torch.zeros(3, 1, **i32)
    rot, pos = rotation(5, 64), torch.zeros(3, dtype=torch.int64, device="cuda")
    refused = [
        lambda: C.kv4_append(codes.cpu(), params.cpu(), k, k, slots),
        lambda: C.kv4_append(codes.int(), params, k, k, slots),
        lambda: C.kv4_append(codes[:, :, :, :8].contiguous(), params[:, :, :, :8].contiguous(), k, k, slots),
        lambda: C.kv4_append(codes[:, :, :1], params[:, :, :1], k[:, :1], k[:, :1], slots),
        lambda: C.kv4_append(codes, params.float(), k, k, slots),
        lambda: C.kv4_append(codes, params[:1], k, k, slots),
        lambda: C.kv4_append(codes, params, k.float(), k.float(), slots),
        lambda: C.kv4_append(codes, params, k, k.half(), slots),
        lambda: C.kv4_append(codes, params, k[:, :1], k, slots),
        lambda: C.kv4_append(codes, params, k[:2], k, slots),
        lambda: C.kv4_append(codes, params, k.transpose(1, 2).contiguous().transpose(1, 2), k, slots),
        lambda: C.kv4_append(codes, params, k, k, slots.int()),
        lambda: C.kv4_append(codes, params, k, k, slots.cpu()),
        lambda: C.kv4_append(codes, params, k, k, slots, positions=pos),
        lambda: C.kv4_append(codes, params, k, k, slots, positions=pos, rotation=rot[:, :24].contiguous()),
        lambda: C.kv4_append(codes, params, k, k, slots, positions=pos, rotation=rot.half()),
        lambda: C.kv4_append(codes, params, k, k, slots, positions=pos, rotation=rotation(5, 128)),
        lambda: C.kv4_append(codes, params, k.clone().requires_grad_(), k, slots),
        lambda: C.kv4_gather(codes, params, slots, torch.float32),
        lambda: C.kv4_attend(q[:, :3], codes, params, pages, ln),
        lambda: C.kv4_attend(q[:2], codes, params, pages, ln),
        lambda: C.kv4_attend(q.float(), codes, params, pages, ln),
        lambda: C.kv4_attend(q[..., :32], codes, params, pages, ln),
        lambda: C.kv4_attend(q, codes, params, pages.long(), ln),
        lambda: C.kv4_attend(q, codes, params, pages[:2], ln),
        lambda: C.kv4_attend(q, codes, params, pages, ln.long()),
        lambda: C.kv4_attend(q, codes, params, pages, ln, q_starts=ln),
        lambda: C.kv4_attend(q, codes, params, pages, ln, max_queries=-1),
        lambda: C.kv4_attend(q, codes, params, pages, ln, lse=torch.zeros(3, 2, device="cuda")),
        lambda: C.kv4_attend(q.clone().requires_grad_(), codes, params, pages, ln),
        lambda: C.kv4_to_symbols(codes, slots.int()),
        lambda: C.kv4_from_symbols(torch.zeros(4, 100, **i32), codes, slots[:1]),
        lambda: C.kv4_from_symbols(torch.zeros(4, 1024, device="cuda"), codes, slots[:1]),
    ]
    for i, f in enumerate(refused):
        with pytest.raises(RuntimeError, match="torch_ans_b200"):
            f()
            pytest.fail(f"call {i} was not refused")
    assert C.device_status() == 0
