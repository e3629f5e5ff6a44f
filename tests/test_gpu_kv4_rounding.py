"""Stored rows are the definition's to the last bit: offset = bf16(min), scale = bf16((max - offset) * r) with r the float nearest
1/15 and the product rounded to float, code = the quotient (x - offset) / scale rounded to the nearest whole number, ties to even.
Rows are not rotated, so every float here is known exactly; quotients are taken on the CPU, where a division is a division."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(x):
    """codes, scale, offset of rows x (any 16-bit type), on the CPU."""
    x = x.cpu().float()
    offset = x.amin(-1, keepdim=True).to(torch.bfloat16).float()
    scale = ((x.amax(-1, keepdim=True) - offset) * torch.tensor(1.0).div(15.0)).to(torch.bfloat16).float()
    scale = torch.where(scale < 2.0 ** -100, torch.zeros_like(scale), scale)
    c = ((x - offset) / scale).round().clamp(0, 15)  # round is to even
    return torch.where(scale > 0, c, torch.zeros_like(c)).to(torch.uint8), scale[..., 0], offset[..., 0]


def check(x):
    from torch_ans_b200 import _C
    n, kv, dim = x.shape
    page = 64
    codes = torch.zeros(-(-n // page), 2, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
    params = torch.zeros(-(-n // page), 2, kv, page, 2, dtype=torch.bfloat16, device="cuda")
    t = torch.arange(n, device="cuda")
    _C.kv4_append(codes, params, x, x, t)
    c, scale, offset = definition(x)
    for side in (0, 1):
        held = codes[t // page, side, :, t % page].cpu()
        got = torch.stack([held & 15, held >> 4], -1).flatten(-2)
        p = params[t // page, side, :, t % page].cpu().float()
        assert torch.equal(p[..., 1], offset)
        assert torch.equal(p[..., 0], scale)
        assert torch.equal(got, c)
    assert _C.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_random_rows(dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(9000, 2, dim, device="cuda", generator=g) * torch.exp(torch.randn(9000, 2, 1, device="cuda", generator=g))
    check(x.to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_at_ties(dtype):
    """max - offset = 15 m with an odd m of nine bits: a quotient by 15 lies half way between two bfloat16 numbers, and the
    product with r on one side for 55 of the 128."""
    rows = []
    for m in range(257, 512, 2):
        for low in range(0, 256):  # an offset that leaves a representable maximum
            top = torch.tensor(15.0 * m - low * 32)
            if float(top.to(dtype)) == float(top):
                x = torch.linspace(0, 1, 64) * (15.0 * m) - low * 32
                x = x.to(dtype).clamp(-low * 32, float(top))
                x[0], x[-1] = -low * 32, float(top)
                rows.append(x)
                break
    assert len(rows) > 50
    x = torch.stack(rows)[:, None].to("cuda")
    c, scale, offset = definition(x)
    exact = (x.amax(-1).cpu().double() - offset.double()) / 15
    assert ((exact - scale.double()).abs() * 2 == exact.log2().floor().exp2() * 2.0 ** -7).float().mean() > 0.9  # ties
    check(x)


def test_codes_at_ties():
    """x - offset = (n + 1/2) scale for every n, and its neighbours in float16."""
    scale = torch.tensor([0.5, 0.75, 0.8125, 0.9921875, 2.0 ** -6])
    x = torch.zeros(5, 1, 64, dtype=torch.float16)
    for i, s in enumerate(scale):
        v = ((torch.arange(15) + 0.5) * s).to(torch.float16)
        x[i, 0, :15] = v
        x[i, 0, 15:30] = torch.nextafter(v, torch.tensor(100.0, dtype=torch.float16))
        x[i, 0, 30:45] = torch.nextafter(v, torch.tensor(-100.0, dtype=torch.float16))
        x[i, 0, 45] = 15 * s
    x = x.cuda()
    c, s, o = definition(x)
    assert torch.equal(s[:, 0], scale) and o.eq(0).all()
    assert c[0, 0, :15].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14]
    check(x)
