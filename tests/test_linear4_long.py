"""GPU: products with 4-bit weights over long rows, where bounds on rounding are too wide to see a lost piece: small whole numbers and scales that are
powers of two, whose sums fp32 holds exactly in any order, so that the result has to be the exact sum rounded once."""
import pytest
import torch

from bitsmoe_b200.layer import dense_mlp4, linear4
from bitsmoe_b200.quant import linear4 as q4

DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def whole_case(seed, tokens, n, k, group, dtype, device=None):
    """x in -3 .. 3, codes over their range, scales 2^-6 .. 2^-4: sums are multiples of 2^-6 below 2^24 of them (k < 174000)."""
    assert k * 3 * 8 * 4 < 2 ** 24
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, (tokens, k), generator=gen).to(dtype)
    codes = torch.randint(-8, 8, (n, k), generator=gen).to(torch.int8)
    scale = (2.0 ** torch.randint(-6, -3, (n, -(-k // group)), generator=gen)).half()
    on = device or DEV
    return x.to(on), codes.to(on), scale.to(on)


def whole_exact(x, codes, scale, group, residual=None):
    w = codes.double() * scale.double().repeat_interleave(group, dim=1)[:, :codes.shape[1]]
    y = x.double() @ w.T
    if residual is not None:
        y = y + residual.double()
    return y


def rounded(y, dtype):
    return y.float().to(dtype)          # exact in fp32


def test_the_comparison_sees_a_lost_piece():
    x, codes, scale = whole_case(1, 4, 24, 65000, 128, torch.float16, device="cpu")
    y = whole_exact(x, codes, scale, 128)
    assert torch.equal(y.float().double(), y)
    for lost in (slice(0, 32), slice(32512, 32640), slice(64960, 65000)):
        less = codes.clone()
        less[:, lost] = 0
        differ = rounded(whole_exact(x, less, scale, 128), torch.float16) != rounded(y, torch.float16)
        assert float(differ.float().mean()) > 0.9


SIZES = [(24, 20000, 128), (7, 65000, 128), (40, 120000, 64), (40, 96256, 32), (33, 96384, 128), (19, 120001, 128), (19, 120001, 32), (5, 173999, 64), (300, 30001, 64)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,group", SIZES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 9, 40, 200])
def test_long_rows(tokens, n, k, group, dtype):
    x, codes, scale = whole_case(n + k, tokens, n, k, group, dtype)
    payload = q4.pack_codes4(codes)
    res = torch.randint(-50, 51, (tokens, n), generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    assert torch.equal(linear4(x, payload, scale, group), rounded(whole_exact(x, codes, scale, group), dtype))
    assert torch.equal(linear4(x, payload, scale, group, residual=res), rounded(whole_exact(x, codes, scale, group, res), dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_long_rows_off_a_16_byte_boundary(tokens, dtype):
    n, k, group = 19, 120000, 64
    x, codes, scale = whole_case(3, tokens, n, k, group, dtype)
    flat = torch.zeros(tokens * k + 1, dtype=dtype, device=DEV)
    off = flat[1:].view(tokens, k)
    off.copy_(x)
    assert torch.equal(linear4(off, q4.pack_codes4(codes), scale, group), rounded(whole_exact(x, codes, scale, group), dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 40])
@pytest.mark.parametrize("hidden,inter", [(120001, 9), (16, 100001)])
def test_mlps_with_long_rows(tokens, hidden, inter, dtype):
    """Gate sums of 0 or far above: silu is then 0 or the sum itself, and the products between the matrices are whole numbers."""
    group = 64
    gen = torch.Generator().manual_seed(hidden)
    pick = torch.randint(0, 2, (inter,), generator=gen)
    x = torch.zeros(tokens, hidden)
    x[:, hidden - 2:] = torch.randint(1, 4, (tokens, 2), generator=gen).float()
    gate = torch.zeros(inter, hidden, dtype=torch.int8)
    gate[:, hidden - 1] = (pick * 4).to(torch.int8)               # sums of 0, or 4 .. 12 times the scale 16
    up = torch.zeros(inter, hidden, dtype=torch.int8)
    up[:, hidden - 2] = torch.randint(-2, 3, (inter,), generator=gen).to(torch.int8)
    down = torch.randint(-2, 3, (hidden, inter), generator=gen).to(torch.int8)
    x, gate, up, down = x.to(DEV, dtype), gate.to(DEV), up.to(DEV), down.to(DEV)
    one = [torch.full((m.shape[0], -(-m.shape[1] // group)), v, dtype=torch.float16, device=DEV) for m, v in ((gate, 16.0), (up, 0.0625), (down, 0.03125))]
    z = (x.double() @ gate.double().T * 16) * (x.double() @ up.double().T * 0.0625)      # silu(64) is 64 to 2^-90
    assert torch.equal(z.to(dtype).double(), z)
    y = z @ down.double().T * 0.03125
    assert torch.equal(y.float().double(), y)
    got = dense_mlp4(x, *((q4.pack_codes4(m), s) for m, s in zip((gate, up, down), one)), group)
    assert torch.equal(got, rounded(y, dtype))
