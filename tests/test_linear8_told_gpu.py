"""What include/tgis_w8.h says of the 8-bit products beyond their formulas: the hidden rows' codes, scales whose product leaves fp32's range, rows whose squares do."""
import pytest
import torch

import linear8_checks as checks
from linear8_checks import GROUP, U

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from vllm_tgis_adapter_b200.engine import linear8

    return linear8


# one size at least for each kernel: tokens as columns (16, 32, 64 of them), pairs whole and cut along k
@pytest.mark.parametrize("t,hidden,ffn", [(1, 4096, 1024), (20, 512, 1536), (60, 1000, 700), (90, 512, 512), (300, 4096, 512), (300, 512, 4096), (1100, 256, 700)])
def test_codes_of_hidden_rows(lib, t, hidden, ffn):
    """A code is that of a number that is off from h / s by no more than sums, exp and quotient are (checks.hidden) and the reciprocal's product, 3 * 2^-24 (1.5 ulp), where
    s is the stored scale."""
    x, gate = checks.case(t, ffn, hidden, 3)
    up = checks.case(1, ffn, hidden, 4)[1]
    rows = lib.quantise(x)
    block = lib.FeedForward8(*(lib.Linear8.from_weight(w) for w in (gate, up, gate.t().contiguous())))
    h = block.hidden(rows)
    want, off = checks.hidden(rows, block.gate, block.up)
    s = checks.spread(h.scales.t(), 1, t, ffn)
    lo, hi = (checks.to_e4m3(((want + sign * off) / s) * (1 + sign * want.sign() * 3 * U)) for sign in (-1, 1))
    got = h.codes.double()
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.parametrize("t,hidden,ffn", [(1, 4096, 1024), (20, 512, 1536), (60, 1000, 700), (90, 512, 512), (300, 4096, 512), (300, 512, 4096), (1100, 256, 700)])
def test_codes_of_hidden_rows_of_exact_sums(lib, t, hidden, ffn):
    """Codes that are whole numbers up to 3 and scales that are powers of two: every sum is exact in fp32 (9 * 4096 < 2^24), whatever its order, so that silu and the
    quotient are all that is off.  |g| < 40 then (the sums' deviation is 4 * 64 at most, the scales bring it to 6): (12 + 2.4 * 40) * 2^-23 + 3 * 2^-24 of a number is less than
    2^-16, where the middles of codes are 2^-4 apart: no room but in 2^-11 of all, and below 2^-6, where they are 2^-9 apart, no more."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    ints = lambda *shape: torch.randint(-3, 4, shape, device="cuda", generator=gen).float()  # noqa: E731
    rows = lib.Rows8(t, hidden, torch.device("cuda", 0))
    rows.codes.copy_(ints(t, hidden).to(torch.float8_e4m3fn))
    down = 2.0 ** -torch.ceil(torch.log2(torch.tensor(4 * hidden ** 0.5 / 6)))
    rows.scales.fill_(float(down))
    gate, up = (lib.Linear8(ints(ffn, hidden).to(torch.float8_e4m3fn), torch.ones(-(-ffn // GROUP), -(-hidden // GROUP), device="cuda")) for _ in range(2))
    block = lib.FeedForward8(gate, up, lib.Linear8.from_weight(torch.ones(8, ffn, device="cuda")))
    h = block.hidden(rows)
    g, u = (checks.product(rows, m)[0] for m in (gate, up))
    assert g.abs().max() < 40
    want = g * torch.sigmoid(g) * u
    off = want.abs() * ((12 + 2.4 * g.abs()) * 2 * U + 3 * U)
    s = checks.spread(h.scales.t(), 1, t, ffn)
    lo, hi = (checks.to_e4m3((want + sign * off) / s) for sign in (-1, 1))
    got = h.codes.double()
    assert ((got >= lo) & (got <= hi)).all()
    assert (lo == hi).double().mean() > 1 - 2.0 ** -8
    top = torch.nn.functional.pad(want.abs(), (0, -ffn % GROUP)).view(t, -1, GROUP).amax(dim=2) / checks.TOP
    room = torch.nn.functional.pad(off, (0, -ffn % GROUP)).view(t, -1, GROUP).amax(dim=2) / checks.TOP
    assert ((h.scales.t().double() - top.clamp(min=checks.TINY)).abs() <= room + 2 * U * top).all()


@pytest.mark.parametrize("t", [1, 100, 300])
def test_scales_whose_product_is_small(lib, t):
    """2^-70 by 2^-70 has nine bits left: the product of the scales is off by half of 2^-149 at most, times the sum of the code products."""
    n, k = 200, 700
    x, w = (v.float() for v in checks.case(t, n, k, 5))
    for down in (2.0 ** -60, 2.0 ** -64, 2.0 ** -70, 2.0 ** -80):
        rows, layer = lib.quantise(x * down), lib.Linear8.from_weight(w * down)
        y = layer(rows, dtype=torch.float32)
        want, off = checks.product(rows, layer)
        sums = rows.codes.double().abs() @ layer.codes.double().abs().t()
        checks.assert_near(y, want, off + sums * 2.0 ** -150 + 2.0 ** -149 * (-(-k // GROUP) + 8), torch.float32)


@pytest.mark.parametrize("t", [1, 100, 300])
def test_scales_whose_product_is_an_infinity(lib, t):
    x, w = (v.float() for v in checks.case(t, 200, 256, 6))
    x[:, 128:] = 0
    w[:5] = 0
    rows, layer = lib.quantise(x * 2.0 ** 80), lib.Linear8.from_weight(w * 2.0 ** 80)
    assert rows.scales[0].min().double() * layer.scales[:, 0].min().double() > 2.0 ** 128   # (scales are the largest numbers' 448th part)
    y = layer(rows, dtype=torch.float32)
    assert y[:, 5:].isinf().all() and y[:, :5].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_squares_are_too_large(lib, dtype):
    x = torch.randn(3, 384, device="cuda").to(dtype)
    x[1] *= 2.0 ** 70
    rows = lib.quantise(x, norm=torch.ones(384, device="cuda", dtype=torch.bfloat16))
    codes, _ = checks.groups_of(x.float(), 1)
    assert torch.equal(rows.codes.double(), codes) and (rows.scales[:, 1] == 0).all() and (rows.scales[:, [0, 2]] > 0).all()
