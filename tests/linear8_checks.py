"""Plain implementations in 64 bits for the tests of products with 8-bit weights, and how far a kernel may be from them.

A product y = sum over groups of sx sw (sum of code products).  A group's sum is four MMAs of 32 products on the sum so far: 33 terms each, none
cut off by more than 2^-24 of the largest, so 4 * 33 * 2^-24 of the group's sum of magnitudes; the product of the scales and the
multiplication by it round by 2^-24 each, an addition to the sum so far by 2^-24 of no more than the sum A of all magnitudes, one for
each of G groups and of 8 pieces of k.  In all (142 + G) * 2^-24 * A, and half a step of the result's type.
"""
import torch

GROUP, TOP, TINY = 128, 448.0, 2.0 ** -126
U = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def to_e4m3(y: torch.Tensor) -> torch.Tensor:
    """float64: the nearest e4m3 number, ties to even"""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def groups_of(v: torch.Tensor, rows: int):
    """fp32 [R, K] -> codes as numbers [R, K], scales [R / rows, K / 128], both by the definition in fp32; groups that hold what is not finite: NaN, zeros"""
    r, k = v.shape
    p = torch.zeros(-(-r // rows) * rows, -(-k // GROUP) * GROUP, dtype=torch.float32, device=v.device)
    p[:r, :k] = v
    p = p.view(p.shape[0] // rows, rows, -1, GROUP)
    top = p.abs().amax(dim=(1, 3))
    fine = p.isfinite().all(dim=3).all(dim=1)
    s = (top * (1 / TOP)).clamp(min=TINY)
    q = torch.where(fine[:, None, :, None], p / s[:, None, :, None], torch.zeros_like(p))
    codes = to_e4m3(q.double()).clamp(-TOP, TOP)   # (a quotient is 448 * (1 + 2^-23) at most)
    return codes.reshape(codes.shape[0] * rows, -1)[:r, :k], torch.where(fine, s, torch.full_like(s, float("nan")))


def spread(scales: torch.Tensor, rows: int, n: int, k: int) -> torch.Tensor:
    return scales.double().repeat_interleave(rows, dim=0)[:n].repeat_interleave(GROUP, dim=1)[:, :k]


def product(rows, layer):
    """(y, what a kernel may be off before it rounds) in 64 bits, from the codes and scales that rows and layer hold"""
    x = rows.codes.double() * spread(rows.scales.t(), 1, *rows.codes.shape)
    w = layer.codes.double() * spread(layer.scales, GROUP, *layer.codes.shape)
    groups = -(-layer.k // GROUP)
    return x @ w.t(), (142 + groups) * U * (x.abs() @ w.abs().t())


def assert_near(got, want, off, dtype, what=""):
    got = got.double()
    bad = (got - want).abs() > off + half_step(dtype) * (want.abs() + off)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()}"


def hidden(rows, gate, up):
    """(h, what a kernel may be off before it rounds): silu has a slope of at most 1.1; exp is within 2 + 1.2 |g| steps of 2^-23, the quotient within
    2, and 1 + exp and two products round once each"""
    (g, dg), (u, du) = product(rows, gate), product(rows, up)
    act = g * torch.sigmoid(g)
    return act * u, 1.1 * dg * (u.abs() + du) + act.abs() * du + act.abs() * u.abs() * (2 * (2 + 1.2 * g.abs()) + 8) * U * 2


def assert_hidden(rows8, want, off):
    """8-bit rows near h: half a step of e4m3 (2^-4 of the number, 2^-10 below 2^-6) of what may be off by `off`; a scale is the largest's share"""
    t, k = want.shape
    s = rows8.scales.t().double()
    pad = torch.nn.functional.pad(want.abs(), (0, -k % GROUP)).view(t, -1, GROUP).amax(dim=2) / TOP
    dpad = torch.nn.functional.pad(off, (0, -k % GROUP)).view(t, -1, GROUP).amax(dim=2) / TOP
    assert ((s - pad.clamp(min=TINY)).abs() <= dpad + 2 * U * pad + 2.0 ** -149).all()
    got = rows8.codes.double() * spread(rows8.scales.t(), 1, t, k)
    each = spread(rows8.scales.t(), 1, t, k)
    room = off + (want.abs() + off) * 2.0 ** -4 * (1 + 4 * U) + each * 2.0 ** -10
    assert ((got - want).abs() <= room).all()


def case(t, n, k, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, k, device="cuda", generator=gen) * torch.exp(torch.randn(t, 1, device="cuda", generator=gen))
    w = torch.randn(n, k, device="cuda", generator=gen) * torch.exp(torch.randn(n, 1, device="cuda", generator=gen)) * k ** -0.5
    return x.to(dtype), w.to(dtype)
