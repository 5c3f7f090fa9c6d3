"""Products with 8-bit weights on the GPU: rows and weights in 8 bits, products, the gated feed-forward block."""
import pytest
import torch

import linear8_checks as checks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from vllm_tgis_adapter_b200.engine import linear8

    return linear8


def bits(x: torch.Tensor) -> torch.Tensor:
    return x.view(torch.int32) if x.dtype == torch.float32 else x


# ------------------------------------------------------------------------------------------------------------ 8-bit rows
def same_groups(codes, scales, want_codes, want_scales):
    assert torch.equal(codes.double(), want_codes)
    assert torch.equal(scales.isnan(), want_scales.isnan())
    assert torch.equal(scales.nan_to_num(nan=0.0), want_scales.nan_to_num(nan=0.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 1), (1, 128), (3, 127), (2, 129), (5, 1000), (1, 4096), (700, 512), (601, 264), (9, 20000), (593, 77)])
def test_rows(lib, t, k, dtype):
    x, _ = checks.case(t, 1, k, t + k, dtype)
    rows = lib.quantise(x)
    assert rows.shape == (t, k) and rows.codes.shape == (t, k)
    codes, scales = checks.groups_of(x.float(), 1)
    same_groups(rows.codes, rows.scales, codes, scales.t())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 4096), (2, 130), (700, 512), (597, 96), (3, 131072)])
def test_rows_of_special_numbers(lib, t, k, dtype):
    """Zeros, the smallest and largest numbers, infinities, NaN: a group of its own each."""
    x, _ = checks.case(t, 1, k, 5, dtype)
    x[:, :3] = 0.0
    kinds = [float("nan"), float("inf"), -float("inf"), 0.0, 1e-40, 3e38, 2.0 ** -133, -2.0 ** -120]
    for g in range(k // 128):
        value = kinds[g % len(kinds)]
        if value in (0.0, 1e-40, 2.0 ** -133):
            x[:, g * 128:(g + 1) * 128] = value
        else:
            x[:, g * 128 + 7 * g % 128] = value
    rows = lib.quantise(x)
    codes, scales = checks.groups_of(x.float(), 1)
    same_groups(rows.codes, rows.scales, codes, scales.t())


def test_rows_that_16_byte_loads_do_not_reach(lib):
    base = torch.randn(40, 777, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        wide = base.to(dtype)
        for x in (wide[:, 3:515], wide[1:, :640], wide[:7, 1:2], wide[:1, 5:133]):
            codes, scales = checks.groups_of(x.float(), 1)
            rows = lib.quantise(x)
            same_groups(rows.codes, rows.scales, codes, scales.t())


def test_codes_of_every_quotient_near_a_tie(lib):
    """Numbers on and beside the middle of two e4m3 numbers round to even, and those beside it to the nearer."""
    numbers = torch.tensor(sorted(set(checks.to_e4m3(torch.linspace(0, 448, 20001, dtype=torch.float64)).tolist())))
    middles = ((numbers[1:] + numbers[:-1]) / 2).float()
    near = torch.cat([middles, torch.nextafter(middles, torch.zeros_like(middles)), torch.nextafter(middles, torch.full_like(middles, 500.0))])
    near = torch.cat([near, -near])
    near = torch.nn.functional.pad(near, (0, -len(near) % 127)).view(-1, 127)
    for unit in (1.0, 0.37, 3e-30, 2.0 ** 90):
        x = torch.cat([near, torch.full((len(near), 1), 448.0)], dim=1).cuda() * unit
        rows = lib.quantise(x.contiguous())
        codes, scales = checks.groups_of(x, 1)
        same_groups(rows.codes, rows.scales, codes, scales.t())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k,residual", [(1, 4096, True), (1, 100, False), (7, 512, True), (650, 768, True), (593, 2000, False), (4, 131072, True), (603, 33, True)])
def test_norm_and_residual(lib, t, k, residual, dtype):
    x, _ = checks.case(t, 1, k, 3, dtype)
    other, _ = checks.case(t, 1, k, 4, dtype)
    norm = (1 + 0.3 * torch.randn(k, device="cuda")).to(torch.bfloat16)
    keep = x.clone()
    r = (x.float() + other.float()).to(dtype) if residual else x
    new = torch.full_like(x, 7.0) if residual else None
    rows = lib.quantise(x, norm=norm, eps=1e-5, residual=other if residual else None, residual_out=new)
    codes, scales = checks.groups_of(r.float() * norm.float(), 1)
    assert torch.equal(rows.codes.double(), codes) and torch.equal(x, keep)
    if residual:
        assert torch.equal(new, r)
    # a row's sum is that of 8 warps of 32 lanes at most and one lane's share the k / 32 of a row at most; half of it in the root; the quotient, the
    # root, the reciprocal and the product round once each
    want = scales.double() / torch.sqrt(r.double().square().mean(dim=1, keepdim=True) + 1e-5)
    off = ((k / 32 + 16) / 2 + 4) * checks.U
    assert ((rows.scales.t().double() - want).abs() <= off * want).all()
    # in place
    if residual:
        again = lib.quantise(x, norm=norm, eps=1e-5, residual=other)
        assert torch.equal(other, r) and torch.equal(again.codes.view(torch.uint8), rows.codes.view(torch.uint8)) and torch.equal(again.scales, rows.scales)


def test_a_row_of_zeros_has_a_norm(lib):
    rows = lib.quantise(torch.zeros(2, 256, device="cuda", dtype=torch.bfloat16), norm=torch.ones(256, device="cuda", dtype=torch.bfloat16))
    assert (rows.codes.float() == 0).all() and rows.scales.isfinite().all()


def test_residual_alone_and_rows_out_of_larger_ones(lib):
    x, res = torch.randn(2, 600, 300, device="cuda").to(torch.bfloat16)
    out = lib.Rows8(600, 200, x.device)
    want = (x[:, 50:250].float() + res[:, 50:250].float()).to(torch.bfloat16)
    untouched = res.clone()
    assert lib.quantise(x[:, 50:250], residual=res[:, 50:250], out=out) is out
    codes, scales = checks.groups_of(want.float(), 1)
    same_groups(out.codes, out.scales, codes, scales.t())
    untouched[:, 50:250] = want
    assert torch.equal(res, untouched)


# --------------------------------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (127, 129), (128, 128), (129, 127), (256, 512), (2128, 2048), (300, 1000), (77, 5001)])
def test_weights(lib, n, k, dtype):
    _, w = checks.case(1, n, k, n + k, dtype)
    if n > 130:
        w[130, 3] = float("nan")
        w[2, k - 1] = float("inf")
        w[140:256] = 0
    layer = lib.Linear8.from_weight(w)
    codes, scales = checks.groups_of(w.float(), 128)
    same_groups(layer.codes, layer.scales, codes, scales)
    view = torch.randn(n + 1, k + 5, device="cuda").to(dtype)[1:, 2:2 + k]
    layer = lib.Linear8.from_weight(view)
    codes, scales = checks.groups_of(view.float(), 128)
    same_groups(layer.codes, layer.scales, codes, scales)


# -------------------------------------------------------------------------------------------------------------- products
SIZES = [(1, 1, 1), (1, 128, 128), (1, 6144, 4096), (2, 127, 129), (16, 129, 127), (17, 256, 1000), (32, 4096, 1536), (33, 300, 4096), (64, 2128, 2048), (65, 512, 256),
         (128, 768, 640), (129, 130, 2048), (200, 1024, 512), (256, 640, 384), (257, 257, 257), (300, 2128, 1024), (511, 512, 1536), (513, 1000, 333),
         (1000, 2176, 640), (1025, 4096, 512), (2048, 1536, 512), (2500, 300, 900), (64, 96, 28672), (3, 33000, 200), (700, 20, 131072)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", SIZES)
def test_product(lib, t, n, k, dtype):
    x, w = checks.case(t, n, k, t + n + k)
    rows, layer = lib.quantise(x), lib.Linear8.from_weight(w)
    y = layer(rows, dtype=dtype)
    layer.check()
    want, off = checks.product(rows, layer)
    assert y.dtype == dtype and y.shape == (t, n)
    checks.assert_near(y, want, off, dtype)
    assert torch.equal(bits(layer(rows, dtype=dtype)), bits(y))


@pytest.mark.parametrize("t", [1, 20, 70, 140, 300, 900])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_out_and_what_lies_around_it(lib, t, dtype):
    x, w = checks.case(t, 331, 520, t)
    rows, layer = lib.quantise(x), lib.Linear8.from_weight(w)
    want = layer(rows, dtype=dtype)
    for first, width in ((0, 331), (3, 337), (8, 344), (1, 333)):
        room = torch.full((t + 3, width + first), 5.0, device="cuda", dtype=dtype)
        out = room[1:t + 1, first:first + 331]
        assert layer(rows, out=out) is out
        assert torch.equal(bits(out.contiguous()), bits(want))
        room[1:t + 1, first:first + 331] = 5.0
        assert (room == 5.0).all()


@pytest.mark.parametrize("t", [3, 100, 300, 1100])
def test_what_is_not_finite_stays_in_its_row_or_block(lib, t):
    x, w = checks.case(t, 400, 1000, 11)
    x[1, 130], x[t - 1, 999] = float("nan"), float("inf")
    w[200, 5] = float("nan")
    rows, layer = lib.quantise(x), lib.Linear8.from_weight(w)
    y = layer(rows)
    bad = torch.zeros(t, 400, dtype=torch.bool, device="cuda")
    bad[1], bad[t - 1], bad[:, 128:256] = True, True, True
    assert torch.equal(y.isnan(), bad)
    clean, ok = lib.quantise(torch.where(torch.isfinite(x), x, torch.zeros_like(x))), lib.Linear8.from_weight(w.nan_to_num(nan=0.0))
    assert torch.equal(y[~bad], ok(clean)[~bad])


@pytest.mark.parametrize("t", [1, 40, 300, 1030])
def test_scales_of_any_rule_and_size(lib, t):
    """A checkpoint's matrix: scales that are not its blocks' largest share, among them 0, tiny and large ones; k and rows that do not start on 16 bytes."""
    n, k = 260, 403
    gen = torch.Generator(device="cuda").manual_seed(t)
    codes = (torch.randn(n, k, device="cuda", generator=gen) * 30).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp(6 * torch.randn(3, 4, device="cuda", generator=gen))
    scales[1, 2], scales[2, 0] = 0.0, 1e-30
    layer = lib.Linear8(codes, scales)
    rows = lib.quantise(checks.case(t, 1, k, 5)[0])
    want, off = checks.product(rows, layer)
    checks.assert_near(layer(rows, dtype=torch.float32), want, off, torch.float32)
    aligned = torch.zeros(n, 416, device="cuda").to(torch.float8_e4m3fn)
    aligned.view(torch.uint8)[:, :k] = codes.view(torch.uint8)
    aligned.view(torch.uint8)[:, k:] = 0x7f                      # (NaN behind the rows is not read)
    view = lib.Linear8(aligned[:, :k], scales)
    assert view.codes.data_ptr() == aligned.data_ptr()
    assert torch.equal(view(rows), layer(rows))


def test_no_rows(lib):
    layer = lib.Linear8.from_weight(torch.randn(130, 200, device="cuda"))
    rows = lib.quantise(torch.zeros(0, 200, device="cuda"))
    assert layer(rows).shape == (0, 130)
    ff = lib.FeedForward8(layer, layer, lib.Linear8.from_weight(torch.randn(200, 130, device="cuda")))
    assert ff(rows).shape == (0, 200) and ff.hidden(rows).shape == (0, 130)


# ---------------------------------------------------------------------------------------------------------- feed-forward
def block(lib, t, hidden, ffn, seed):
    x, gate = checks.case(t, ffn, hidden, seed)
    _, up = checks.case(1, ffn, hidden, seed + 1)
    _, down = checks.case(1, hidden, ffn, seed + 2)
    return lib.quantise(x), lib.FeedForward8(*(lib.Linear8.from_weight(w) for w in (gate, up, down)))


@pytest.mark.parametrize("t,hidden,ffn", [(1, 1, 1), (1, 4096, 1024), (3, 100, 129), (16, 512, 1536), (17, 256, 127), (33, 300, 500), (64, 512, 640), (65, 1024, 256),
                                          (128, 200, 384), (129, 640, 300), (203, 512, 1536), (257, 300, 260), (300, 512, 1000), (600, 256, 512), (1030, 512, 700), (2048, 256, 512)])
def test_feed_forward(lib, t, hidden, ffn):
    rows, ff = block(lib, t, hidden, ffn, t)
    h = ff.hidden(rows)
    checks.assert_hidden(h, *checks.hidden(rows, ff.gate, ff.up))
    y = ff(rows)
    ff.check()
    assert torch.equal(y, ff.down(h))
    want, off = checks.product(h, ff.down)
    checks.assert_near(y, want, off, torch.bfloat16)
    y32 = ff(rows, dtype=torch.float32)
    assert torch.equal(bits(y32), bits(ff.down(h, dtype=torch.float32)))


@pytest.mark.parametrize("t", [2, 70, 300, 1050])
def test_gates_far_from_zero(lib, t):
    """silu of large negative and positive numbers; what is not finite stays in its row."""
    x, gate = checks.case(t, 256, 256, 9)
    rows = lib.quantise(x * 30)
    ff = lib.FeedForward8(lib.Linear8.from_weight(gate), lib.Linear8.from_weight(gate.flip(0)), lib.Linear8.from_weight(gate))
    checks.assert_hidden(ff.hidden(rows), *checks.hidden(rows, ff.gate, ff.up))
    x[t - 1, 3] = float("inf")
    h = ff.hidden(lib.quantise(x))
    assert h.scales[:, t - 1].isnan().all() and h.scales[:, : t - 1].isfinite().all() and (h.codes[t - 1].float() == 0).all()


# ------------------------------------------------------------------------------------------------- as they are used together
def layer_of(lib, x, res, norm, qkv, ff):
    """The linear half of a decoder layer: norm -> qkv product; norm -> feed-forward."""
    a = qkv(lib.quantise(x, norm=norm, residual=res))
    return ff(lib.quantise(a[:, : x.shape[1]], norm=norm, residual=res))


@pytest.mark.parametrize("t", [1, 24, 150, 400, 1100])
def test_a_layer_captured_replayed_and_on_other_streams(lib, t):
    hidden = 512
    _, ff = block(lib, 1, hidden, 1536, 3)
    qkv = lib.Linear8.from_weight(checks.case(1, 768, hidden, 4)[1])
    norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
    xs = [checks.case(t, 1, hidden, 20 + i)[0] for i in range(4)]
    ress = [checks.case(t, 1, hidden, 40 + i)[0] for i in range(4)]
    want, want_res = [], []
    for x, r in zip(xs, ress):
        r = r.clone()
        want.append(layer_of(lib, x, r, norm, qkv, ff))
        want_res.append(r)
    # captured once, replayed on other data
    x, r = xs[0].clone(), ress[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_of(lib, x, r, norm, qkv, ff)
    for i in (2, 0, 3):
        x.copy_(xs[i])
        r.copy_(ress[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(r, want_res[i])
    # four streams at once
    streams = [torch.cuda.Stream() for _ in range(4)]
    here = [a.clone() for a in ress]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                here[i].copy_(ress[i])
                got.append(layer_of(lib, xs[i], here[i], norm, qkv, ff))
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(got[i], want[i]) and torch.equal(here[i], want_res[i])


def test_rows_of_a_call_do_not_depend_on_their_neighbours(lib):
    """What one row's result is does not depend on what the other rows of the call hold."""
    for t in (5, 40, 200, 500, 1500):
        x, w = checks.case(t, 384, 896, 6)
        layer = lib.Linear8.from_weight(w)
        y = layer(lib.quantise(x))
        other = x.clone()
        other[: t - 1] *= 1e6
        assert torch.equal(layer(lib.quantise(other))[t - 1], y[t - 1])


def test_refusals(lib):
    dev = torch.device("cuda", 0)
    layer = lib.Linear8.from_weight(torch.randn(130, 200, device=dev))
    rows = lib.quantise(torch.randn(4, 200, device=dev))
    for call, says in [
            (lambda: lib.quantise(torch.randn(4, 200)), "x:"), (lambda: lib.quantise(torch.randn(4, 200, device=dev).half()), "x:"),
            (lambda: lib.quantise(torch.randn(200, 4, device=dev).t()), "contiguous rows"), (lambda: lib.quantise(torch.randn(1, 200, device=dev).expand(3, 200)), "x:"),
            (lambda: lib.quantise(torch.zeros(3, 0, device=dev)), "x:"), (lambda: lib.quantise(torch.zeros(1, 131073, device=dev)), "x:"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), norm=torch.ones(200, device=dev)), "norm"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), norm=torch.ones(200, device=dev).bfloat16(), eps=0.0), "eps"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), norm=torch.ones(200, device=dev).bfloat16(), eps=float("nan")), "eps"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), residual=torch.randn(4, 200, device=dev).bfloat16()), "residual"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), residual=torch.randn(3, 200, device=dev)), "residual"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), residual_out=torch.randn(4, 200, device=dev)), "residual_out"),
            (lambda: lib.quantise(torch.randn(4, 200, device=dev), out=lib.Rows8(4, 201, dev)), "out"),
            (lambda: lib.Linear8(layer.codes.float(), layer.scales), "codes"), (lambda: lib.Linear8(layer.codes, layer.scales[:, :1]), "scales"),
            (lambda: lib.Linear8(layer.codes, layer.scales.double()), "scales"), (lambda: lib.Linear8(layer.codes[:0], layer.scales), "codes"),
            (lambda: lib.Linear8.from_weight(torch.zeros(0, 5, device=dev)), "w:"),
            (lambda: layer(lib.quantise(torch.randn(4, 201, device=dev))), "x:"), (lambda: layer(rows, out=torch.empty(4, 131, device=dev)), "out"),
            (lambda: layer(rows, out=torch.empty(130, 4, device=dev).t()), "contiguous rows"), (lambda: layer(rows, dtype=torch.float16), "dtype"),
            (lambda: lib.FeedForward8(layer, layer, layer), "feed-forward"), (lambda: lib.FeedForward8(layer, layer, lib.Linear8.from_weight(torch.randn(9, 130, device=dev)))(
                lib.quantise(torch.randn(4, 130, device=dev))), "x:")]:
        with pytest.raises(ValueError, match=says):
            call()


def test_codes_of_bf16_numbers_by_many_scales(lib):
    """Quotients are made by corrections, not by a division: every bf16 number against scales of all kinds and sizes."""
    gen = torch.Generator().manual_seed(1)
    top = torch.cat([torch.randint(0x0001, 0x7f80, (300,), generator=gen), torch.arange(0x3f80, 0x4000), torch.arange(0x0001, 0x0100, 7), torch.arange(0x7f00, 0x7f80, 3)])
    every = torch.randint(0, 0x7f80, (len(top), 127 * 40), generator=gen)
    every = torch.minimum(every % (0x0700) + (top[:, None] - 0x0700).clamp(min=0), top[:, None])   # (within 2^14 of the group's largest)
    x = torch.cat([every.view(-1, 127), top.repeat_interleave(40)[:, None]], dim=1).to(torch.int16).view(torch.bfloat16)
    x = (x * (1 - 2 * torch.randint(0, 2, x.shape, generator=gen)).to(torch.bfloat16)).cuda()
    rows = lib.quantise(x)
    codes, scales = checks.groups_of(x.float(), 1)
    same_groups(rows.codes, rows.scales, codes, scales.t())
    assert torch.equal(rows.codes.float().signbit(), x.signbit())
    more = x.float() * (1 + 2.0 ** -8 * torch.rand(x.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"))
    more = torch.where(more.isfinite(), more, x.float())
    codes, scales = checks.groups_of(more, 1)
    rows = lib.quantise(more)
    same_groups(rows.codes, rows.scales, codes, scales.t())


def test_matrices_that_lie_otherwise(lib):
    """Codes by columns, broadcast, out of a larger tensor, a single row at an odd place."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    codes = (torch.randn(300, 260, device="cuda", generator=gen) * 40).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.rand(3, 3, device="cuda", generator=gen)
    rows = lib.quantise(torch.randn(20, 260, device="cuda", generator=gen))
    want = lib.Linear8(codes.clone(), scales)(rows)
    by_columns = codes.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    assert by_columns.stride(1) != 1 and torch.equal(lib.Linear8(by_columns, scales)(rows), want)
    for left in (0, 1, 16):
        wide = torch.zeros(300, 304, dtype=torch.uint8, device="cuda")
        wide[:, left:left + 260] = codes.view(torch.uint8)
        assert torch.equal(lib.Linear8(wide.view(torch.float8_e4m3fn)[:, left:left + 260], scales)(rows), want)
    one = lib.Linear8(codes[7:8], scales[:1])
    assert torch.equal(one(rows)[:, 0], lib.Linear8(codes[7:8].clone(), scales[:1])(rows)[:, 0])
    same = lib.Linear8(codes[:1].expand(300, 260), scales)
    assert torch.equal(same(rows), lib.Linear8(codes[:1].expand(300, 260).contiguous(), scales)(rows))


def test_offsets_behind_32_bits(lib):
    """Codes and results whose places need more than 31 bits."""
    t, k = 16500, 131072                                    # 2.16e9 codes
    x = torch.zeros(t, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, k, device="cuda").bfloat16()
    x[5] = 1.0
    layer = lib.Linear8.from_weight(torch.randn(40, k, device="cuda") * k ** -0.5)
    rows = lib.quantise(x)
    del x
    y = layer(rows, dtype=torch.float32)
    some = lib.Rows8(4, k, y.device)
    some.codes.view(torch.uint8)[:] = rows.codes.view(torch.uint8)[[5, t - 3, t - 2, t - 1]]
    some.scales[:] = rows.scales[:, [5, t - 3, t - 2, t - 1]]
    want, off = checks.product(some, layer)
    checks.assert_near(y[[5, t - 3, t - 2, t - 1]], want, off, torch.float32)
    assert (y[6:t - 3] == 0).all() and (y[:5] == 0).all()
    del rows, y, some
    t, n, k = 70000, 33000, 130                             # 2.3e9 results
    x = torch.randn(t, k, device="cuda")
    layer = lib.Linear8.from_weight(torch.randn(n, k, device="cuda"))
    rows = lib.quantise(x)
    y = layer(rows)
    for at in (0, 40000, t - 1):
        some = lib.quantise(x[at:at + 1])
        want, off = checks.product(some, layer)
        checks.assert_near(y[at:at + 1], want, off, torch.bfloat16)
    del y
    h = lib.FeedForward8(layer, layer, lib.Linear8.from_weight(torch.randn(8, n, device="cuda"))).hidden(rows)   # 2.3e9 codes
    some = lib.quantise(x[t - 1:])
    want, off = checks.hidden(some, layer, layer)
    got = lib.Rows8(1, n, x.device)
    got.codes.view(torch.uint8)[:] = h.codes.view(torch.uint8)[t - 1:]
    got.scales[:] = h.scales[:, t - 1:]
    checks.assert_hidden(got, want, off)


def test_first_calls_in_a_capture():
    """A process whose first quantisation and product are captured."""
    import subprocess
    import sys

    code = """
import torch
from vllm_tgis_adapter_b200.engine import linear8 as lib
x = torch.randn(3, 256, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        lib.Linear8.from_weight(x)
    raise SystemExit("a layer was made")
except ValueError as e:
    assert "before a capture" in str(e), e
with torch.cuda.graph(graph):
    first = lib.quantise(x)
graph.replay()
assert torch.equal(first.codes.float(), lib.quantise(x).codes.float())
layers = [lib.Linear8.from_weight(torch.randn(n, 256, device="cuda")) for n in (300, 300, 200)]
layers[2] = lib.Linear8.from_weight(torch.randn(256, 300, device="cuda"))
ff, wide = lib.FeedForward8(*layers), torch.randn(400, 256, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = [ff(lib.quantise(z)) for z in (x, wide)]
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, ff(lib.quantise(z))) for a, z in zip(y, (x, wide)))
ff.check()
print("ok")
"""
    from pathlib import Path

    got = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip().endswith("ok"), got.stderr[-2000:] + got.stdout


def test_threads_call_at_once(lib):
    """Host threads on streams of their own: launches, shared layers, first calls of a size."""
    import threading

    layer = lib.Linear8.from_weight(torch.randn(512, 640, device="cuda"))
    xs = [torch.randn(t, 640, device="cuda") for t in (1, 30, 90, 200, 600, 1200)]
    want = [layer(lib.quantise(x)) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(30):
                    j = (i + k) % len(xs)
                    y = layer(lib.quantise(xs[j]))
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[j]):
                        bad.append((i, j))
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


# 65 to 128 tokens and more than eight k-blocks: the widest form of the kernel that has the weights on its rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", [(65, 1, 1025), (65, 129, 1100), (96, 300, 2048), (100, 77, 1200), (127, 2128, 4096), (128, 128, 1152), (128, 513, 20001), (128, 6144, 4096), (72, 40, 131072)])
def test_product_of_a_wide_batch(lib, t, n, k, dtype):
    x, w = checks.case(t, n, k, t + n + k)
    rows, layer = lib.quantise(x), lib.Linear8.from_weight(w)
    out = torch.full((t + 2, n + 5), 7.0, device="cuda", dtype=dtype)
    y = layer(rows, out=out[1 : t + 1, 2 : n + 2])
    want, off = checks.product(rows, layer)
    checks.assert_near(y, want, off, dtype)
    assert torch.equal(bits(layer(rows, dtype=dtype).contiguous()), bits(y.contiguous()))
    out[1 : t + 1, 2 : n + 2] = 7.0
    assert (out == 7.0).all()


def test_what_is_not_finite_in_a_wide_batch(lib):
    x, w = checks.case(100, 300, 2000, 5)
    x[3, 700], x[41, 0], x[99, 1999], w[140, 1500] = float("nan"), float("inf"), float("-inf"), float("nan")
    y = lib.Linear8.from_weight(w)(lib.quantise(x))
    gone = torch.zeros(100, 300, dtype=torch.bool, device="cuda")
    gone[[3, 41, 99]] = True
    gone[:, 128:256] = True
    assert torch.equal(y.isnan(), gone) and y[~gone].isfinite().all()


def test_rows_of_a_wide_batch_do_not_depend_on_their_neighbours(lib):
    x, w = checks.case(120, 640, 4096, 9)
    layer = lib.Linear8.from_weight(w)
    y = layer(lib.quantise(x))
    x[:60] = 3.0
    assert torch.equal(layer(lib.quantise(x))[60:], y[60:])


# as many rows as run at once, one more, and those around the sizes where a row's CTA grows
@pytest.mark.parametrize("t", [147, 149, 295, 297, 591, 593])
@pytest.mark.parametrize("k", [1024, 1040, 2048, 2056, 4096])
def test_rows_around_full_waves(lib, t, k):
    x, _ = checks.case(t, 1, k, t + k)
    rows = lib.quantise(x)
    codes, scales = checks.groups_of(x.float(), 1)
    same_groups(rows.codes, rows.scales, codes, scales.t())


def test_hidden_rows_do_not_take_the_place_of_x(lib):
    ff = block(lib, 5, 256, 256, 1)[1]
    rows = lib.quantise(checks.case(5, 1, 256, 3)[0])
    keep = rows.codes.view(torch.uint8).clone()
    with pytest.raises(ValueError, match="x itself"):
        ff.hidden(rows, out=rows)
    assert torch.equal(rows.codes.view(torch.uint8), keep)


@pytest.mark.parametrize("t,k,norm", [(1, 4096, True), (300, 1000, False), (600, 77, True), (200, 2304, True)])
def test_the_sum_takes_the_place_of_x_or_of_both(lib, t, k, norm):
    w = torch.rand(k, device="cuda").to(torch.bfloat16) + 0.5 if norm else None
    x, other = checks.case(t, 1, k, 1)[0], checks.case(t, 1, k, 2)[0]
    r = (x.float() + other.float()).to(x.dtype)
    want = lib.quantise(r.clone(), norm=w)
    rows = lib.quantise(x, norm=w, residual=other, residual_out=x)
    assert torch.equal(x, r) and torch.equal(rows.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(rows.scales, want.scales)
    twice = (other.float() * 2).to(x.dtype)
    want = lib.quantise(twice.clone(), norm=w)
    rows = lib.quantise(other, norm=w, residual=other)
    assert torch.equal(other, twice) and torch.equal(rows.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(rows.scales, want.scales)
