"""Products with 8-bit weights behind a kernel that takes long: their waits have a limit, what comes before them has none."""
import pytest
import torch

import linear8_checks as checks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from vllm_tgis_adapter_b200.engine import linear8

    return linear8


@pytest.fixture(scope="module")
def hold():
    from vllm_tgis_adapter_b200.engine import _lib

    library = _lib.load_library()
    limit = 4_000_000_000   # clocks, the kernels' own (csrc/tc_attention.cuh WAIT_LIMIT)

    def call():
        assert library.tgis_k_hold(limit + limit // 8, torch.cuda.current_stream().cuda_stream) == 0

    return call


# one for each kernel: tokens as columns (plain, wide, gated), pairs (plain, cut along k, gated)
@pytest.mark.parametrize("t,n,k,gated", [(1, 256, 1024, False), (100, 256, 2048, False), (40, 256, 1024, True), (300, 4096, 1024, False), (300, 256, 4096, False), (300, 1024, 512, True)])
def test_a_long_kernel_before_a_product_is_no_stall(lib, hold, t, n, k, gated):
    x, w = checks.case(t, n, k, 1)
    rows, one = lib.quantise(x), lib.Linear8.from_weight(w)
    if gated:
        block = lib.FeedForward8(one, lib.Linear8.from_weight(w.flip(0)), lib.Linear8.from_weight(checks.case(1, 128, n, 2)[1]))
        call, out = block.hidden, lib.Rows8(t, n, x.device)
    else:
        call, out = one, torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    want = call(rows)
    torch.cuda.synchronize()
    begun, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begun.record()
    hold()
    call(rows, out=out)
    ended.record()
    one.check()
    assert begun.elapsed_time(ended) > 2000
    if gated:
        assert torch.equal(out.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(out.scales, want.scales)
    else:
        assert torch.equal(out, want)


def test_hook_refuses():
    from vllm_tgis_adapter_b200.engine import _lib

    library = _lib.load_library()
    assert library.tgis_k_hold(-1, None) == -1 and library.tgis_k_hold(1 << 40, None) == -1
