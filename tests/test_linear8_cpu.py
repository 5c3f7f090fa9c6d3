"""Products with 8-bit weights without a GPU: exports, refusals before any launch."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from vllm_tgis_adapter_b200.engine import _lib, linear8

ROOT = Path(__file__).resolve().parent.parent
AT = 1 << 20   # an address that nothing is read from


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def test_every_declared_symbol_is_exported_and_bound(lib):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "tgis_w8.h").read_text(), flags=re.S)
    declared = set(re.findall(r"\b(tgis_w8_[a-z0-9_]+)\s*\(", text))
    assert declared == set(_lib.W8_SYMBOLS)
    for name in declared:
        assert hasattr(lib, name)
    sizes = {k: int(v) for k, v in re.findall(r"#define TGIS_W8_(\w+) (\d+)", text)}
    assert (sizes["GROUP"], sizes["MAX_K"]) == (linear8.GROUP, linear8.MAX_K)
    assert linear8.TYPES == {torch.bfloat16: sizes["BF16"], torch.float32: sizes["F32"]}
    assert C.sizeof(_lib.TgisW8Matrix) == 32 and C.sizeof(_lib.TgisW8Rows) == 40


def rows(**change):
    v = {**dict(codes=AT, scales=AT, ld=256, lds=4, t=3, k=200), **change}
    return _lib.TgisW8Rows(*v.values())


def matrix(**change):
    v = {**dict(codes=AT, scales=AT, ld=256, n=130, k=200), **change}
    return _lib.TgisW8Matrix(*v.values())


def refused(lib, rc, says):
    assert rc == -1 and says in lib.tgis_w8_last_error().decode()


BAD_ROWS = [(dict(codes=None), "codes"), (dict(codes=AT + 8), "codes"), (dict(ld=264), "codes"), (dict(scales=None), "scales"), (dict(scales=AT + 2), "scales"), (dict(lds=2), "scales"),
            (dict(t=-1), "rows"), (dict(t=1 << 23, lds=1 << 24), "rows"), (dict(k=0), "numbers"), (dict(k=131073, ld=131200), "numbers"), (dict(ld=1 << 40), "codes")]
BAD_MATRIX = [(dict(codes=None), "codes"), (dict(codes=AT + 4), "codes"), (dict(ld=250), "codes"), (dict(scales=None), "scales"), (dict(n=0), "rows"), (dict(n=-3), "rows"),
              (dict(k=0), "numbers"), (dict(ld=192), "codes")]


@pytest.mark.parametrize("change,says", [(c, s) for c, s in BAD_ROWS + [(dict(ld=208), "codes")]])
def test_quantise_rows_refuses_its_record(lib, change, says):
    r = rows(**change)
    refused(lib, lib.tgis_w8_quantise_rows(AT, 0, 200, None, 1e-5, None, 0, None, 0, C.addressof(r), None), says)


@pytest.mark.parametrize("args,says", [
    ((None, 0, 200, None, 1e-5, None, 0, None, 0), "x:"), ((AT + 1, 0, 200, None, 1e-5, None, 0, None, 0), "x:"), ((AT + 2, 1, 200, None, 1e-5, None, 0, None, 0), "x:"),
    ((AT, 0, 199, None, 1e-5, None, 0, None, 0), "x:"), ((AT, 2, 200, None, 1e-5, None, 0, None, 0), "type"), ((AT, 0, 200, AT, 0.0, None, 0, None, 0), "eps"),
    ((AT, 0, 200, AT, float("inf"), None, 0, None, 0), "eps"), ((AT, 0, 200, AT, float("nan"), None, 0, None, 0), "eps"), ((AT, 0, 200, AT + 1, 1e-5, None, 0, None, 0), "norm"),
    ((AT, 0, 200, None, 1e-5, AT, 100, AT, 200), "residual"), ((AT, 0, 200, None, 1e-5, AT, 200, None, 200), "residual_out"),
    ((AT, 0, 200, None, 1e-5, 2 * AT, 200, 2 * AT, 208), "in place"), ((AT, 0, 200, None, 1e-5, 2 * AT, 200, AT, 208), "in place")])
def test_quantise_rows_refuses(lib, args, says):
    r = rows()
    refused(lib, lib.tgis_w8_quantise_rows(*args, C.addressof(r), None), says)


@pytest.mark.parametrize("change,says", BAD_MATRIX + [(dict(ld=208), "codes")])
def test_quantise_weight_refuses(lib, change, says):
    m = matrix(**change)
    refused(lib, lib.tgis_w8_quantise_weight(AT, 0, 200, C.addressof(m), None), says)
    m = matrix()
    refused(lib, lib.tgis_w8_quantise_weight(None, 0, 200, C.addressof(m), None), "w:")
    refused(lib, lib.tgis_w8_quantise_weight(AT, 5, 200, C.addressof(m), None), "type")
    refused(lib, lib.tgis_w8_quantise_weight(AT, 0, 199, C.addressof(m), None), "w:")


def test_products_refuse(lib):
    at = C.byref
    for change, says in BAD_ROWS:
        r, m = rows(**change), matrix()
        refused(lib, lib.tgis_w8_product(at(r), at(m), AT, 0, 130, None, None), says)
        refused(lib, lib.tgis_w8_gated(at(r), at(m), at(m), at(rows(k=130)), None, None), says)
    for change, says in BAD_MATRIX:
        r, m, good = rows(), matrix(**change), matrix()
        refused(lib, lib.tgis_w8_product(at(r), at(m), AT, 0, 130, None, None), says)
        refused(lib, lib.tgis_w8_gated(at(r), at(good), at(m), at(rows(k=130)), None, None), says)
    r, m, h = rows(), matrix(), rows(k=130)
    refused(lib, lib.tgis_w8_product(at(rows(k=199)), at(m), AT, 0, 130, None, None), "numbers")
    refused(lib, lib.tgis_w8_product(at(r), at(m), None, 0, 130, None, None), "y:")
    refused(lib, lib.tgis_w8_product(at(r), at(m), AT + 2, 1, 130, None, None), "y:")
    refused(lib, lib.tgis_w8_product(at(r), at(m), AT, 0, 129, None, None), "y:")
    refused(lib, lib.tgis_w8_product(at(r), at(m), AT, 3, 130, None, None), "type")
    refused(lib, lib.tgis_w8_product(None, at(m), AT, 0, 130, None, None), "record")
    refused(lib, lib.tgis_w8_gated(at(r), at(m), at(matrix(n=131)), at(h), None, None), "up")
    refused(lib, lib.tgis_w8_gated(at(r), at(m), at(m), at(rows(k=131)), None, None), "out")
    refused(lib, lib.tgis_w8_gated(at(r), at(m), at(m), at(rows(k=130, t=2)), None, None), "out")
    down = matrix(n=64, k=130)
    refused(lib, lib.tgis_w8_feed_forward(at(r), at(m), at(m), at(matrix(n=64, k=128)), at(h), AT, 0, 64, None, None), "down")
    refused(lib, lib.tgis_w8_feed_forward(at(r), at(m), at(m), at(down), at(h), None, 0, 64, None, None), "y:")


@pytest.mark.parametrize("change", [dict(), dict(scales=AT + 4096), dict(codes=AT + 4096)])
def test_rows_do_not_take_the_place_of_those_they_are_made_of(lib, change):
    at = C.byref
    r, m, h, down = rows(), matrix(), rows(k=130, **change), matrix(n=64, k=130)
    refused(lib, lib.tgis_w8_gated(at(r), at(m), at(m), at(h), None, None), "out: x itself")
    refused(lib, lib.tgis_w8_feed_forward(at(r), at(m), at(m), at(down), at(h), AT, 0, 64, None, None), "hidden: x itself")


def test_nothing_to_do_is_no_error(lib):
    at, r, m = C.byref, rows(t=0, codes=None), matrix()
    assert lib.tgis_w8_quantise_rows(None, 0, 0, None, 0.0, None, 0, None, 0, at(r), None) == 0
    assert lib.tgis_w8_product(at(r), at(m), None, 0, 0, None, None) == 0
    h = rows(t=0, k=130)
    assert lib.tgis_w8_gated(at(r), at(m), at(m), at(h), None, None) == 0
    assert lib.tgis_w8_feed_forward(at(r), at(m), at(m), at(matrix(n=64, k=130)), at(h), None, 0, 0, None, None) == 0


def test_binding_refuses_tensors_off_the_device():
    with pytest.raises(ValueError, match="x:"):
        linear8.quantise(torch.zeros(2, 128))
    with pytest.raises(ValueError, match="codes"):
        linear8.Linear8(torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="w:"):
        linear8.Linear8.from_weight(torch.zeros(2, 128))


@pytest.mark.parametrize("weights,change,says", [(7, {}, "weights"), (1, dict(arch=_lib.ARCH_OPT, head_dim=64, hidden=64), "Llama"), (1, dict(tp_size=2, n_kv_heads=2, n_q_heads=2), "single GPU"),
                                                 (1, dict(max_loras=1, max_lora_rank=8), "LoRA"), (1, dict(debug_gemm_ref=1), "debug_gemm_ref"), (1, dict(ffn=131136), "131072")])
def test_engine_refuses(lib, weights, change, says):
    cfg = _lib.TgisConfig()
    cfg.abi_version = _lib.ABI_VERSION
    values = dict(n_layers=1, hidden=128, n_q_heads=1, n_kv_heads=1, head_dim=128, ffn=128, vocab=64, max_model_len=64, max_num_seqs=1, max_batched_tokens=64, tp_size=1)
    for name, value in {**values, **change}.items():
        setattr(cfg, name, value)
    handle = C.c_void_p()
    assert lib.tgis_engine_create_weights(C.byref(cfg), weights, C.byref(handle)) != 0
    assert says in lib.tgis_last_error().decode()


def test_flag():
    from vllm_tgis_adapter_b200.engine.core import PRESETS, EngineError, NativeEngine
    from vllm_tgis_adapter_b200.engine.ponenex import PRESETS as LISTS
    from vllm_tgis_adapter_b200.tgis_utils.args import parse_args

    assert parse_args(["--model", "tiny"]).quantization is None
    assert parse_args(["--model", "tiny", "--quantization", "fp8"]).quantization == "fp8"
    with pytest.raises(SystemExit):
        parse_args(["--model", "tiny", "--quantization", "int4"])
    with pytest.raises(EngineError, match="quantization"):
        NativeEngine(PRESETS["tiny"], quantization="int4")
    with pytest.raises(EngineError, match="Llama"):
        NativeEngine(LISTS["ponenex-1k"], quantization="fp8")
