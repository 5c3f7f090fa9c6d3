"""The 8-bit cache's C ABI and binding without a GPU: exports, refusals before any launch, workspace bounds, layout."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from vllm_tgis_adapter_b200.engine import _lib, cache8

ROOT = Path(__file__).resolve().parent.parent
AT = 1 << 20   # an address that nothing is read from


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def header() -> str:
    return re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "tgis_kv8.h").read_text(), flags=re.S)


def test_every_declared_symbol_is_exported_and_bound(lib):
    declared = set(re.findall(r"\b(tgis_kv8_[a-z0-9_]+)\s*\(", header()))
    assert declared == set(_lib.KV8_SYMBOLS)
    for name in declared:
        assert hasattr(lib, name)
    sizes = {k: int(v) for k, v in re.findall(r"#define TGIS_KV8_(\w+) (\d+)", header())}
    assert (sizes["PAGE_TOKENS"], sizes["PAGE_BYTES"], sizes["MAX_TREE"], sizes["MAX_SEQS"]) == (cache8.PAGE_TOKENS, cache8.PAGE_BYTES, cache8.MAX_TREE, cache8.MAX_SEQS)
    assert sizes["PAGE_BYTES"] == 2 * 32 * 128 + 2 * 32 * 4


WRITE = dict(pages=AT, n_pages=4, n_kv=2, qkv=AT, ld=1024, T=3, n_q=4, positions=AT, slots=AT, cos_sin=AT, n_positions=9, q_out=AT, ldq=512, status=None, stream=None)
READ = dict(pages=AT, n_pages=4, n_kv=2, slots=AT, T=3, k_out=AT, ldk=256, v_out=AT, ldv=256, status=None, stream=None)
ATTEND = dict(pages=AT, n_pages=4, n_kv=2, q=AT, ldq=512, T=3, n_q=4, seqs=AT, n_seqs=1, block_table=AT, bt_rows=1, bt_stride=4, tree=None, scale=0.1, max_q=3,
              max_kv=100, out=AT, ldo=512, workspace=AT, workspace_bytes=1 << 30, status=None, stream=None)


@pytest.mark.parametrize("change,says", [
    (dict(pages=None), "pages"), (dict(pages=AT + 8), "pages"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 26), "n_pages"), (dict(n_kv=0), "n_kv"),
    (dict(n_q=-1), "n_q"), (dict(T=-1), "T "), (dict(qkv=None), "qkv"), (dict(qkv=AT + 2), "qkv"), (dict(ld=1016), "qkv"), (dict(ld=1028), "qkv"),
    (dict(q_out=AT + 8), "q_out"), (dict(ldq=504), "q_out"), (dict(q_out=AT, qkv=AT, ldq=512), "in place"), (dict(positions=None), "positions"), (dict(slots=AT + 1), "slots"),
    (dict(cos_sin=None), "cos_sin"), (dict(n_positions=0), "cos_sin")])
def test_write_refuses(lib, change, says):
    args = {**WRITE, "qkv": AT + 4096, **change}
    assert lib.tgis_kv8_write(*args.values()) == -1
    assert says in lib.tgis_kv8_last_error().decode()


@pytest.mark.parametrize("change,says", [(dict(pages=None), "pages"), (dict(slots=None), "slots"), (dict(T=-3), "T "), (dict(ldk=248), "k_out"), (dict(v_out=AT + 4), "v_out"), (dict(ldv=260), "v_out")])
def test_read_refuses(lib, change, says):
    assert lib.tgis_kv8_read(*{**READ, **change}.values()) == -1
    assert says in lib.tgis_kv8_last_error().decode()


@pytest.mark.parametrize("change,says", [
    (dict(n_kv=3), "n_q"), (dict(n_q=0), "n_q"), (dict(n_q=2048, n_kv=2), "n_q"), (dict(T=-1), "T "), (dict(n_seqs=-1), "n_seqs"), (dict(n_seqs=4097), "n_seqs"),
    (dict(max_q=-1), "max_q"), (dict(max_kv=-1), "max_kv"), (dict(q=None), "q:"), (dict(ldq=511), "q:"), (dict(out=AT + 2), "out"), (dict(ldo=256), "out"),
    (dict(seqs=None), "seqs"), (dict(seqs=AT + 4), "seqs"), (dict(block_table=None), "block_table"), (dict(bt_stride=0), "block_table"), (dict(bt_rows=0), "block_table"),
    (dict(tree=AT + 4), "tree"), (dict(tree=AT, max_q=65), "tree"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(workspace=None, max_kv=9000), "workspace"), (dict(workspace_bytes=7, max_kv=9000), "workspace"), (dict(workspace=AT + 8, max_kv=9000), "workspace")])
def test_attention_refuses(lib, change, says):
    assert lib.tgis_kv8_attention(*{**ATTEND, **change}.values()) == -1
    assert says in lib.tgis_kv8_last_error().decode()


def test_nothing_to_do_is_no_error(lib):
    assert lib.tgis_kv8_write(*{**WRITE, "T": 0, "qkv": None}.values()) == 0
    assert lib.tgis_kv8_read(*{**READ, "T": 0}.values()) == 0
    assert lib.tgis_kv8_attention(*{**ATTEND, "n_seqs": 0}.values()) == 0
    assert lib.tgis_kv8_attention(*{**ATTEND, "max_q": 0}.values()) == 0


def test_workspace_grows_with_the_bounds(lib):
    """Whoever keeps one workspace sizes it for the largest call: no smaller call of the same heads may need more."""
    size = lib.tgis_kv8_attention_workspace
    for n_q, n_kv in ((32, 8), (64, 8), (4, 1)):
        for tokens, seqs, q in ((1, 1, 1), (32, 32, 1), (96, 12, 8)):
            last = 0
            for kv in (1, 31, 128, 129, 500, 2048, 8192, 60000):
                now = size(tokens, seqs, n_q, n_kv, q, kv)
                assert now >= last >= 0
                last = now
    assert size(1, 1, 4, 3, 1, 1) == -1 and b"n_q" in lib.tgis_kv8_last_error()


def test_binding_refuses_tensors_off_the_device():
    with pytest.raises(ValueError, match="pages"):
        cache8.Cache8(torch.zeros(2, 1, cache8.PAGE_BYTES, dtype=torch.uint8))


@pytest.mark.parametrize("change,says", [(dict(kv_cache_dtype=7), "kv_cache_dtype"), (dict(kv_cache_dtype=1, arch=_lib.ARCH_OPT, head_dim=64, hidden=64), "Llama"),
                                         (dict(kv_cache_dtype=1, max_num_seqs=5000), "sequences")])
def test_engine_refuses(lib, change, says):
    cfg = _lib.TgisConfig()
    cfg.abi_version = _lib.ABI_VERSION
    values = dict(n_layers=1, hidden=128, n_q_heads=1, n_kv_heads=1, head_dim=128, ffn=128, vocab=64, max_model_len=64, max_num_seqs=1, max_batched_tokens=64, tp_size=1)
    for name, value in {**values, **change}.items():
        setattr(cfg, name, value)
    handle = C.c_void_p()
    assert lib.tgis_engine_create(C.byref(cfg), C.byref(handle)) != 0
    assert says in lib.tgis_last_error().decode()


def test_flag_and_block_bytes():
    from vllm_tgis_adapter_b200.engine.core import PRESETS, EngineError, NativeEngine, cache_block_bytes
    from vllm_tgis_adapter_b200.tgis_utils.args import parse_args

    assert parse_args(["--model", "tiny"]).kv_cache_dtype == "auto"
    assert parse_args(["--model", "tiny", "--kv-cache-dtype", "fp8"]).kv_cache_dtype == "fp8"
    with pytest.raises(SystemExit):
        parse_args(["--model", "tiny", "--kv-cache-dtype", "int4"])
    mc = PRESETS["llama3-8b"]
    assert cache_block_bytes(mc) == 2 * 32 * 8 * 32 * 128 * 2 and cache_block_bytes(mc, "fp8") == 32 * 8 * 8448
    with pytest.raises(EngineError, match="kv_cache_dtype"):
        NativeEngine(mc, kv_cache_dtype="int4")


@pytest.mark.parametrize("n_q,n_kv", [(32, 8), (6, 2), (64, 8), (8, 1)])
@pytest.mark.parametrize("max_q", [1, 4, 12])
def test_workspace_grows_with_sequences_and_their_lengths(lib, n_q, n_kv, max_q):
    """A workspace for the largest call holds every smaller one (what a server allocates once)."""
    ask = lambda n, kv: lib.tgis_kv8_attention_workspace(n * max_q, n, n_q, n_kv, max_q, kv)
    for n in (1, 7, 12, 56, 256):
        sizes = [ask(n, kv) for kv in [*range(16, 5000, 61), 8192, 32768, 131072]]
        assert sizes == sorted(sizes)
    for kv in (600, 1000, 3000, 8192):
        sizes = [ask(n, kv) for n in range(1, 200)]
        assert sizes == sorted(sizes)
