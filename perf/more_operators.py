"""Products with 8-bit weights, as a serving program calls them in a layer.

Four kinds of case:

  rows     a step's rows on their way into a product: residual added and RMS norm taken where a layer does so, then 8 bits: every
           128 neighbouring numbers of a row are e4m3 codes with one fp32 scale.  Out: codes, scales, the new residual.
  weights  a weight matrix when a model is loaded: every block of 128 x 128 as e4m3 codes with one fp32 scale.  Out: codes, scales.
  product  8-bit rows times an 8-bit weight matrix.  Out: one row a token, bf16 or fp32.
  ffn      a gated feed-forward block: silu(gate x) * (up x) in 8-bit rows, then the down projection.  Out: one row a token, bf16.

A group of numbers v (1 x 128 of a row, 128 x 128 of a weight; smaller at the ends) has s = max(max |v| * (1 / 448), 2^-126) and codes
c = e4m3(v / s), and stands for c * s.  With a norm, v = r w / rms(r): the codes are those of r w, and 1 / rms goes into the scales.
Sizes are those of the repository's Llama presets (hidden and feed-forward sizes, fused qkv), of its products' tests, and generic odd ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

GROUP, TOP, TINY, EPS = 128, 448.0, 2.0 ** -126, 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# rows x columns of the presets' weights: fused qkv, attention output, down projection, the two feed-forward halves
WEIGHTS = [(512, 256), (256, 512), (1536, 512), (512, 1536), (1280, 768), (1536, 1024), (2048, 2048), (11264, 2048), (2048, 11264), (2128, 2048), (6144, 4096),
           (4096, 4096), (14336, 4096), (4096, 14336), (10240, 8192), (8192, 8192)]
FEED_FORWARDS = [(256, 512), (512, 1536), (2048, 11264), (4096, 14336)]   # hidden, feed-forward


# ------------------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # the next token of one request on its way into the qkv product: nothing but latency
        dict(name="rows-one", kind="rows", t=1, k=4096, dtype="bf16", norm=True, residual=True),
        # a full prefill step, the same place
        dict(name="rows-prompts", kind="rows", t=2048, k=4096, dtype="bf16", norm=True, residual=True),
        # a small odd matrix of a checkpoint
        dict(name="weights-odd", kind="weights", n=2128, k=2048, dtype="bf16"),
        # the largest matrix of a large model's layer, from fp32
        dict(name="weights-large", kind="weights", n=28672, k=8192, dtype="fp32"),
        # the next token of one request: its qkv product
        dict(name="product-one", kind="product", t=1, n=6144, k=4096, out="bf16"),
        # the headline batch of 32 decoding requests: the down projection
        dict(name="product-batch", kind="product", t=32, n=4096, k=14336, out="bf16"),
        # a short prompt beside decoding requests, rows that fill no tile, results in fp32
        dict(name="product-odd", kind="product", t=301, n=2128, k=11264, out="fp32"),
        # a full prefill step of a large model: the attention's output projection
        dict(name="product-prompts", kind="product", t=2048, n=8192, k=8192, out="bf16"),
        # one request's next token through the feed-forward block
        dict(name="ffn-one", kind="ffn", t=1, hidden=4096, ffn=14336),
        # a busy server's decode step
        dict(name="ffn-batch", kind="ffn", t=48, hidden=4096, ffn=14336),
        # a prompt on a small model
        dict(name="ffn-small", kind="ffn", t=203, hidden=512, ffn=1536),
        # a full prefill step
        dict(name="ffn-prompts", kind="ffn", t=2048, hidden=4096, ffn=14336),
    ]


def _between(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rows", "weights", "product", "product", "product", "ffn", "ffn"])
    n, k = rng.choice(WEIGHTS) if rng.random() < 0.7 else (_between(rng, 40, 9000), _between(rng, 100, 9000))
    if kind == "rows":
        norm = rng.random() < 0.6
        return dict(kind=kind, t=_between(rng, 1, 2048), k=k, dtype=rng.choice(["bf16", "bf16", "fp32"]), norm=norm, residual=norm and rng.random() < 0.7)
    if kind == "weights":
        return dict(kind=kind, n=n, k=k, dtype=rng.choice(["bf16", "fp32"]))
    if kind == "product":
        return dict(kind=kind, t=_between(rng, 1, 2048), n=n, k=k, out=rng.choice(["bf16", "bf16", "fp32"]))
    hidden, ffn = rng.choice(FEED_FORWARDS) if rng.random() < 0.7 else (_between(rng, 100, 4096), _between(rng, 200, 14336))
    return dict(kind=kind, t=_between(rng, 1, 2048), hidden=hidden, ffn=ffn)


# ------------------------------------------------------------------------------------------------------------ inputs
def _rows(gen, t: int, k: int) -> torch.Tensor:
    """Activations: a few channels carry large numbers, and tokens differ in size."""
    channel = torch.ones(k, device="cuda")
    channel[5::97] = 8.0
    return torch.randn(t, k, device="cuda", generator=gen) * channel * torch.exp(0.4 * torch.randn(t, 1, device="cuda", generator=gen))


def _weight(gen, n: int, k: int) -> torch.Tensor:
    """A weight matrix whose rows and columns differ in size."""
    w = torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5
    return w * torch.exp(0.3 * torch.randn(n, 1, device="cuda", generator=gen)) * torch.exp(0.3 * torch.randn(k, device="cuda", generator=gen))


def _matrix(gen, n: int, k: int) -> dict:
    codes, scales = _quantise_blocks(_weight(gen, n, k).to(torch.bfloat16))
    return dict(codes=codes, scales=scales)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(kind=case["kind"])
    if case["kind"] == "rows":
        t, k, dtype = case["t"], case["k"], TYPES[case["dtype"]]
        st.update(x=_rows(gen, t, k).to(dtype), norm=None, residual=None)
        if case["norm"]:
            st["norm"] = (1 + 0.2 * torch.randn(k, device="cuda", generator=gen)).to(torch.bfloat16)
        if case["residual"]:
            st["residual"] = _rows(gen, t, k).to(dtype)
        return st
    if case["kind"] == "weights":
        return dict(st, w=_weight(gen, case["n"], case["k"]).to(TYPES[case["dtype"]]))
    t, k = case["t"], case["k"] if case["kind"] == "product" else case["hidden"]
    x = _rows(gen, t, k).to(torch.bfloat16)
    if case["kind"] == "product":
        st.update(out=TYPES[case["out"]], weights=[_matrix(gen, case["n"], k)])
    else:
        st["weights"] = [_matrix(gen, case["ffn"], k), _matrix(gen, case["ffn"], k), _matrix(gen, k, case["ffn"])]
    if own:
        # the program's layers hold the checkpoint's matrices, and its last operator left the rows
        from vllm_tgis_adapter_b200.engine.linear8 import FeedForward8, Linear8, quantise

        layers = [Linear8(w["codes"], w["scales"]) for w in st.pop("weights")]
        st["layer"] = layers[0] if case["kind"] == "product" else FeedForward8(*layers)
        st["rows"] = quantise(x)
    else:
        st["codes"], st["scales"] = _quantise_rows(x.float())
    return st


# --------------------------------------------------------------------------------------------------------- plain form
def _padded(x: torch.Tensor, n: int, k: int) -> torch.Tensor:
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % k, 0, -x.shape[-2] % n))


def _codes(v: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return (v / s).to(torch.float8_e4m3fn)


def _quantise_rows(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 [T, K] -> codes [T, K], scales [groups, T]"""
    t, k = v.shape
    v = _padded(v, 1, GROUP).view(t, -1, GROUP)
    s = (v.abs().amax(dim=-1, keepdim=True) * (1 / TOP)).clamp(min=TINY)
    return _codes(v, s).view(t, -1)[:, :k], s[..., 0].t()


def _quantise_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[N, K] -> codes [N, K], scales [blocks of rows, groups]"""
    n, k = w.shape
    v = _padded(w.float(), GROUP, GROUP)
    v = v.view(v.shape[0] // GROUP, GROUP, -1, GROUP)
    s = (v.abs().amax(dim=(1, 3), keepdim=True) * (1 / TOP)).clamp(min=TINY)
    return _codes(v, s).view(v.shape[0] * GROUP, -1)[:n, :k].contiguous(), s[:, 0, :, 0].contiguous()


def _row_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return codes.float() * scales.t().repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]]


def _weight_values(w: dict) -> torch.Tensor:
    n, k = w["codes"].shape
    s = w["scales"].repeat_interleave(GROUP, dim=0)[:n].repeat_interleave(GROUP, dim=1)[:, :k]
    return w["codes"].float() * s


def _plain_rows(st: dict):
    x, new = st["x"].float(), None
    if st["residual"] is not None:
        new = (x + st["residual"].float()).to(st["x"].dtype)
        x = new.float()
    if st["norm"] is None:
        codes, scales = _quantise_rows(x)
        return dict(codes=codes, scales=scales)
    codes, scales = _quantise_rows(x * st["norm"].float())
    scales = scales * torch.rsqrt(x.square().mean(dim=-1) + EPS)
    return dict(codes=codes, scales=scales) if new is None else dict(codes=codes, scales=scales, residual=new)


def _plain_ffn(st: dict):
    gate, up, down = st["weights"]
    x = _row_values(st["codes"], st["scales"])
    g, u = x @ _weight_values(gate).t(), x @ _weight_values(up).t()
    codes, scales = _quantise_rows(g / (1 + torch.exp(-g)) * u)
    return (_row_values(codes, scales) @ _weight_values(down).t()).to(torch.bfloat16)


def run(st: dict):
    kind = st["kind"]
    if not own:
        if kind == "rows":
            return _plain_rows(st)
        if kind == "weights":
            codes, scales = _quantise_blocks(st["w"])
            return dict(codes=codes, scales=scales)
        if kind == "product":
            return (_row_values(st["codes"], st["scales"]) @ _weight_values(st["weights"][0]).t()).to(st["out"])
        return _plain_ffn(st)
    from vllm_tgis_adapter_b200.engine.linear8 import Linear8, quantise

    if kind == "rows":
        new = torch.empty_like(st["x"]) if st["residual"] is not None else None
        rows = quantise(st["x"], norm=st["norm"], eps=EPS, residual=st["residual"], residual_out=new)
        got = dict(codes=rows.codes, scales=rows.scales)
        return got if new is None else dict(got, residual=new)
    if kind == "weights":
        layer = Linear8.from_weight(st["w"])
        return dict(codes=layer.codes, scales=layer.scales)
    if kind == "product":
        return st["layer"](st["rows"], dtype=st["out"])
    return st["layer"](st["rows"])


# --------------------------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    size = {"bf16": 2, "fp32": 4}
    if case["kind"] == "rows":
        t, k, b = case["t"], case["k"], size[case["dtype"]]
        each = b + 1 + 4 / GROUP + (2 * b if case["residual"] else 0)
        return dict(bytes=t * k * each + (2 * k if case["norm"] else 0), flops=t * k * (4 + (3 if case["norm"] else 0)))
    if case["kind"] == "weights":
        n, k = case["n"], case["k"]
        return dict(bytes=n * k * (size[case["dtype"]] + 1 + 4 / GROUP ** 2), flops=4 * n * k)
    t = case["t"]
    if case["kind"] == "product":
        n, k = case["n"], case["k"]
        return dict(bytes=n * k * (1 + 4 / GROUP ** 2) + t * k * (1 + 4 / GROUP) + t * n * size[case["out"]], flops=2 * t * n * k)
    k, f = case["hidden"], case["ffn"]
    return dict(bytes=3 * f * k * (1 + 4 / GROUP ** 2) + t * k * (1 + 4 / GROUP + 2), flops=6 * t * f * k)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest number with three bits behind the first, none below 2^-6 with steps smaller than 2^-9; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_groups(v: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [R, K] and scales [R / rows, K / 128] of groups of `rows` x 128; a scale is a stored number of 32 bits."""
    r, k = v.shape
    padded = torch.zeros(-(-r // rows) * rows, -(-k // GROUP) * GROUP, dtype=torch.float64, device=v.device)
    padded[:r, :k] = v
    groups = padded.view(padded.shape[0] // rows, rows, padded.shape[1] // GROUP, GROUP)
    top = groups.abs().amax(dim=3).amax(dim=1)
    s = (top.float() * (1 / TOP)).clamp(min=TINY).double()
    return _to_e4m3(groups / s[:, None, :, None]).reshape(padded.shape)[:r, :k], s


def _spread(codes: torch.Tensor, s: torch.Tensor, rows: int) -> torch.Tensor:
    """What codes of groups of `rows` x 128 stand for."""
    i, j = (torch.arange(n, device=codes.device) // g for n, g in zip(codes.shape, (rows, GROUP)))
    return codes.double() * s.double()[i][:, j]


def exact(case: dict, seed: int):
    global own
    keep, own = own, False
    st = prepare(case, seed)
    own = keep
    if case["kind"] == "weights":
        codes, s = _exact_groups(st["w"].double(), GROUP)
        return dict(codes=codes, scales=s)
    if case["kind"] == "rows":
        r, out = st["x"].double(), {}
        if st["residual"] is not None:
            r = r + st["residual"].double()
            out["residual"] = r
            r = r.to(st["x"].dtype).double()
        if st["norm"] is None:
            codes, s = _exact_groups(r, 1)
        else:
            codes, s = _exact_groups(r * st["norm"].double(), 1)
            s = s / torch.sqrt((r * r).sum(dim=1, keepdim=True) / case["k"] + EPS)
        return dict(out, codes=codes, scales=s.t())
    x = _spread(st["codes"], st["scales"].t(), 1)
    if case["kind"] == "product":
        w, = st["weights"]
        return x @ _spread(w["codes"], w["scales"], GROUP).t()
    g, u = (x @ _spread(w["codes"], w["scales"], GROUP).t() for w in st["weights"][:2])
    h = _spread(*_exact_groups(g * torch.sigmoid(g) * u, 1), 1)
    return h @ _spread(st["weights"][2]["codes"], st["weights"][2]["scales"], GROUP).t()
